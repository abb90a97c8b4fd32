"""A checkpoint that does not fit is refused as a whole: nothing of the optimizer has changed by then."""
import numpy as np
import pytest

U8, U16, F32 = np.uint8, np.uint16, np.float32


def _memory(dev):
    return {ptr: bytes(b) for ptr, b in dev.blocks.items()}


def _adamw_keys(params, bits, value=1):
    out = {"t": np.int64(7)}
    for n, p in params.items():
        R, kind = p.size // 64, F32 if bits == 32 else U8
        out.update({f"{n}/p32": np.full((R, 64), value, F32), f"{n}/m": np.full((R, 64), value, kind), f"{n}/v": np.full((R, 64), value, kind),
                    f"{n}/p16": np.full((R, 64), value, U16)})
        if bits == 8:
            out.update({f"{n}/ms": np.full(R, value, U8), f"{n}/vs": np.full(R, value, U8)})
    return out


def _but(d, key, value=None):
    out = {k: v for k, v in d.items() if k != key}
    if value is not None:
        out[key] = value
    return out


PARAMS = {"a": np.zeros((3, 64), F32), "b_norm": np.zeros(128, F32)}


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw(fake_device, bits):
    from ancora_cutile_amd import AdamW
    opt, good = AdamW(PARAMS, state_bits=bits), _adamw_keys(PARAMS, bits)
    opt.t = 3
    before = _memory(fake_device)
    bad = [_adamw_keys(PARAMS, 40 - bits), _but(good, "t"), _but(good, "b_norm/p16"), _but(good, "b_norm/v", np.zeros((2, 64), np.float64)),
           _but(good, "b_norm/m", good["a/m"]), {}]
    if bits == 8:
        bad += [_but(good, "b_norm/vs"), _but(good, "a/ms"), _but(good, "b_norm/ms", np.zeros(3, U8))]
    for sd in bad:
        with pytest.raises(ValueError, match="AdamW.load_state_dict"):
            opt.load_state_dict(sd)
        assert _memory(fake_device) == before and opt.t == 3
    opt.load_state_dict(good)
    assert opt.t == 7
    for n, s in opt.st.items():
        for k in ("p32", "m", "v", "p16") + (("ms", "vs") if bits == 8 else ()):
            assert bytes(fake_device.at(s[k].ptr, s[k].nbytes)) == good[f"{n}/{k}"].tobytes(), (n, k)


def test_hybrid(fake_device):
    from ancora_cutile_amd import HybridOptimizer
    p = {"q_proj": np.zeros((128, 256), F32), "o_proj": np.zeros((256, 128), F32), "w_norm": np.zeros(64, F32)}
    opt = HybridOptimizer(p, adamw_kw=dict(state_bits=8))
    opt.adamw.t = opt.muon.engine.t = 5
    good = {"muon/t": np.int64(9)}
    for n in opt.muon_names:
        s = opt.muon.st[n]
        good.update({f"muon/{n}/{k}": np.full(s[k].shape, 2, s[k].dtype) for k in ("p32", "buf", "p16")})
    good.update({f"adamw/{k}": v for k, v in _adamw_keys({"w_norm": p["w_norm"]}, 8, 2).items()})
    before = _memory(fake_device)
    wide = {f"adamw/{k}": v for k, v in _adamw_keys({"w_norm": p["w_norm"]}, 32).items()}
    for sd in ({**{k: v for k, v in good.items() if k.startswith("muon/")}, **wide}, _but(good, "adamw/w_norm/vs"), _but(good, "adamw/t"), _but(good, "muon/t"),
               _but(good, "muon/o_proj/p16"), _but(good, "muon/o_proj/buf", np.zeros((2, 2), F32)), _but(good, "muon/o_proj/p32", np.zeros((256, 128)))):
        with pytest.raises(ValueError, match="load_state_dict"):
            opt.load_state_dict(sd)
        assert _memory(fake_device) == before and opt.adamw.t == opt.muon.engine.t == 5
    opt.load_state_dict(good)
    assert opt.adamw.t == 7 and opt.muon.engine.t == 9
    s = opt.muon.st["o_proj"]["buf"]
    assert bytes(fake_device.at(s.ptr, s.nbytes)) == good["muon/o_proj/buf"].tobytes()


@pytest.mark.parametrize("bits", [8, 32])
def test_fresh_state_is_in_place_for_every_stream(fake_device, bits):
    """The zeros of a new optimizer are filled in on the null stream; a checkpoint may be loaded on one that does not wait for it. Every constructor ends with the
    wait, behind its last fill."""
    from ancora_cutile_amd import AdamW, HybridOptimizer, Muon
    for make in (lambda: AdamW(PARAMS, state_bits=bits), lambda: Muon({"q": np.zeros((128, 256), F32)}),
                 lambda: HybridOptimizer({"q": np.zeros((128, 256), F32), "w_norm": np.zeros(64, F32)}, adamw_kw=dict(state_bits=bits))):
        before = len(fake_device.log)
        make()
        log = fake_device.log[before:]
        fills = [i for i, (n, _) in enumerate(log) if n == "anc_fill_u32"]
        waits = [i for i, (n, a) in enumerate(log) if n == "anc_stream_sync" and a == (0,)]
        assert fills and waits and waits[-1] > fills[-1]
