"""A step whose gradients are refused leaves the optimizer as it was: the count of steps, the table of addresses and the next launch."""
import numpy as np
import pytest

U16, F32 = np.uint16, np.float32


@pytest.mark.parametrize("bits", [8, 32])
def test_the_next_launch_is_the_step_that_was_refused(fake_device, monkeypatch, bits):
    from ancora_cutile_amd import AdamW, DevBuf
    from ancora_cutile_amd._lib import AncoraError, api
    entry = "anc_adamw8_multi" if bits == 8 else "anc_adamw_multi"
    opt = AdamW({"a": np.zeros(192, F32), "b": np.zeros(64, F32)}, state_bits=bits)
    good = {n: DevBuf(shape=(s,), dtype=F32) for n, s in (("a", 192), ("b", 64))}
    opt.launch(good, 7)
    first, = fake_device.calls(entry)
    bad = [{**good, "b": DevBuf(shape=(128,), dtype=F32)}, {**good, "b": np.zeros(100, F32)}, {"a": good["a"]},
           {**good, "b": DevBuf(shape=(64,), dtype=np.int32)}]
    if bits == 8:
        bad.append({**good, "b": DevBuf(shape=(64,), dtype=F32, ptr=DevBuf(shape=(68,), dtype=F32).ptr + 4)})
    for grads in bad:
        with pytest.raises((ValueError, TypeError, KeyError)):
            opt.launch(grads, 7)
        assert opt.t == 1

    def fails(*args):
        raise AncoraError("refused")
    with monkeypatch.context() as m:
        m.setattr(api, entry, fails)
        with pytest.raises(AncoraError):
            opt.launch(good, 7)
    assert opt.t == 1
    opt.launch(good, 7)
    again = fake_device.calls(entry)[-1]
    assert opt.t == 2 and again[:3] == first[:3] and again[0] in fake_device.blocks
    opt.free()
