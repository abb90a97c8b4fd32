"""What the profiler books the layer's operators under: nothing of theirs under the weight gradients, which a step has beside them."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U16, F32 = np.uint16, np.float32


@pytest.mark.parametrize("rows", [32, 320])
def test_weight_gradients_are_counted_alone(gpu, rows):
    from ancora_cutile_amd import DevBuf, DwWorkspace, NormWorkspace, ffn_down, gated_ffn, gated_ffn_dx, gated_ffn_grad, gemm_dW, rms_norm, rms_norm_grad
    H, I = 128, 256
    b = {n: DevBuf.zeros(s, U16) for n, s in dict(x=(rows, H), y=(rows, H), h=(rows, I), g=(rows, I), u=(rows, I), Wg=(H, I), Wu=(H, I), Wd=(I, H), gain=(1, H)).items()}
    r, dg, dW = DevBuf.zeros((rows,), F32), DevBuf.zeros((H,), F32), DevBuf.zeros((H, I), F32)
    ws, dws = NormWorkspace(rows, H), DwWorkspace()

    def weights():
        gemm_dW([dict(x=b["x"], dy=b["g"], dW=dW, T=rows, K=H, N=I, workspace=dws)], 0)
    weights()
    gpu.stream_sync(0)
    gpu.profile_enable(True)
    gpu.profile_read()
    weights()
    alone = gpu.profile_read()
    weights()
    rms_norm(b["x"], b["gain"], 0, y=b["y"], rstd=r)
    gated_ffn(b["y"], b["Wg"], b["Wu"], 0, b["h"], gate=b["g"], up=b["u"])
    ffn_down(b["h"], b["Wd"], 0, b["y"])
    gated_ffn_grad(b["y"], b["g"], b["u"], b["Wd"], 0, b["g"], b["u"])
    gated_ffn_dx(b["g"], b["u"], b["Wg"], b["Wu"], 0, b["y"])
    rms_norm_grad(b["y"], b["x"], b["gain"], r, 0, b["y"], dg, ws)
    got = gpu.profile_read()
    gpu.profile_enable(False)
    for kind in got:
        assert got[kind][1] - alone[kind][1] == (6 if kind == "misc" else 0), (kind, alone[kind], got[kind])
    for x in (*b.values(), r, dg, dW, ws, dws):
        x.free()
