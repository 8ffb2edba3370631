"""The norms around a block (shv_hip_norm_block) at the edges of their values and layouts, against float64 torch.
Tolerances: those of test_norm_block.py, except where a test derives its own."""
import pytest

torch = pytest.importorskip("torch")

import test_norm_block as base  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 4, 8, 9, 64, 200, 300, 1030, 5000])
@pytest.mark.parametrize("eps", [1e-6, 1.2e-38, 1e-39, 1e-42])
def test_small_eps(shv, n, eps):
    """Any positive eps, subnormal ones too (2^-126 from 9 values on): rows of zeros stay zero, rows of tiny values get the
    formula's."""
    x = torch.zeros(3, n)
    x[1] = 1e-20 * (1 + torch.arange(n) % 5)
    x[2] = torch.randn(n, generator=torch.Generator().manual_seed(1))
    xg, w, h, y, dx = x.cuda(), torch.ones(n, device="cuda"), *(torch.empty(3, n, device="cuda") for _ in range(3))
    args = shv.norm_args("fp32", rows=3, n=n, x=xg.data_ptr(), post_w=w.data_ptr(), pre_w=w.data_ptr(), h=h.data_ptr(),
                         y=y.data_ptr(), eps=eps)
    print(f"[gpu] norm block eps {eps} n {n}", flush=True)
    shv.norm_block(args)
    up = torch.ones_like(xg)
    shv.norm_block_backward(args, shv.norm_grads(dh=up.data_ptr(), dx=dx.data_ptr()))
    torch.cuda.synchronize()
    e = float(torch.tensor(eps, dtype=torch.float32))   # as the call gets it
    if n > 8:
        e = max(e, 2.0 ** -126)

    def rms(v):
        return v / (v.pow(2).mean(-1, keepdim=True) + e).sqrt()

    want = rms(x.double())
    base.close(h.cpu(), want, 1e-5, 0.0, "h")
    base.close(y.cpu(), rms(want), 1e-5, 0.0, "y")
    assert (h[0] == 0).all() and (y[0] == 0).all()
    root = 1 / torch.tensor(e, dtype=torch.float64).sqrt()   # a row of zeros: dx = up / sqrt(eps)
    assert float((dx[0].cpu().double() / root - 1).abs().max()) <= 1e-5
    assert torch.isfinite(dx).all()
