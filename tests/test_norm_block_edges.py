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


def gradient_of_x(s, n, act, scale, eps):
    """(dx, the size per row of the terms whose difference it is) in float64; the loss is sum(h dh) + sum(y dy)."""
    d = {k: v.double() for k, v in s.items()}
    x = d["x"][:, :n]
    r1 = 1 / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    p = (x * r1 * d["post_w"]).requires_grad_()
    t = p
    if "gate" in d:
        z = d["gate"][..., :n]
        t = p * {"none": z, "silu": z * torch.sigmoid(z), "sigmoid": torch.sigmoid(z)}[act]
    h = scale * t + (d["residual"][:, :n] if "residual" in d else 0)
    y = h / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt() * d["pre_w"]
    dp, = torch.autograd.grad((h * d["dh"]).sum() + (y * d["dy"]).sum(), p)
    w, xh = dp * d["post_w"], x * r1
    terms = r1 * (w.abs() + xh.abs() * (w * xh).abs().mean(-1, keepdim=True))
    # the cancellation by itself: mean over the others and eps, so that nothing is lost in float64 either
    dx = r1 * (w - xh * (w * xh).mean(-1, keepdim=True))
    if n == 1:
        dx = r1 ** 3 * w * eps   # w (1 - x^2 r1^2) r1 with 1 - x^2 r1^2 = eps r1^2
    return dx, terms.amax(-1, keepdim=True)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15])
def test_gradient_of_narrow_rows(shv, mode, n):
    """With a norm after the block, dx of a row of few values is a difference that cancels (of one value, down to eps).  Up to 8
    values it is taken in double, and held to 2e-5 of the row's largest value like any other; from 9 on to 2e-5 of its
    terms.  fp16 adds half a unit of its subnormals, 2^-25."""
    rows, scale, eps = 41, float(torch.tensor(0.7)), float(torch.tensor(base.EPS))
    for gate, act, residual in (("none", "none", False), ("rows", "silu", True), ("vector", "sigmoid", True)):
        s = base.make(mode, rows, n, True, gate, residual, True, 20 + n)
        g = {k: v.cuda() for k, v in s.items()}
        dx = torch.full((rows, n), float("nan"), dtype=g["x"].dtype, device="cuda")
        args = shv.norm_args(mode, rows=rows, n=n, act=act, x=g["x"].data_ptr(), post_w=g["post_w"].data_ptr(),
                             gate=g["gate"].data_ptr() if gate != "none" else None, gate_vector=gate == "vector",
                             residual=g["residual"].data_ptr() if residual else None, residual_fp32=1, scale=scale, eps=eps,
                             pre_w=g["pre_w"].data_ptr())
        print(f"[gpu] norm block dx {mode} n {n} gate {gate}", flush=True)
        shv.norm_block_backward(args, shv.norm_grads(dh=g["dh"].data_ptr(), dy=g["dy"].data_ptr(), dx=dx.data_ptr()))
        torch.cuda.synchronize()
        want, terms = gradient_of_x(s, n, act, scale, eps)
        top = want.abs().amax(-1, keepdim=True) if n <= 8 else terms
        assert torch.isfinite(dx).all()
        bad = (dx.cpu().double() - want).abs() - (2e-5 * top + base.ULP[mode] * want.abs() + (2.0 ** -25 if mode == "fp16" else 0))
        assert float(bad.max()) <= 0, (gate, float(bad.max()), float(want.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("mode,wide", [("fp32", True), ("fp16", False), ("bf16", True), ("bf16", False)])
@pytest.mark.parametrize("n", [5, 100, 385, 513, 1030, 2048, 4099, 5000, 8191])
def test_in_place(shv, mode, wide, n):
    """h over the residual and y over x; d_residual over dh and dx over dy: bitwise what buffers of their own get."""
    rows = 70
    s = base.make(mode, rows, n, True, "rows", True, wide, 12)
    g = {k: v.cuda() for k, v in s.items()}
    rdt = g["residual"].dtype

    def both(x, h, y, dh, dy, dx, dr):
        args = shv.norm_args(mode, rows=rows, n=n, act="silu", x=x.data_ptr(), post_w=g["post_w"].data_ptr(),
                             gate=g["gate"].data_ptr(), residual=g["residual"].data_ptr(), residual_fp32=wide, scale=0.7,
                             pre_w=g["pre_w"].data_ptr(), h=h.data_ptr(), y=y.data_ptr())
        work = torch.empty(shv.norm_bytes(args), dtype=torch.uint8, device="cuda")
        more = {k: torch.full_like(g[v], float("nan")) for k, v in (("dgate", "gate"), ("dpost_w", "post_w"), ("dpre_w", "pre_w"))}
        shv.norm_block_backward(args, shv.norm_grads(dh=dh.data_ptr(), dy=dy.data_ptr(), dx=dx.data_ptr(), dresidual=dr.data_ptr(),
                                                     workspace=work.data_ptr(), workspace_bytes=work.numel(),
                                                     **{k: t.data_ptr() for k, t in more.items()}))
        shv.norm_block(args)   # last, since it may take the place of its inputs
        torch.cuda.synchronize()
        return {"h": h, "y": y, "dx": dx, "dr": dr, **more}

    print(f"[gpu] norm block in place {mode} n {n}", flush=True)
    want = both(g["x"], *(torch.empty(rows, n, dtype=t, device="cuda") for t in (rdt, g["x"].dtype)), g["dh"], g["dy"],
                torch.empty_like(g["dy"]), torch.empty_like(g["dh"]))
    x, r, dh, dy = (g[k].clone() for k in ("x", "residual", "dh", "dy"))
    g["residual"] = r
    got = both(x, r, x, dh, dy, dy, dh)
    for k in want:
        assert torch.isfinite(want[k]).all() and torch.equal(got[k], want[k]), k
