"""What the gated delta rule carries on its way has fp32's precision in every storage type (shv_hip_gated_delta).

Tolerances.  Inputs are exact in the kernels' bf16 parts, and what is computed from them is carried as three parts, 24 bits.
A value passes through about eight roundings of at most 2^-24 of the largest term that meets it (a state's and u's three
parts, the triangular product's dropped pairs, fp32 sums): 16 of them, 1e-6 of that term, are twice that.  A value
stored in fp16 or bf16 adds half a unit of its last place, 2^-11 or 2^-8 of it.
"""
import pytest

torch = pytest.importorskip("torch")

import test_gated_delta as base  # noqa: E402  (the recurrence in float64 and the calls' arguments)


def overwritten(mode, n, dk, dv, state):
    """Pairs of tokens with one key (a unit vector, q alike): the first writes values of 2^14 .. 2^15 with a beta that gives
    them all their bits, the second replaces them (beta 1) by values around 1.  The second's o is what is left where terms
    of 2^15 cancel; the true one is scale v."""
    s = base.make(mode, [n], 1, 1, dk, dv, seed=51, decay=0.003)
    gen = torch.Generator().manual_seed(52)
    t = torch.arange(n)
    key = torch.nn.functional.one_hot(t // 2 % dk, dk).float().unsqueeze(1)
    s["q"] = s["k"] = key.to(s["q"].dtype)
    large = (1 + torch.rand(n, 1, dv, generator=gen)) * torch.randn(n, 1, dv, generator=gen).sign() * 2.0 ** 14
    s["v"] = torch.where((t % 2 == 0)[:, None, None], large.to(s["v"].dtype), s["v"])
    s["beta"] = torch.where((t % 2 == 0)[:, None], 0.5 + 0.5 * s["beta"], torch.ones(n, 1))
    if state:
        s["state"] = 2.0 ** 14 * s["state"].sign() * (1 + torch.rand(s["state"].shape, generator=gen))
    return s


@pytest.mark.gpu
@pytest.mark.parametrize("mode", base.MODES)
@pytest.mark.parametrize("n,dk,dv", [(70, 64, 64), (70, 128, 128), (70, 40, 24), (1100, 64, 64), (12, 128, 32)])
def test_outputs_whose_terms_cancel(shv, mode, n, dk, dv):
    """Values that a key held are replaced by ones 2^-14 as large: o is good to fp32's rounding of what was replaced."""
    for state in (False, True):
        s = overwritten(mode, n, dk, dv, state)
        want, _ = base.reference(s, state)
        for max_len in (0, 1):
            got = base.forward(shv, s, f"cancelling, max_len {max_len}", state=state, max_len=max_len)["o"].cpu().double()
            second = slice(1, None, 2)
            o, w = got[second], want["o"][second]
            top = s["scale"] * 2.0 ** 15
            assert float(want["o"][::2].abs().max()) > 0.3 * top and float(w.abs().max()) < 1e-3 * top
            bad = (o - w).abs() - (1e-6 * top + base.ULP[mode] * w.abs())
            assert float(bad.max()) <= 0, (state, max_len, float((o - w).abs().max() / top))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", base.MODES)
@pytest.mark.parametrize("lens,h,dk,dv", [([70, 9], 2, 64, 64), ([130], 2, 128, 128), ([70, 9], 2, 40, 24), ([1900], 2, 64, 96)],
                         ids=str)
def test_fp32_outputs_have_fp32_precision(shv, mode, lens, h, dk, dv):
    """States, their gradients and those of g and beta are fp32 in every mode, and the inputs are exact: they are held to
    what fp32 inputs are held to (test_gated_delta.py: 1e-5, gradients 3 times that, g's 10 times)."""
    s = base.make(mode, lens, h, h, dk, dv, seed=53, decay=0.01)
    want, grads = base.reference(s, True, True)
    got = base.forward(shv, s, "states")["state"].cpu()
    base.close(got, want["state"], 1e-5, 0.0, "state")
    out, got = base.backward(shv, s)
    base.close(out["state"].cpu(), want["state"], 1e-5, 0.0, "state of a training call")
    base.close(got["state"].cpu(), grads["state"], 3e-5, 0.0, "gradient of the state")
    for n, tol in (("beta", 3e-5), ("g", 1e-4)):
        for i, (a, b) in enumerate(zip(base.by_seq(s, got[n].cpu()), base.by_seq(s, grads[n]))):
            base.close(a, b, tol, 0.0, f"gradient of {n}, sequence {i}")


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["fp32", "bf16"])   # (o passes fp16's range here)
@pytest.mark.parametrize("lens,most,dk", [([64, 3], 1.0, 64), ([150], 0.5, 40), ([1100], 0.06, 64)], ids=str)
def test_growing_states(shv, mode, lens, most, dk):
    """g above 0: right while exp of its sum over any run of tokens is finite (here up to exp(64))."""
    s = base.make(mode, lens, 1, 2, dk, 48, seed=54)
    s["g"] = most * torch.rand(s["g"].shape, generator=torch.Generator().manual_seed(55))
    if lens[0] == 64:
        s["g"][:64] = most
    assert float(s["g"].double().sum(0).max()) < 80
    want, _ = base.reference(s)
    for max_len in (0, 1):
        base.check(s, base.forward(shv, s, f"growing, max_len {max_len}", max_len=max_len), want, mode)
