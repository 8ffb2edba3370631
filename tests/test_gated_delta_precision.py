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
