"""Which kernels serve a call of few tokens a sequence (shv_hip_gated_delta), on both sides of the rule: token by token up to
12 tokens, up to 32 where sequences times heads are 256 or more; and that a sequence's values do not depend on the others'
values.  Token by token takes no work memory.  Tolerances: those of test_gated_delta.py."""
import pytest

torch = pytest.importorskip("torch")

import test_gated_delta as base  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("mode", base.MODES)
@pytest.mark.parametrize("n_seqs,h,longest", [(32, 8, 12), (32, 8, 13), (32, 8, 32), (32, 8, 33), (3, 2, 12), (3, 2, 13), (5, 51, 13),
                                              (4, 64, 20)])
def test_both_sides_of_the_rule(shv, mode, n_seqs, h, longest):
    by_token = longest <= (32 if n_seqs * h >= 256 else 12)
    for packed in (True, False):
        lens = [longest] * n_seqs if not packed else [max(0, longest - i % 5 * (longest // 4)) for i in range(n_seqs)]
        s = base.make(mode, lens, h // 2 if h % 2 == 0 else h, h, 24, 40, seed=71)
        args, out = base.device_args(shv, s, offsets=packed, max_len=longest if packed else 0)
        assert (args.workspace_bytes == 0) == by_token
        print(f"[gpu] gated delta {mode} {n_seqs} sequences of up to {longest}, {h} heads, packed {packed}", flush=True)
        shv.gated_delta(args)
        torch.cuda.synchronize()
        want, _ = base.reference(s)
        base.check(s, out, want, mode)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", base.MODES)
@pytest.mark.parametrize("lens,h", [([13] * 20 + [32] * 12, 8), ([90, 33, 7, 64], 2), ([900, 1300, 20], 2)], ids=str)
def test_independent_of_other_values(shv, mode, lens, h):
    """Other values in the other sequences and heads: bitwise the same, by tokens, by chunks and in segments."""
    s = base.make(mode, lens, h, h, 64, 64, seed=72)
    longest = max(lens)
    first = base.forward(shv, s, "values", max_len=longest)
    other = base.make(mode, lens, h, h, 64, 64, seed=73)
    at = base.offsets_of(lens).tolist()
    seq, head = len(lens) - 1, 1
    for n in ("q", "k", "v", "g", "beta"):
        other[n][at[seq]:at[seq + 1], head] = s[n][at[seq]:at[seq + 1], head]
    other["state"][seq, head] = s["state"][seq, head]
    got = base.forward(shv, other, "other values", max_len=longest)
    assert torch.equal(got["o"][at[seq]:, head], first["o"][at[seq]:, head])
    assert torch.equal(got["state"][seq, head], first["state"][seq, head])
    assert not torch.equal(got["o"][:at[1]], first["o"][:at[1]])
