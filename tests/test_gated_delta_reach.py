"""How large a call of the gated delta rule may be (shv_hip_gated_delta): checked on the host, so no GPU is needed."""
import pytest

pytest.importorskip("torch")


def sizes(shv, train=False, mode="bf16", **fields):
    return shv.delta_bytes(shv.delta_args(mode, **(dict(heads_qk=1, heads=1, dim_k=64, dim_v=64) | fields)), train)


@pytest.mark.parametrize("train", [False, True])
def test_more_threads_than_a_launch_takes(shv, train):
    """2^32 threads in any of a call's launches are refused; what is just below is not."""
    def refused(**fields):
        with pytest.raises(shv.ShvError, match="too many sequences, heads or tokens for one call"):
            sizes(shv, train, **fields)

    refused(n_seqs=1, n_tokens=1 << 31, heads=4096)              # chunks times heads
    refused(n_seqs=1, n_tokens=1 << 30, heads=1)                 # 2^24 chunks of 256 threads
    assert sizes(shv, train, n_seqs=1, n_tokens=1 << 28).saved >= 0
    refused(n_seqs=1 << 20, n_tokens=1 << 26, heads=8, dim_v=256)
    refused(n_seqs=1 << 23, n_tokens=1 << 23, heads=16, dim_v=256)
    if not train:   # a token of each of many sequences: 16 threads a sequence, head and column of 8
        refused(n_seqs=1 << 24, n_tokens=1 << 24, heads=4, dim_v=256)
        assert sizes(shv, n_seqs=1 << 22, n_tokens=1 << 22, heads=8, dim_v=32) == (0, 0)


def test_the_call_itself_refuses_too(shv):
    args = shv.delta_args("bf16", n_seqs=1 << 24, n_tokens=1 << 24, heads_qk=4, heads=4, dim_k=8, dim_v=256, q=4096, k=4096,
                          v=4096, g=4096, beta=4096, o=4096)
    with pytest.raises(shv.ShvError, match="too many sequences"):
        shv.gated_delta(args)
    args.n_seqs, args.n_tokens, args.heads, args.heads_qk, args.saved, args.saved_bytes = 1, 1 << 31, 4096, 1, 4096, 1 << 62
    args.workspace, args.workspace_bytes = 4096, 1 << 62
    with pytest.raises(shv.ShvError, match="too many sequences"):
        shv.gated_delta_backward(args, shv.delta_grads(d_o=4096, d_q=4096, d_k=4096, d_v=4096, d_g=4096, d_beta=4096))
