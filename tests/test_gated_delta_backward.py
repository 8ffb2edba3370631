"""Backward calls of the gated delta rule (shv_hip_gated_delta_backward) as training programs make them: several on one
forward call, states through a table, fused and head-major layouts.  Tolerances: those of test_gated_delta.py."""
import pytest

torch = pytest.importorskip("torch")

import test_gated_delta as base  # noqa: E402

GRADS = ("q", "k", "v", "g", "beta")


def gradients(shv, args, keep, d_o, d_state=None, stream=None, work=None):
    """One backward call with outputs, and where asked a workspace, of its own."""
    got = {n: torch.full_like(keep[n], float("nan")) for n in (*GRADS, "state")}
    if work is not None:
        args.workspace, args.workspace_bytes = work.data_ptr(), work.numel()
    shv.gated_delta_backward(args, shv.delta_grads(d_o=d_o.data_ptr(), d_state_out=None if d_state is None else d_state.data_ptr(),
                                                   d_state_in=got["state"].data_ptr(),
                                                   **{f"d_{n}": got[n].data_ptr() for n in GRADS}), stream)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("mode", base.MODES)
@pytest.mark.parametrize("lens,h,dk,dv", [([2100, 5], 2, 64, 64), ([1900], 2, 128, 96), ([70, 30], 3, 40, 24)], ids=str)
def test_saved_is_only_read(shv, mode, lens, h, dk, dv):
    """Two backward calls on one forward call, each with its workspace, one after the other and on two streams at once: each
    gives its own gradients, and what the forward call saved stays as it was."""
    s = base.make(mode, lens, h, h, dk, dv, seed=61, decay=0.005)
    assert base.in_segments(shv, s, True) == (sum(lens) > 1500)
    args, _ = base.device_args(shv, s, train=True)
    keep = args.keep
    print(f"[gpu] gated delta, two backward calls, {mode} {lens} {dk}x{dv}", flush=True)
    keep["saved"].zero_()   # what the forward call does not write stays as it was too
    shv.gated_delta(args)
    torch.cuda.synchronize()
    saved = keep["saved"].clone()
    ups = [(keep["do"], keep["dstate"]), (-2 * keep["do"].flip(2), 3 * keep["dstate"].flip(2))]
    works = [torch.empty_like(keep["work"]) for _ in ups]
    alone = [gradients(shv, args, keep, *up, work=w) for up, w in zip(ups, works)]
    torch.cuda.synchronize()
    assert torch.equal(keep["saved"], saved), "a backward call wrote into what the forward call saved"
    want, grads = base.reference(s, True, True)
    base.check_grads(s, alone[0], grads)
    other = dict(s, do=ups[1][0].cpu(), dstate=ups[1][1].cpu())
    base.check_grads(other, alone[1], base.reference(other, True, True)[1])
    streams = [torch.cuda.Stream() for _ in ups]
    for _ in range(3):
        got = []
        for up, w, stream in zip(ups, works, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append(gradients(shv, args, keep, *up, stream=stream.cuda_stream, work=w))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            for n in a:
                assert torch.equal(a[n].view(torch.uint8), b[n].view(torch.uint8)), f"gradient of {n}"


def test_backward_work_holds_the_segments(shv):
    """A workspace for the scans alone is refused where sequences are split (nothing is launched, so no GPU is needed)."""
    fields = dict(n_seqs=1, n_tokens=4096, heads_qk=2, heads=2, dim_k=64, dim_v=64, q=4096, k=4096, v=4096, g=4096, beta=4096,
                  o=4096, saved=4096, saved_bytes=1 << 40, workspace=4096)
    scans = 64 * 2 * 4 * (4 * 1024 + 4 * 1024) + 2 * 4 * (4 + 4) * 1024   # ends and dR, 1 KB a tile; a slot more per sequence
    args = shv.delta_args("bf16", workspace_bytes=scans, **fields)
    assert shv.delta_bytes(args, True).workspace > scans
    with pytest.raises(shv.ShvError, match="workspace too small"):
        shv.gated_delta_backward(args, shv.delta_grads(d_o=4096, d_q=4096, d_k=4096, d_v=4096, d_g=4096, d_beta=4096))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", base.MODES)
@pytest.mark.parametrize("lens", [[40, 70, 0, 9, 1], [40, 2000, 0, 9, 1]], ids=str)
def test_states_through_a_table(shv, mode, lens):
    """States and their gradients in pools: permuted, absent (-1, past the end); the other slots stay as they were."""
    h, dk, dv, slots = 2, 64, 48, 7
    index = [5, 0, 3, -1, 7]
    s = base.make(mode, lens, 1, h, dk, dv, seed=62, decay=0.02)
    gen = torch.Generator().manual_seed(63)
    pool, d_pool = torch.randn(slots, h, dk, dv, generator=gen), 0.3 * torch.randn(slots, h, dk, dv, generator=gen)
    for name, p in (("state", pool), ("dstate", d_pool)):
        s[name] = torch.stack([p[i] if 0 <= i < slots else torch.zeros(h, dk, dv) for i in index])
    want, grads = base.reference(s, True, True)
    dev = {n: x.cuda() for n, x in dict(pool=pool, d_pool=d_pool, out=torch.full_like(pool, 7.0),
                                        d_in=torch.full_like(pool, 9.0)).items()}
    idx = torch.tensor(index, dtype=torch.int32, device="cuda")
    args, out = base.device_args(shv, s, train=True, state_in=dev["pool"].data_ptr(), state_out=dev["out"].data_ptr(),
                                 state_index=idx.data_ptr(), n_states=slots)
    print(f"[gpu] gated delta backward with a table, {mode} {lens}", flush=True)
    shv.gated_delta(args)
    got = {n: torch.full_like(args.keep[n], float("nan")) for n in GRADS}
    shv.gated_delta_backward(args, shv.delta_grads(d_o=args.keep["do"].data_ptr(), d_state_out=dev["d_pool"].data_ptr(),
                                                   d_state_in=dev["d_in"].data_ptr(), **{f"d_{n}": got[n].data_ptr() for n in GRADS}))
    torch.cuda.synchronize()
    out.pop("state")
    base.check(s, out, want, mode)
    base.check_grads(s, got, grads, state=False)
    tol = base.TOL[mode]
    for i, slot in enumerate(index):
        if 0 <= slot < slots:
            base.close(dev["out"][slot:slot + 1].cpu(), want["state"][i:i + 1], tol, 0.0, f"state {slot}")
            base.close(dev["d_in"][slot:slot + 1].cpu(), grads["state"][i:i + 1], 3 * tol, 0.0, f"gradient of state {slot}")
    for slot in set(range(slots)) - set(index):
        assert (dev["out"][slot] == 7).all() and (dev["d_in"][slot] == 9).all()
    assert torch.equal(dev["pool"].cpu(), pool) and torch.equal(dev["d_pool"].cpu(), d_pool)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", base.MODES)
@pytest.mark.parametrize("hk,h,dk,dv,gap", [(2, 4, 64, 64, 0), (1, 2, 128, 96, 16), (2, 4, 24, 33, 1), (1, 2, 64, 64, 3)], ids=str)
@pytest.mark.parametrize("lens", [[70, 5], [1700]], ids=str)
def test_layouts(shv, mode, hk, h, dk, dv, gap, lens):
    """q, k and v as columns of one projection's rows (aligned or at odd places), g and beta of another's, o head-major: the
    gradients come out dense."""
    s = base.make(mode, lens, hk, h, dk, dv, seed=64, decay=0.01)
    total, nan = sum(lens), float("nan")
    width = 2 * hk * dk + h * dv + 3 * gap
    rows = torch.full((total, width), nan, dtype=s["q"].dtype)
    at = {"q": gap, "k": 2 * gap + hk * dk, "v": 3 * gap + 2 * hk * dk}
    for n, x in at.items():
        rows[:, x:x + s[n][0].numel()] = s[n].reshape(total, -1)
    gb = torch.full((total, 2 * h + 1), nan)
    gb[:, :h], gb[:, h + 1:] = s["g"], s["beta"]
    rows, gb = rows.cuda(), gb.cuda()
    oh = torch.full((h, total, dv + gap), nan, dtype=rows.dtype, device="cuda")
    size = rows.element_size()
    args, out = base.device_args(shv, s, train=True, o=oh.data_ptr(), o_stride=dv + gap, o_head=total * (dv + gap),
                                 g=gb.data_ptr(), g_stride=2 * h + 1, beta=gb.data_ptr() + 4 * (h + 1), beta_stride=2 * h + 1,
                                 **{n: rows.data_ptr() + size * x for n, x in at.items()},
                                 **{f"{n}_stride": width for n in at})
    print(f"[gpu] gated delta backward, columns of rows of {width}, {mode} {lens}", flush=True)
    shv.gated_delta(args)
    got = gradients(shv, args, args.keep, args.keep["do"], args.keep["dstate"])
    torch.cuda.synchronize()
    want, grads = base.reference(s, True, True)
    out["o"] = oh[:, :, :dv].transpose(0, 1)
    base.check(s, out, want, mode)
    base.check_grads(s, got, grads)
    assert torch.isnan(oh[:, :, dv:]).all(), "wrote outside its rows"
