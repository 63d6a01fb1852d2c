"""GPU tests of the training losses where values cancel, vanish or end: confident rows, a student near
its teacher, exact logits, non-finite rows, the largest sizes, and memory beside the buffers.

Tolerances are bounds, derived before the first run, in the terms of test_gpu_losses.py: u = 2^-24,
logits within 64 u A, so a probability within 128 u A relative. Here they follow |dz| = f |p - q|, the
gradient itself, not f (p + q): a confident row's gradient is the small difference of the two.
  * Classes that no label names: dz = f p, 128 u A relative; bf16 rounds it once, 2^-8.
  * One label: p - 1 is minus the other classes' share, 128 u A relative as well.
  * Several labels: p_i is off by 128 u A p_i, q_i by 16 u q_i (an exponential, a sum of 64, a
    quotient) and by its teacher logit's rounding (8 u A: here it lies near the student's), both by the
    subtraction's rounding.
Products and sums as there: (80 + tiles) u of the sum of the terms' sizes. f32 operands hold nothing
below 2^-38 of the largest of the 128 values they stand beside.
"""
import numpy as np
import pytest

from test_gpu_losses import check, cuda, definition, grad, make, packed, rounded

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def rh():
    import rust_ppocrv6_b200 as rh

    rh.load()
    return rh


@pytest.fixture(scope="module")
def ctx(rh):
    c = rh.Context()
    yield c
    c.close()


@pytest.mark.parametrize("form", ["int8", "compact", "f32"])
@pytest.mark.parametrize("rows", [1, 200])
def test_score_with_every_class_masked(rh, ctx, form, rows):
    d = make(rows, 40, 300, seed=14, ignored=0.0)
    d["b"][:] = -np.inf
    qw, _ = packed(rh, ctx, d, form)
    loss, lse = rh.head_cross_entropy(d["x"], qw, d["t"])
    assert np.isnan(loss).all() and (lse == -np.inf).all()
    qw.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_largest_vocabulary_and_most_entries(rh, ctx, dtype):
    n, n_top = 131_072, 64
    d = make(130, 24, n, seed=71, n_top=n_top)
    d["idx"][:, 1] = np.where(d["idx"][:, 1] >= 0, n - 1, -1)
    d = rounded(d, dtype)
    check(grad(rh, ctx, d, dtype, 2.0), definition(d, 2.0), dtype == "bf16")
    with pytest.raises(rh.RecHeadError):
        rh.head_grad_workspace_bytes(ctx, dtype, 1, 24, n + 1)


@pytest.mark.parametrize("k", [124, 125, 126, 127])
@pytest.mark.parametrize("t_len", [0, 27])
def test_bf16_with_few_spare_slots(rh, ctx, k, t_len):
    d = rounded(make(270, k, 1100, seed=k), "bf16")
    check(grad(rh, ctx, d, "bf16", t_len=t_len), definition(d), True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n,n_top,t_len", [(1, 1, 1, 0, 0), (129, 121, 131, 0, 0), (3, 120, 18710, 5, 3),
                                                  (700, 120, 300, 0, 7), (127, 33, 257, 64, 0)])
def test_nothing_is_written_outside_the_buffers(rh, ctx, rows, k, n, n_top, t_len, dtype):
    """Every output and the exact workspace between patterns that have to be there afterwards."""
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    d = make(rows, k, n, seed=rows + n, n_top=n_top)
    ref = grad(rh, ctx, d, dtype, 2.0 if n_top else 1.0, t_len=t_len)
    x = cuda(d["x"], td)
    if t_len:
        x = x.view(-1, t_len, k).transpose(1, 2).contiguous()
    w, b, g = cuda(d["w"], td), cuda(d["b"]), cuda(d["g"])
    guard, bufs = 4096, []

    def fenced(nbytes):
        buf = torch.full((nbytes + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda")
        bufs.append((buf, nbytes))
        return buf[guard:guard + nbytes]

    out = {i: fenced(t.numel() * t.element_size()) for i, t in ref.items()}
    ws = fenced(rh.head_grad_workspace_bytes(ctx, dtype, rows, k, n, n_top))
    head = (ctx, dtype, x.data_ptr(), rows, k, w.data_ptr(), n, b.data_ptr())
    tail = (g.data_ptr(), *[out[i].data_ptr() for i in ("loss", "lse", "da", "dw", "db")], ws.data_ptr(), ws.numel())
    torch.cuda.synchronize()
    if n_top == 0:
        t = cuda(d["t"], torch.int32)
        rh.head_cross_entropy_grad_device(*head, t.data_ptr(), *tail, t_len=t_len)
    else:
        idx, logits = cuda(d["idx"], torch.int32), cuda(d["logits"])
        rh.head_distill_grad_device(*head, idx.data_ptr(), logits.data_ptr(), n_top, 2.0, *tail, t_len=t_len)
    torch.cuda.synchronize()
    ctx.sync()
    for buf, nbytes in bufs:
        assert (buf[:guard] == 0xA5).all() and (buf[guard + nbytes:] == 0xA5).all()
    for i, t in ref.items():
        got = out[i].view(t.dtype)
        if i == "da" and t_len:
            got = got.view(-1, k, t_len).transpose(1, 2).reshape(rows, k)
        assert torch.equal(got.view(t.shape), t), i


@pytest.mark.parametrize("form", ["int8", "compact", "f32"])
@pytest.mark.parametrize("rows,n,n_top", [(1, 18710, 0), (257, 533, 7)])
def test_score_writes_nothing_outside_its_buffers(rh, ctx, form, rows, n, n_top):
    d = make(rows, 120, n, seed=rows, n_top=n_top)
    qw, _ = packed(rh, ctx, d, form)
    x = cuda(d["x"])
    need = rh.head_loss_workspace_bytes(qw, rows)
    sizes, guard = (4 * rows, 4 * rows, need), 4096
    bufs = [torch.full((s + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda") for s in sizes]
    o = [b[guard:guard + s].data_ptr() for b, s in zip(bufs, sizes)]
    torch.cuda.synchronize()
    if n_top == 0:
        t = cuda(d["t"], torch.int32)
        rh.head_cross_entropy_device(qw, x.data_ptr(), rows, t.data_ptr(), *o, need)
    else:
        idx, logits = cuda(d["idx"], torch.int32), cuda(d["logits"])
        rh.head_distill_device(qw, x.data_ptr(), rows, idx.data_ptr(), logits.data_ptr(), n_top, 2.0, *o, need)
    torch.cuda.synchronize()
    ctx.sync()
    for b, s in zip(bufs, sizes):
        assert (b[:guard] == 0xA5).all() and (b[guard + s:] == 0xA5).all()
    want = rh.head_cross_entropy(d["x"], qw, d["t"]) if n_top == 0 else rh.head_distill(d["x"], qw, d["idx"], d["logits"], 2.0)
    for b, i in zip(bufs, want):
        assert np.array_equal(b[guard:guard + 4 * rows].view(torch.float32).cpu().numpy(), i)
    qw.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", [(900, 121, 200), (120, 120, 700), (3000, 33, 130), (257, 80, 2000)])
def test_steps_back_to_back_in_one_workspace(rh, ctx, rows, k, n, dtype):
    """Two steps of other inputs in turn, in one workspace and without a wait between them: each finds
    what its own kernels wrote, never what the other's left at the same addresses."""
    one, two = make(rows, k, n, seed=81), make(rows, k, n, seed=82)
    ka, kb = {}, {}
    want = [{i: v.clone() for i, v in grad(rh, ctx, d, dtype, keep=keep).items()} for d, keep in ((one, ka), (two, kb))]
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    ws = torch.empty(rh.head_grad_workspace_bytes(ctx, dtype, rows, k, n), dtype=torch.uint8, device="cuda")
    runs, st = [], torch.cuda.Stream()
    torch.cuda.synchronize()
    for i in range(40):
        s = (ka, kb)[i % 2]["s"]
        o = {j: torch.empty_like(v) for j, v in want[i % 2].items()}
        runs.append(o)
        st.wait_stream(torch.cuda.current_stream())
        assert s["x"].dtype == td
        rh.head_cross_entropy_grad_device(ctx, dtype, s["x"].data_ptr(), rows, k, s["w"].data_ptr(), n, s["b"].data_ptr(),
                                          s["t"].data_ptr(), s["g"].data_ptr(),
                                          *[o[j].data_ptr() for j in ("loss", "lse", "da", "dw", "db")], ws.data_ptr(),
                                          ws.numel(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    ctx.sync()
    for i, o in enumerate(runs):
        for j, v in want[i % 2].items():
            assert torch.equal(o[j], v), (i, j)
