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

from test_gpu_losses import BF, U, check, cuda, definition, grad, make, packed, rounded

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


def confident(rows, k, n, seed, low=-5.0, high=-1.0):
    """Targets with 1 - p spread over 10^low .. 10^high: noise on every class, and the target's own
    weight row in the share that lifts its logit to there."""
    g = np.random.default_rng(seed)
    w = (0.5 / np.sqrt(k) * g.standard_normal((n, k))).astype(np.float32)
    t = g.integers(0, n, rows)
    t[g.random(rows) < 0.5] = 0
    x = g.standard_normal((rows, k))
    b = (0.01 * g.standard_normal(n)).astype(np.float32)
    miss = 10.0 ** g.uniform(low, high, rows)
    wt = w[t].astype(np.float64)
    for _ in range(3):  # (the share moves the other logits too)
        z = x @ w.T.astype(np.float64) + b
        zt = z[np.arange(rows), t].copy()
        z[np.arange(rows), t] = -np.inf
        rest = np.log(np.exp(z - z.max(1, keepdims=True)).sum(1)) + z.max(1)
        x += ((rest + np.log((1 - miss) / miss) - zt) / (wt ** 2).sum(1))[:, None] * wt
    return {"x": x.astype(np.float32), "w": w, "b": b, "t": t.astype(np.int32),
            "g": (g.choice([-1.0, 1.0], rows) * g.uniform(0.5, 1.5, rows) / rows).astype(np.float32)}


def near_teacher(rows, k, n, n_top, seed, temp, spread=0.03):
    """A student whose best classes' logits are the teacher's but for a few percent of a unit."""
    d = confident(rows, k, n, seed, -4.0, 0.0)
    d["x"] = torch.as_tensor(d["x"]).bfloat16().float().numpy()
    d["w"] = torch.as_tensor(d["w"]).bfloat16().float().numpy()
    z = d["x"].astype(np.float64) @ d["w"].T.astype(np.float64) + d["b"]
    idx = np.argsort(-z, axis=1)[:, :n_top]
    g = np.random.default_rng(seed + 1)
    logits = np.take_along_axis(z, idx, 1) + temp * spread * g.standard_normal(idx.shape)
    del d["t"]
    return dict(d, idx=idx.astype(np.int32), logits=logits.astype(np.float32))


def value_bounds(ref, bf16, several):
    """Elementwise bounds of da, dw and db against |dz| (several: rows may have several labels)."""
    rows, n = ref["x"].shape[0], ref["w"].shape[0]
    tr, tc = (rows + 127) // 128, (n + 127) // 128
    fp, fq, A, w, x = ref["fp"], ref["fq"], ref["A"][:, None], ref["w"].abs(), ref["x"].abs()
    dz = (fp - fq).abs()
    lab = fq > 0
    own = 128 * U * A * dz
    if several:
        own = own + torch.where(lab, 128 * U * A * fp + 16 * U * (fp + fq) + 8 * U * A * fq, 0.0)
    rnd = BF if bf16 else 0.0
    e_da = (own + (80 + tc) * U * dz + rnd * torch.where(lab, 0.0, dz)) @ w
    e_dw = (own + (80 + tr) * U * dz + rnd * dz).T @ x
    e_db = (own + (32 + tr) * U * dz).sum(0)
    if not bf16:
        e_da = e_da + 2.0 ** -38 * torch.where(lab, 0.0, fp).amax(1, keepdim=True) * w.sum(0)
        top = torch.cat([t.amax().expand(t.shape[0], 1) for t in dz.split(128)])
        e_dw = e_dw + 2.0 ** -38 * (top * x).sum(0)
    return {"da": e_da + rnd * (ref["da"].abs() + e_da), "dw": e_dw + rnd * (ref["dw"].abs() + e_dw), "db": e_db}


def check_values(got, ref, bf16, several):
    for name, bound in value_bounds(ref, bf16, several).items():
        err = (got[name].double() - ref[name]).abs()
        over = (err > bound) | torch.isnan(got[name].double())
        assert not over.any(), (f"{name}: {int(over.sum())} of {over.numel()} beyond the bound, error / bound "
                                f"{(err / bound.clamp(min=1e-300)).max():.3g}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n,t_len", [(384, 120, 18710, 0), (130, 80, 6906, 65), (1, 120, 18710, 0),
                                            (1300, 120, 1500, 0), (200, 128, 300, 0), (60, 17, 129, 20)])
def test_gradients_of_confident_rows(rh, ctx, rows, k, n, t_len, dtype):
    """p of the target from 0.9 to 0.99999: a trained head's rows."""
    d = rounded(confident(rows, k, n, seed=rows + k), dtype)
    ref = definition(d)
    got = grad(rh, ctx, d, dtype, t_len=t_len)
    check_values(got, ref, dtype == "bf16", False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n,n_top,temp", [(256, 120, 18710, 8, 2.0), (256, 80, 6906, 32, 1.0), (1, 120, 700, 4, 1.0),
                                                 (1200, 120, 2000, 3, 2.0), (40, 64, 129, 64, 4.0)])
def test_gradients_of_a_student_near_its_teacher(rh, ctx, rows, k, n, n_top, temp, dtype):
    d = near_teacher(rows, k, n, n_top, seed=rows + n, temp=temp)
    ref = definition(d, temp)
    check_values(grad(rh, ctx, d, dtype, temp), ref, dtype == "bf16", True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [300, 18710])
def test_losses_near_zero_keep_their_digits(rh, ctx, n, dtype):
    """The loss of a confident row is what the other classes leave, down to 1 - p = 1e-9: within 128 u A
    and (112 + tiles) u of itself (the sum over the tiles, the logarithm), and never negative."""
    d = rounded(confident(200, 120, n, seed=5, low=-9.0, high=-1.0), dtype)
    ref = definition(d)
    p = ref["fq"] > 0
    miss = torch.where(p, 0.0, ref["fp"] / ref["f"].abs()[:, None]).sum(1)
    want = torch.log1p(miss / (1 - miss))
    loss = grad(rh, ctx, d, dtype, want=("loss", "lse"))["loss"].double()
    err = (loss - want).abs()
    assert (loss >= 0).all() and not (err > want * (128 * U * ref["A"] + (112 + (n + 127) // 128) * U)).any(), float((err / want).max())


def exact_logits(rh, ctx, dtype):
    """Rows of one feature: every product is exact and each of n classes has the row's z as its logit.
    Returns z, n and the step's lse and loss."""
    k, n = 120, 700
    z = np.array([1, 3, 40, 96, 376, 1000, 1504, 3008, -3008, 12032], np.float64)
    x, w = np.zeros((z.size, k), np.float32), np.zeros((n, k), np.float32)
    x[:, 3], w[:, 3] = z / 8, 8.0
    d = {"x": x, "w": w, "b": np.zeros(n, np.float32), "t": np.full(z.size, 5, np.int32), "g": np.ones(z.size, np.float32)}
    got = grad(rh, ctx, d, dtype)
    return z, n, got["lse"].double().cpu().numpy(), got["loss"].double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_exact_logits_give_an_exact_sum(rh, ctx, dtype):
    """lse = z + log n. Roundings on the way: z in log2 units (the factor and the product: 1.2 u |z|), the
    offset (u |z|), the sum and its logarithm (16 u of a value below 16), the way back (2.2 u |lse|)."""
    z, n, lse, _ = exact_logits(rh, ctx, dtype)
    err = np.abs(lse - (z + np.log(n)))
    assert (err <= 4.4 * U * np.abs(z) + 64 * U * np.log(n)).all(), err / (U * np.abs(z))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_exact_logits_give_an_exact_loss(rh, ctx, dtype):
    """The loss is log n whatever z is: it is formed from differences of logits, which are zero."""
    z, n, _, loss = exact_logits(rh, ctx, dtype)
    assert (np.abs(loss - np.log(n)) <= 64 * U * np.log(n)).all(), loss - np.log(n)


def test_weight_gradient_of_unnamed_classes_in_confident_tiles(rh, ctx):
    """f32, every row with 1 - p near 1e-9: the classes that no row names have gradients of 1e-13 of a row's
    weight, and keep their digits (each class row by itself, against its own size)."""
    d = confident(256, 120, 18710, seed=8, low=-9.2, high=-8.8)
    ref = definition(d)
    got = grad(rh, ctx, d)
    named = ref["fq"].sum(0) > 0
    dz = (ref["fp"] - ref["fq"]).abs()
    bound = ((128 * U * ref["A"][:, None] + 82 * U) * dz).T @ ref["x"].abs()
    top = torch.cat([t.amax().expand(t.shape[0], 1) for t in dz.split(128)])
    bound = bound + 2.0 ** -38 * (top * ref["x"].abs()).sum(0)
    err = (got["dw"].double() - ref["dw"]).abs()[~named]
    assert not (err > bound[~named]).any(), float((err / bound[~named]).max())
    size = ref["dw"][~named].norm(dim=1)
    assert ((got["dw"].double() - ref["dw"])[~named].norm(dim=1) <= 1e-3 * size).all()


@pytest.mark.parametrize("exp", [-14, 0, 17])
@pytest.mark.parametrize("what", [np.inf, -np.inf, np.nan])
def test_a_row_that_is_not_finite_keeps_to_itself(rh, ctx, what, exp):
    """f32: one infinity or NaN in a counted row; the rows beside it are as their definition."""
    d = make(200, 60, 300, seed=61, ignored=0.0)
    d["x"], d["w"] = d["x"] * np.float32(2.0 ** exp), d["w"] * np.float32(2.0 ** -exp)
    ref = definition(d)
    x = d["x"].copy()
    x[17, 5] = what
    got = grad(rh, ctx, dict(d, x=x))
    others = torch.arange(200, device="cuda") != 17
    got = {i: got[i][others] for i in ("loss", "lse", "da")}
    whole = {i: torch.zeros_like(ref[i]) for i in got}
    for i in got:
        whole[i][others] = got[i].double()
        whole[i][17] = ref[i][17]
    check(whole, ref, False, ("loss", "lse", "da"))


def test_a_bad_class_on_the_device_fails_no_other_call(rh, ctx):
    """It is the next sync's to report; calls on the same device go on."""
    d = make(50, 24, 90, seed=24, ignored=0.0)
    qw, _ = packed(rh, ctx, d, "int8")
    want = rh.head_decode(d["x"], qw)
    step = rh.head_cross_entropy_grad(d["x"], d["w"], d["t"], d["b"], ctx=ctx)
    keep = {}
    grad(rh, ctx, d, keep=keep)
    keep["s"]["t"][7] = 90
    for _ in range(2):
        keep["call"](0)
        torch.cuda.synchronize()
        got = rh.head_decode(d["x"], qw)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        again = rh.head_cross_entropy_grad(d["x"], d["w"], d["t"], d["b"], ctx=ctx)
        assert all(np.array_equal(i, j) for i, j in zip(again, step))
        with pytest.raises(rh.RecHeadError) as e:
            ctx.sync()
        assert e.value.code == rh.RH_ERR_INVALID_ARG and "class" in str(e.value)
        ctx.sync()  # reported once
    qw.free()


@pytest.mark.parametrize("form", ["int8", "f32"])
def test_score_losses_are_as_near_as_f32_arithmetic(rh, ctx, form):
    """4,000 rows with targets 0 to 16 above the noise of 18,710 classes: the losses' distance from the
    definition, as a norm, is within half again of elementary f32 arithmetic's, and 4 u for the row's sum,
    which the decode hands on as one f32 number."""
    rows, k, n = 4000, 120, 18710
    g = np.random.default_rng(92)
    w = (0.05 * g.standard_normal((n, k))).astype(np.float32)
    t = g.integers(0, n, rows)
    x = g.standard_normal((rows, k)) + (16 * g.random(rows) / (w[t] ** 2).sum(1))[:, None] * w[t]
    d = {"x": x.astype(np.float32), "w": w, "b": (0.01 * g.standard_normal(n)).astype(np.float32),
         "t": t.astype(np.int32), "g": np.ones(rows, np.float32)}
    qw, wq = packed(rh, ctx, d, form)
    loss, _ = rh.head_cross_entropy(d["x"], qw, d["t"])
    ref = definition(dict(d, w=wq))["loss"]
    z = cuda(d["x"]) @ cuda(wq).T + cuda(d["b"])
    top = z.amax(1, keepdim=True)
    total = torch.exp(z - top).sum(1)
    plain = (top[:, 0] + torch.log(total)) - z.gather(1, cuda(t, torch.int64)[:, None])[:, 0]
    off, plain_off = ((i.double() - ref).norm() / ref.norm() for i in (cuda(loss), plain))
    assert off <= 1.5 * plain_off + 4 * U, (float(off), float(plain_off))
    qw.free()


@pytest.mark.parametrize("form", ["int8", "compact", "f32"])
@pytest.mark.parametrize("rows", [1, 200, 19_000])  # the last with rows whose classes one unit has
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


def needs(call):
    """The workspace bytes that a call asks for when it is refused for want of them."""
    with pytest.raises(Exception) as e:
        call()
    return int(str(e.value).rsplit(" ", 1)[1])


def grad_needs(rh, ctx, dtype, rows, k, n, n_top):
    p = 256  # never read: refused before
    head, out = (ctx, dtype, p, rows, k, p, n, p), (p, p, p, p, p, p, p, 0)
    if n_top == 0:
        return needs(lambda: rh.head_cross_entropy_grad_device(*head, p, *out))
    return needs(lambda: rh.head_distill_grad_device(*head, p, p, n_top, 1.0, *out))


def score_needs(rh, qw, rows, n_top):
    p = 256
    if n_top == 0:
        return needs(lambda: rh.head_cross_entropy_device(qw, p, rows, p, p, p, p, 0))
    return needs(lambda: rh.head_distill_device(qw, p, rows, p, p, n_top, 1.0, p, p, p, 0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("k,n,n_top", [(120, 18710, 0), (80, 6906, 16), (128, 300, 3), (40, 131_072, 64)])
def test_a_workspace_serves_every_smaller_batch(rh, ctx, k, n, n_top, dtype):
    rows = [1, 100, 128, 129, 500, 2000, 4018, 9000, 18_943, 18_945, 25_000, 61_440, 100_000, 122_880, 128_896]
    named = [rh.head_grad_workspace_bytes(ctx, dtype, r, k, n, n_top) for r in rows]
    asked = [grad_needs(rh, ctx, dtype, r, k, n, n_top) for r in rows]
    assert named == sorted(named) and all(a <= b for a, b in zip(asked, named))
    assert all(max(asked[:i + 1]) <= named[i] for i in range(len(rows)))


@pytest.mark.parametrize("form", ["int8", "f32"])
def test_a_score_workspace_serves_every_smaller_batch(rh, ctx, form):
    qw, _ = packed(rh, ctx, make(1, 40, 18710, seed=1), form)
    rows = [1, 127, 128, 129, 500, 2000, 4018, 9000, 18_943, 18_945, 25_000, 61_440, 122_880, 128_896]
    named = [rh.head_loss_workspace_bytes(qw, r) for r in rows]
    asked = [score_needs(rh, qw, r, 0) for r in rows]
    assert named == sorted(named) and all(max(asked[:i + 1]) <= named[i] for i in range(len(rows)))
    qw.free()


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
    ws = fenced(grad_needs(rh, ctx, dtype, rows, k, n, n_top))
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
    need = score_needs(rh, qw, rows, n_top)
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
