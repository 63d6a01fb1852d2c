"""GPU tests of the head's training losses against the definition in float64.

Tolerances are bounds, derived before the first run, not fitted. u = 2^-24 (half a step of f32).

Logits. f32 operands are fp16 pairs (2^-22 relative, both operands: 8 u; the dropped product of the
low parts: 4 u) and a logit is at most 24 accumulations that may each round toward zero (2 u): with
A = sum_k |x_k w_k| + |bias| (over T), |dz| <= 64 u A. A probability 2^(z - lse) is then off by
2 * 64 u A relative (its logit and the lse), and 16 u for the exponential, the products around it
and the sum's rounding.
Gradients. dz = f (p - q) enters a product whose operands are off by 12 u relative, accumulated over
8 steps of 3 products a tile (48 u) and the tiles (u each): elementwise
  |d da| <= sum_j f p_j |w_j| (128 u A + (80 + tiles) u) + sum_i f q_i |w_ci| (80 + tiles) u,
likewise for dw with the roles exchanged. An fp16 pair cannot follow a value below 2^-38 of its
tile's largest: 2^-38 of the largest f times sum_r |x_r| (the largest |w| row sum) beside it.
bf16: operands exact; p (and p - q) is rounded once, 2^-8 relative at most, and so is the output.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
BF = 2.0 ** -8


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


def cuda(x, dtype=torch.float32):
    return torch.as_tensor(x, device="cuda").to(dtype)


def make(rows, k, n, seed, n_top=0, scale=1.0, ignored=0.2):
    """Features, weight, bias, targets or teacher entries, row weights: values with confident rows,
    labels that favour class 0, a share of ignored rows, absent entries and repeated classes."""
    g = np.random.default_rng(seed)
    w = (0.3 * scale / np.sqrt(k) * g.standard_normal((n, k))).astype(np.float32)
    b = (0.1 * g.standard_normal(n)).astype(np.float32)
    t = g.integers(0, n, rows)
    t[g.random(rows) < 0.5] = 0
    x = g.standard_normal((rows, k)).astype(np.float32)
    x += (g.random(rows) * 10 / np.maximum((w[t] ** 2).sum(1), 0.05))[:, None].astype(np.float32) * w[t]
    keep = g.random(rows) >= ignored
    out = {"x": x, "w": w, "b": b, "g": (g.standard_normal(rows) / rows).astype(np.float32)}
    if n_top == 0:
        out["t"] = np.where(keep, t, -1 - g.integers(0, 100, rows)).astype(np.int32)
    else:
        idx = g.integers(0, n, (rows, n_top))
        idx[:, 0] = t
        there = g.random((rows, n_top)) < 0.8
        out["idx"] = np.where(there & keep[:, None], idx, -1).astype(np.int32)
        out["logits"] = (3 * g.standard_normal((rows, n_top))).astype(np.float32)
    return out


def definition(d, temp=1.0, row_grad=True):
    """loss, lse, da, dw, db and the sums that the bounds need, in float64 on the GPU."""
    x, w, b = (cuda(d[i], torch.float64) for i in ("x", "w", "b"))
    rows, n = x.shape[0], w.shape[0]
    z = (x @ w.T + b) / temp
    lse = torch.logsumexp(z, 1)
    if "t" in d:
        idx, u = cuda(d["t"], torch.int64)[:, None], torch.zeros(rows, 1, device="cuda", dtype=torch.float64)
    else:
        idx, u = cuda(d["idx"], torch.int64), cuda(d["logits"], torch.float64) / temp
    there = idx >= 0
    valid = there.any(1)
    u = torch.where(there, u, -torch.inf)
    u[~valid] = 0
    q = torch.where(there, torch.softmax(u, 1), 0.0)
    log_q = torch.where(there, u - torch.logsumexp(u, 1, keepdim=True), 0.0)
    zc = z.gather(1, idx.clamp(min=0))
    part = torch.where(q > 0, q * (log_q - (zc - lse[:, None])), 0.0)
    f = torch.where(valid, temp * (cuda(d["g"], torch.float64) if row_grad else torch.ones_like(lse)), 0.0)
    qd = torch.zeros_like(z).scatter_add_(1, idx.clamp(min=0), q)
    p = torch.exp(z - lse[:, None])
    dz = torch.where(valid[:, None], f[:, None] * (p - qd), 0.0)
    xv = torch.where(valid[:, None], x, 0.0)
    fp, fq = f.abs()[:, None] * p, f.abs()[:, None] * qd
    fp, fq = torch.where(valid[:, None], fp, 0.0), torch.where(valid[:, None], fq, 0.0)
    A = ((xv.abs() @ w.abs().T + torch.where(torch.isfinite(b), b.abs(), 0.0)) / temp).amax(1)
    return {"valid": valid, "loss": torch.where(valid, temp ** 2 * part.sum(1), 0.0),
            "lse": torch.where(valid, lse, 0.0), "da": dz @ w, "dw": dz.T @ xv, "db": dz.sum(0),
            "A": A, "fp": fp, "fq": fq, "w": w, "x": xv, "f": f, "temp": temp,
            "abs_terms": torch.where(valid, (q * (log_q.abs() + torch.where(there, zc.abs(), 0.0) + lse.abs()[:, None])).sum(1),
                                     0.0)}


def bounds(ref, bf16):
    rows, n = ref["x"].shape[0], ref["w"].shape[0]
    A, w, x, fp, fq, f = (ref[i] for i in ("A", "w", "x", "fp", "fq", "f"))
    A = torch.where(torch.isfinite(A), A, 0.0)
    rnd = BF if bf16 else 0.0
    tr, tc = (rows + 127) // 128, (n + 127) // 128
    relp = (128 * U * A)[:, None] * fp
    e_da = (relp + (80 + tc) * U * (fp + fq) + rnd * (fp + fq)) @ w.abs()
    e_dw = (relp + (80 + tr) * U * (fp + fq) + rnd * (fp + fq)).T @ x.abs()
    e_db = (relp + (32 + tr) * U * (fp + fq)).sum(0)
    floor = 2.0 ** -38 * f.abs().amax()
    e_da = e_da + floor * w.abs().sum(0) + rnd * (ref["da"].abs() + e_da)
    e_dw = e_dw + floor * x.abs().sum(0) + rnd * (ref["dw"].abs() + e_dw)
    e_loss = ref["temp"] ** 2 * (128 * U * A + 64 * U + 64 * U * ref["abs_terms"])
    e_lse = 64 * U * A + 16 * U * (ref["lse"].abs() + 1)
    return {"da": e_da, "dw": e_dw, "db": e_db + floor, "loss": e_loss, "lse": e_lse}


def check(got, ref, bf16, names=("loss", "lse", "da", "dw", "db")):
    b = bounds(ref, bf16)
    for name in names:
        err = (got[name].double() - ref[name]).abs()
        over = (err > b[name]) | torch.isnan(got[name].double())
        assert not over.any(), (f"{name}: {int(over.sum())} of {over.numel()} beyond the bound; largest error "
                                f"{err.max():.3g}, error / bound {(err / b[name].clamp(min=1e-300)).max():.3g}")


def grad(rh, ctx, d, dtype="f32", temp=1.0, t_len=0, row_grad=True, want=("loss", "lse", "da", "dw", "db"), stream=0,
         keep=None):
    """One training step through the device entry points; returns its outputs (da as rows)."""
    td = torch.bfloat16 if dtype == "bf16" else torch.float32
    rows, k = d["x"].shape
    n = d["w"].shape[0]
    x = cuda(d["x"], td)
    if t_len:
        x = x.view(-1, t_len, k).transpose(1, 2).contiguous()
    s = {"x": x, "w": cuda(d["w"], td), "b": cuda(d["b"]), "g": cuda(d["g"])}
    nan = float("nan")
    o = {"loss": torch.full((rows,), nan, device="cuda"), "lse": torch.full((rows,), nan, device="cuda"),
         "da": torch.full_like(s["x"], nan), "dw": torch.full_like(s["w"], nan), "db": torch.full_like(s["b"], nan)}
    n_top = 0 if "t" in d else d["idx"].shape[1]
    ws = torch.empty(rh.head_grad_workspace_bytes(ctx, dtype, rows, k, n, n_top), dtype=torch.uint8, device="cuda")
    ws.fill_(0xFF)  # nothing in it may be taken for granted
    ptr = {i: (o[i].data_ptr() if i in want else 0) for i in o}
    head = (ctx, dtype, s["x"].data_ptr(), rows, k, s["w"].data_ptr(), n, s["b"].data_ptr())
    out = (s["g"].data_ptr() if row_grad else 0, ptr["loss"], ptr["lse"], ptr["da"], ptr["dw"], ptr["db"],
           ws.data_ptr(), ws.numel())
    if n_top == 0:
        s["t"] = cuda(d["t"], torch.int32)
        call = lambda st: rh.head_cross_entropy_grad_device(*head, s["t"].data_ptr(), *out, t_len=t_len, stream=st)  # noqa: E731
    else:
        s["idx"], s["logits"] = cuda(d["idx"], torch.int32), cuda(d["logits"])
        call = lambda st: rh.head_distill_grad_device(*head, s["idx"].data_ptr(), s["logits"].data_ptr(), n_top, temp,  # noqa: E731
                                                      *out, t_len=t_len, stream=st)
    if keep is not None:
        keep.update(call=call, s=s, o=o, ws=ws)
    torch.cuda.synchronize()
    call(stream)
    torch.cuda.synchronize()
    ctx.sync()
    if t_len:
        o["da"] = o["da"].transpose(1, 2).reshape(rows, k)
    return o


def rounded(d, dtype):
    """The inputs as the device holds them (bf16: rounded), for the definition."""
    if dtype == "f32":
        return d
    r = dict(d)
    for i in ("x", "w"):
        r[i] = torch.as_tensor(d[i]).bfloat16().double().numpy()
    return r


SHAPES = [(1, 8, 1), (1, 120, 300), (2, 128, 129), (3, 1, 2), (127, 80, 128), (128, 16, 127), (129, 17, 533),
          (130, 64, 1000), (257, 128, 2048), (300, 120, 18710), (1000, 33, 5), (2500, 120, 640)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", SHAPES)
def test_cross_entropy_step_matches_the_definition(rh, ctx, rows, k, n, dtype):
    d = make(rows, k, n, seed=rows * 7 + k)
    check(grad(rh, ctx, d, dtype), definition(rounded(d, dtype)), dtype == "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n,n_top,temp", [(1, 120, 300, 1, 1.0), (5, 8, 3, 7, 2.0), (129, 80, 6906, 8, 2.0),
                                                 (300, 120, 18710, 33, 4.0), (260, 128, 200, 64, 0.5),
                                                 (1000, 33, 5, 16, 3.0)])
def test_distillation_step_matches_the_definition(rh, ctx, rows, k, n, n_top, temp, dtype):
    d = make(rows, k, n, seed=rows * 5 + n_top, n_top=n_top)
    check(grad(rh, ctx, d, dtype, temp), definition(rounded(d, dtype), temp), dtype == "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lines,t_len,k,n", [(1, 120, 120, 500), (7, 37, 80, 300), (130, 1, 24, 130), (3, 250, 121, 257)])
def test_tail_layout_is_the_row_layout_transposed(rh, ctx, lines, t_len, k, n, dtype):
    d = make(lines * t_len, k, n, seed=lines)
    rows, tail = grad(rh, ctx, d, dtype), grad(rh, ctx, d, dtype, t_len=t_len)
    for i in rows:
        assert torch.equal(rows[i], tail[i]), i


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [18_944, 20_100, 4_735])
def test_full_vocabulary_batch_in_waves_and_ranges(rh, ctx, rows, dtype):
    """Several units per SM, of odd and even numbers of tiles, whole and split, on the full vocabulary."""
    d = make(rows, 120, 18710, seed=3)
    check(grad(rh, ctx, d, dtype), definition(rounded(d, dtype)), dtype == "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n", [(40_000, 300), (57_000, 129), (300, 40_000), (19_000, 6906)])
def test_many_short_units(rh, ctx, rows, n, dtype):
    """Long batches on small vocabularies and short ones on large: many units of few tiles each way."""
    d = make(rows, 24, n, seed=4, n_top=3)
    check(grad(rh, ctx, d, dtype, 2.0), definition(rounded(d, dtype), 2.0), dtype == "bf16")


@pytest.mark.parametrize("op", ["ce", "distill"])
def test_ignored_rows_reach_nothing(rh, ctx, op):
    """Padding rows hold NaN and infinity; all other results are as without them."""
    d = make(300, 120, 700, seed=11, n_top=0 if op == "ce" else 6)
    gone = (d["t"] < 0) if op == "ce" else (d["idx"] < 0).all(1)
    assert 0 < gone.sum() < 300
    clean = grad(rh, ctx, d)
    x = d["x"].copy()
    x[gone] = np.where(np.arange(120) % 2, np.nan, np.inf).astype(np.float32)
    g = d["g"].copy()
    g[gone] = np.nan
    dirty = grad(rh, ctx, dict(d, x=x, g=g))
    for i in clean:
        assert torch.equal(clean[i], dirty[i]), i
    at = torch.as_tensor(gone)
    assert not dirty["da"].cpu()[at].any() and not dirty["loss"].cpu()[at].any() and not dirty["lse"].cpu()[at].any()


@pytest.mark.parametrize("op", ["ce", "distill"])
def test_no_row_left(rh, ctx, op):
    d = make(150, 80, 300, seed=12, n_top=0 if op == "ce" else 3, ignored=2.0)
    got = grad(rh, ctx, d)
    for i in got:
        assert not got[i].any(), i


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masked_classes(rh, ctx, dtype):
    """-inf, and the lowest f32, as bias: the classes take no share, over a whole tile too."""
    d = make(200, 64, 600, seed=13, ignored=0.0)
    d["b"][128:256] = -np.inf
    d["b"][300:310] = np.finfo(np.float32).min
    d["b"][0:5] = -np.inf
    d["t"] = np.where((d["t"] < 5) | ((d["t"] >= 128) & (d["t"] < 310)), 400, d["t"]).astype(np.int32)
    got = grad(rh, ctx, d, dtype)
    ref = definition(dict(rounded(d, dtype), b=np.where(d["b"] < -1e30, -1e4, d["b"])))
    check(got, ref, dtype == "bf16", ("loss", "da", "lse", "dw", "db"))
    gone = torch.as_tensor(np.flatnonzero(d["b"] < -1e30))
    assert not got["dw"].cpu()[gone].any() and not got["db"].cpu()[gone].any()


def test_every_class_masked_is_nan_for_the_row_only_in_name(rh, ctx):
    d = make(4, 16, 40, seed=14, ignored=0.0)
    d["b"][:] = -np.inf
    got = grad(rh, ctx, d, want=("loss", "lse"))
    assert torch.isnan(got["loss"]).all() and (got["lse"] == -np.inf).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["rising", "falling", "last class", "far below"])
def test_logits_that_rise_by_hundreds(rh, ctx, order, dtype):
    """The running maximum moves late and far: sums and mean rows are brought to each new one."""
    rows, k, n = 140, 32, 900
    d = make(rows, k, n, seed=15, ignored=0.0)
    ramp = np.linspace(-300, 300, n).astype(np.float32)
    if order == "falling":
        ramp = ramp[::-1].copy()
    elif order == "last class":
        ramp = np.zeros(n, np.float32)
        ramp[-1] = 200
    elif order == "far below":
        ramp = ramp - 20_000
    d["b"] = ramp
    check(grad(rh, ctx, d, dtype), definition(rounded(d, dtype)), dtype == "bf16")


@pytest.mark.parametrize("exp", [-60, -20, 20])
def test_scales_of_operands_and_row_weights(rh, ctx, exp):
    """Features scaled by 2^exp and weights by 2^-exp, row weights over forty orders of magnitude."""
    d = make(260, 48, 400, seed=16)
    d["x"] = d["x"] * np.float32(2.0 ** exp)
    d["w"] = d["w"] * np.float32(2.0 ** -exp)
    d["g"] = d["g"] * np.float32(2.0 ** -exp)
    check(grad(rh, ctx, d), definition(d), False)


def test_bf16_offsets_by_bound_and_by_maximum(rh, ctx):
    """Blocks of rows whose logits cannot reach far around the largest bias (their offset is a bound)
    between blocks that reach hundreds (their offset follows the maximum), several units per SM."""
    d = make(20_100, 40, 700, seed=25, scale=3.0)
    far = (np.arange(20_100) // 128) % 3 == 1
    d["x"] = (d["x"] * np.where(far, 6.0, 0.05)[:, None]).astype(np.float32)
    x, w = np.linalg.norm(d["x"], axis=1), np.linalg.norm(d["w"], axis=1).max()
    assert (x[~far] * w).max() < 25 and (x[far] * w).max() > 80
    check(grad(rh, ctx, d, "bf16"), definition(rounded(d, "bf16")), True)


def test_teacher_logits_of_minus_infinity_are_absent(rh, ctx):
    d = make(150, 40, 260, seed=26, n_top=5, ignored=0.0)
    out = np.random.default_rng(27).random((150, 5)) < 0.3
    out[10:20] = True  # whole rows: ignored
    a = dict(d, logits=np.where(out, -np.inf, d["logits"]).astype(np.float32))
    b = dict(d, idx=np.where(out, -1, d["idx"]).astype(np.int32))
    qw, _ = packed(rh, ctx, d, "int8")
    for one, two in zip(rh.head_distill(d["x"], qw, a["idx"], a["logits"], 2.0),
                        rh.head_distill(d["x"], qw, b["idx"], b["logits"], 2.0)):
        assert np.array_equal(one, two) and not one[10:20].any()
    one, two = grad(rh, ctx, a, temp=2.0), grad(rh, ctx, b, temp=2.0)
    for i in one:
        assert torch.equal(one[i], two[i]), i
    assert not one["da"][10:20].any()
    check(one, definition(b, 2.0), False)


@pytest.mark.parametrize("want", [("loss",), ("lse",), ("loss", "lse", "da"), ("loss", "dw"), ("dw", "db"), ("da",)])
def test_only_what_is_asked_for(rh, ctx, want):
    d = make(200, 120, 700, seed=17)
    full = grad(rh, ctx, d)
    part = grad(rh, ctx, d, want=want)
    for i in full:
        if i in want:
            assert torch.equal(full[i], part[i]), i
        else:
            assert torch.isnan(part[i].float()).all(), i


def test_without_bias_and_row_weights(rh, ctx):
    d = make(150, 40, 260, seed=18)
    got = grad(rh, ctx, d, row_grad=False)
    check(got, definition(d, row_grad=False), False)
    loss, lse, da, dw, db = rh.head_cross_entropy_grad(d["x"], d["w"], d["t"], ctx=ctx)
    ref = definition(dict(d, b=np.zeros(260, np.float32)), row_grad=False)
    check({"loss": cuda(loss), "lse": cuda(lse), "da": cuda(da), "dw": cuda(dw), "db": cuda(db)}, ref, False)


def test_zero_rows_clear_the_sums(rh, ctx):
    dw, db = torch.ones(30, 8, device="cuda"), torch.ones(30, device="cuda")
    rh.head_cross_entropy_grad_device(ctx, "f32", 0, 0, 8, 0, 30, 0, 0, 0, 0, 0, 0, dw.data_ptr(), db.data_ptr(), 0, 0)
    torch.cuda.synchronize()
    assert not dw.any() and not db.any()
    out = rh.head_distill_grad(np.zeros((0, 8), np.float32), np.ones((30, 8), np.float32), np.zeros((0, 2), np.int32),
                               np.zeros((0, 2), np.float32), ctx=ctx)
    assert out[0].shape == (0,) and not out[3].any() and not out[4].any()


def test_unaligned_views(rh, ctx):
    """Features and weight that start 4 (f32) or 2 (bf16) bytes past any vector boundary, outputs too."""
    for dtype, td in (("f32", torch.float32), ("bf16", torch.bfloat16)):
        d = make(140, 24, 150, seed=19)
        base = grad(rh, ctx, d, dtype)
        rows, k, n = 140, 24, 150

        def odd(t):
            buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
            buf[1:] = t.reshape(-1)
            return buf[1:].view(t.shape)

        x, w = odd(cuda(d["x"], td)), odd(cuda(d["w"], td))
        b, g, t = odd(cuda(d["b"])), odd(cuda(d["g"])), odd(cuda(d["t"], torch.int32))
        o = [odd(torch.zeros(rows, device="cuda")), odd(torch.zeros(rows, device="cuda")), odd(torch.zeros_like(x)),
             odd(torch.zeros_like(w)), odd(torch.zeros_like(b))]
        ws = torch.empty(rh.head_grad_workspace_bytes(ctx, dtype, rows, k, n) + 1, dtype=torch.uint8, device="cuda")[1:]
        rh.head_cross_entropy_grad_device(ctx, dtype, x.data_ptr(), rows, k, w.data_ptr(), n, b.data_ptr(), t.data_ptr(),
                                          g.data_ptr(), *[i.data_ptr() for i in o], ws.data_ptr(), ws.numel())
        torch.cuda.synchronize()
        ctx.sync()
        for i, name in zip(o, ("loss", "lse", "da", "dw", "db")):
            assert torch.equal(i, base[name]), (dtype, name)


def test_results_repeat_bit_for_bit_on_streams_and_in_graphs(rh, ctx):
    """The same call again, on another stream, captured and replayed twice, and beside another
    replayed graph with its own workspace on a second stream."""
    d, e = make(700, 120, 3000, seed=20, n_top=9), make(500, 80, 1700, seed=21)
    kd, ke = {}, {}
    first = {i: v.clone() for i, v in grad(rh, ctx, d, temp=2.0, keep=kd).items()}
    other = {i: v.clone() for i, v in grad(rh, ctx, e, keep=ke).items()}
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    for keep, st in zip((kd, ke), streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            keep["call"](torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for keep in (kd, ke):
        for v in keep["o"].values():
            v.fill_(float("nan"))
        keep["ws"].fill_(0xFF)
    torch.cuda.synchronize()
    for _ in range(2):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    ctx.sync()
    for ref, keep in ((first, kd), (other, ke)):
        for i, v in ref.items():
            assert torch.equal(v, keep["o"][i]), i


def test_gradients_against_differences(rh, ctx):
    """Central differences of the losses (host form) along random directions of a, w and bias. The
    losses are f32: with h = 2^-7 and sums of 40 losses near 6, their rounding leaves
    40 * 6 * 16 u / h = 0.03 of the sum's derivative at most, and the third derivative's h^2 / 6
    term 1e-4 of it; the directions' derivatives are of order ten."""
    g = np.random.default_rng(22)
    for n_top in (0, 5):
        d = make(40, 24, 90, seed=23, n_top=n_top, ignored=0.1)
        step = (lambda x, w, b: rh.head_cross_entropy_grad(x, w, d["t"], b, ctx=ctx)) if n_top == 0 else (  # noqa: E731
            lambda x, w, b: rh.head_distill_grad(x, w, d["idx"], d["logits"], 2.0, b, ctx=ctx))  # noqa: E731
        x, w, b = d["x"], d["w"], d["b"]
        _, _, da, dw, db = step(x, w, b)
        h = 2.0 ** -7
        for which, grad_of in ((0, da), (1, dw), (2, db)):
            at = [x, w, b]
            v = np.sign(grad_of).astype(np.float32) * g.integers(0, 2, grad_of.shape).astype(np.float32)
            v /= np.linalg.norm(v)
            hi, lo = list(at), list(at)
            hi[which], lo[which] = at[which] + h * v, at[which] - h * v
            diff = (step(*hi)[0].astype(np.float64).sum() - step(*lo)[0].astype(np.float64).sum()) / (2 * h)
            along = float((grad_of.astype(np.float64) * v).sum())
            assert abs(diff - along) <= 0.03 + 1e-3 * abs(along), (n_top, which, diff, along)


def test_class_at_or_above_n_is_reported(rh, ctx):
    d = make(50, 24, 90, seed=24, ignored=0.0)
    ref = grad(rh, ctx, dict(d, t=np.where(np.arange(50) == 7, -1, d["t"]).astype(np.int32)))
    bad = np.where(np.arange(50) == 7, 90, d["t"]).astype(np.int32)
    keep = {}
    with pytest.raises(rh.RecHeadError) as e:
        grad(rh, ctx, dict(d, t=bad), keep=keep)
    assert e.value.code == rh.RH_ERR_INVALID_ARG and "class" in str(e.value)
    for i, v in ref.items():
        assert torch.equal(v, keep["o"][i]), i
    ctx.sync()  # reported once
    with pytest.raises(rh.RecHeadError):
        rh.head_cross_entropy_grad(d["x"], d["w"], bad, ctx=ctx)


# ------------------------------------------------------------------------------ packed heads


def packed(rh, ctx, d, form):
    if form == "f32":
        return rh.Fp32Weight.from_f32_transposed(d["w"], ctx=ctx, bias=d["b"]), d["w"].astype(np.float64)
    qw = rh.QuantizedWeight.from_f32_transposed(d["w"], ctx=ctx, bias=d["b"], compact=form == "compact")
    return qw, qw.data.astype(np.float64) * qw.scales.astype(np.float64)[:, None]


def check_score(loss, lse, ref):
    # the decode kernel's probability beside the bounds above: its bar is 1e-5 relative
    b = bounds(ref, False)
    for name, got in (("loss", loss), ("lse", lse)):
        err = (cuda(got).double().reshape(-1) - ref[name]).abs()
        t2 = ref["temp"] ** 2 if name == "loss" else 1.0
        assert not (err > b[name] + t2 * 1e-5).any(), (name, float(err.max()))


@pytest.mark.parametrize("form", ["int8", "compact", "f32"])
@pytest.mark.parametrize("rows,k,n,n_top,temp", [(1, 120, 18710, 0, 1.0), (130, 120, 18710, 0, 1.0), (300, 80, 6906, 8, 2.0),
                                                 (257, 17, 533, 0, 1.0), (40, 128, 129, 64, 0.7), (1, 8, 1, 0, 1.0),
                                                 (33, 64, 300, 5, 4.0)])
def test_score_of_a_packed_head(rh, ctx, form, rows, k, n, n_top, temp):
    d = make(rows, k, n, seed=rows + k, n_top=n_top, scale=2.0)
    qw, w = packed(rh, ctx, d, form)
    ref = definition(dict(d, w=w), temp)
    if n_top == 0:
        loss, lse = rh.head_cross_entropy(d["x"], qw, d["t"])
    else:
        loss, lse = rh.head_distill(d["x"], qw, d["idx"], d["logits"], temp)
    check_score(loss, lse, ref)
    qw.free()


def test_score_in_the_tail_layout_on_a_stream_and_in_a_graph(rh, ctx):
    d = make(6 * 50, 120, 2000, seed=31, n_top=4)
    qw, w = packed(rh, ctx, d, "int8")
    ref = definition(dict(d, w=w), 2.0)
    x = cuda(d["x"]).view(6, 50, 120).transpose(1, 2).contiguous()
    loss, lse = rh.head_distill(x.cpu().numpy(), qw, d["idx"].reshape(6, 50, 4), d["logits"].reshape(6, 50, 4), 2.0, kt=True)
    check_score(loss, lse, ref)
    idx, logits = cuda(d["idx"], torch.int32), cuda(d["logits"])
    o = torch.full((2, 300), float("nan"), device="cuda")
    ws = torch.empty(rh.head_loss_workspace_bytes(qw, 300), dtype=torch.uint8, device="cuda")
    call = lambda: rh.head_distill_device(qw, x.data_ptr(), 300, idx.data_ptr(), logits.data_ptr(), 4, 2.0,  # noqa: E731
                                          o[0].data_ptr(), o[1].data_ptr(), ws.data_ptr(), ws.numel(), t_len=50,
                                          stream=torch.cuda.current_stream().cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    o.fill_(float("nan"))
    g.replay()
    torch.cuda.synchronize()
    ctx.sync()
    assert np.array_equal(o[0].cpu().numpy(), loss.reshape(-1)) and np.array_equal(o[1].cpu().numpy(), lse.reshape(-1))
    qw.free()


def test_score_of_ignored_rows_is_zero_whatever_they_hold(rh, ctx):
    d = make(300, 120, 2000, seed=33)
    gone = d["t"] < 0
    qw, w = packed(rh, ctx, d, "int8")
    clean = rh.head_cross_entropy(d["x"], qw, d["t"])
    x = d["x"].copy()
    x[gone] = np.nan
    dirty = rh.head_cross_entropy(x, qw, d["t"])
    for a, b in zip(clean, dirty):
        assert np.array_equal(a, b) and not b[gone].any()
    qw.free()


def test_score_leaves_decoding_as_it_was(rh, ctx):
    d = make(200, 120, 3001, seed=32)
    qw, _ = packed(rh, ctx, d, "int8")
    before = rh.head_decode(d["x"], qw)
    rh.head_distill(d["x"], qw, d["t"][:, None], np.zeros((200, 1), np.float32), 3.0)
    after = rh.head_decode(d["x"], qw)
    assert np.array_equal(before[0], after[0]) and np.array_equal(before[1], after[1])
    qw.free()


# ------------------------------------------------------------------------- as they are used


def test_a_head_is_distilled_packed_and_scored(rh, ctx):
    """A teacher head's top logits, a student trained on them for a few steps by gradient descent,
    its packed int8 form scored and decoded: the parts agree with each other throughout."""
    g = np.random.default_rng(41)
    rows, k, n, top = 256, 80, 700, 8
    x = g.standard_normal((rows, k)).astype(np.float32)
    teacher = (0.3 * g.standard_normal((n, k))).astype(np.float32)
    fw = rh.Fp32Weight.from_f32_transposed(teacher, ctx=ctx)
    z = rh.matmul_transposed_b(x, fw)
    idx = np.argsort(-z, axis=1)[:, :top].astype(np.int32)
    logits = np.take_along_axis(z, idx, 1)
    w, b = (0.05 * g.standard_normal((n, k))).astype(np.float32), np.zeros(n, np.float32)
    weight = np.full(rows, 1.0 / rows, np.float32)
    for _ in range(3):
        loss, lse, da, dw, db = rh.head_distill_grad(x, w, idx, logits, 2.0, b, weight, ctx=ctx)
        ref = definition({"x": x, "w": w, "b": b, "g": weight, "idx": idx, "logits": logits}, 2.0)
        check({"loss": cuda(loss), "lse": cuda(lse), "da": cuda(da), "dw": cuda(dw), "db": cuda(db)}, ref, False)
        w, b = w - 2.0 * dw, b - 2.0 * db
    sw = rh.Fp32Weight.from_f32_transposed(w, ctx=ctx, bias=b)
    score, _ = rh.head_distill(x, sw, idx, logits, 2.0)
    again = rh.head_distill_grad(x, w, idx, logits, 2.0, b, weight, ctx=ctx)[0]
    # the same losses two ways: each within its bound of the definition (and 1e-5 for the decode)
    ref = definition({"x": x, "w": w, "b": b, "g": weight, "idx": idx, "logits": logits}, 2.0)
    err = np.abs(score.astype(np.float64) - again)
    assert (err <= 2 * bounds(ref, False)["loss"].cpu().numpy() + 4e-5).all(), err.max()
    best, prob = rh.head_decode(x, sw)
    ce, _ = rh.head_cross_entropy(x, sw, best)
    assert np.abs(ce + np.log(prob.astype(np.float64))).max() <= 1e-4
    fw.free()
    sw.free()


# --------------------------------------------------------------------------------- refusals


def test_refusals_launch_nothing(rh, ctx):
    """Every refused call names its reason, launches nothing and leaves the outputs alone."""
    d = make(12, 24, 90, seed=51, n_top=3)
    qw, _ = packed(rh, ctx, d, "int8")
    buf = torch.zeros(1 << 20, device="cuda")
    p, ws = buf.data_ptr(), buf.numel() * 4
    ce = dict(dtype="f32", a_ptr=p, rows=12, k=24, w_ptr=p, n=90, bias_ptr=p, target_ptr=p, row_grad_ptr=p, loss_ptr=p,
              lse_ptr=p, da_ptr=p, dw_ptr=p, dbias_ptr=p, workspace_ptr=p, workspace_bytes=ws)
    ds = dict(dtype="f32", a_ptr=p, rows=12, k=24, w_ptr=p, n=90, bias_ptr=p, top_idx_ptr=p, top_logits_ptr=p, n_top=3,
              temperature=1.0, row_grad_ptr=p, loss_ptr=p, lse_ptr=p, da_ptr=p, dw_ptr=p, dbias_ptr=p, workspace_ptr=p,
              workspace_bytes=ws)
    sc = dict(a_ptr=p, rows=12, target_ptr=p, loss_ptr=p, lse_ptr=p, workspace_ptr=p, workspace_bytes=ws)
    sd = dict(a_ptr=p, rows=12, top_idx_ptr=p, top_logits_ptr=p, n_top=3, temperature=1.0, loss_ptr=p, lse_ptr=p,
              workspace_ptr=p, workspace_bytes=ws)
    bad = {"inv": rh.RH_ERR_INVALID_ARG, "uns": rh.RH_ERR_UNSUPPORTED}
    both = [(dict(rows=-1), "inv"), (dict(rows=(1 << 30) + 1), "uns"), (dict(t_len=-1), "inv"), (dict(t_len=5), "inv"),
            (dict(slot=1), "inv"), (dict(slot=-1), "inv"), (dict(a_ptr=0), "inv"), (dict(workspace_ptr=0), "inv"),
            (dict(workspace_bytes=100), "inv")]
    grads = [(dict(k=129), "uns"), (dict(k=0), "inv"), (dict(n=0), "inv"), (dict(n=(1 << 17) + 1), "uns"),
             (dict(w_ptr=0), "inv"), (dict(dw_ptr=0), "inv"), (dict(dtype="f16"), "inv")]
    tops = [(dict(n_top=0), "inv"), (dict(n_top=65), "inv"), (dict(temperature=0.0), "inv"),
            (dict(temperature=-1.0), "inv"), (dict(temperature=float("nan")), "inv"),
            (dict(temperature=float("inf")), "inv"), (dict(temperature=1e-45), "inv"), (dict(top_idx_ptr=0), "inv"),
            (dict(top_logits_ptr=0), "inv")]
    calls = ([(rh.head_cross_entropy_grad_device, (ctx,), dict(ce, **c), e) for c, e in both + grads + [(dict(target_ptr=0), "inv")]]
             + [(rh.head_distill_grad_device, (ctx,), dict(ds, **c), e) for c, e in both + grads + tops]
             + [(rh.head_cross_entropy_device, (qw,), dict(sc, **c), e) for c, e in both + [(dict(target_ptr=0), "inv")]]
             + [(rh.head_distill_device, (qw,), dict(sd, **c), e) for c, e in both + tops])
    before = ctx.launch_count(0)
    for fn, head, kw, code in calls:
        with pytest.raises(rh.RecHeadError) as e:
            fn(*head, **kw)
        assert e.value.code == bad[code], (fn.__name__, kw, str(e.value))
    for args in (("f32", -1, 24, 90), ("f32", 12, 129, 90), ("bf16", 12, 24, 0), ("f32", 12, 24, 90, 65)):
        with pytest.raises(rh.RecHeadError):
            rh.head_grad_workspace_bytes(ctx, *args)
    with pytest.raises(rh.RecHeadError):
        rh.head_loss_workspace_bytes(qw, -1)
    torch.cuda.synchronize()
    ctx.sync()
    assert ctx.launch_count(0) == before and not buf.any()
    qw.free()


@pytest.mark.parametrize("rows,k,n,n_top,t_len", [(1, 120, 18_710, 0, 0), (3, 80, 6906, 0, 3), (5, 61, 724, 13, 0),
                                                  (8, 120, 18_710, 17, 0), (126, 128, 300, 3, 42), (129, 122, 620, 0, 0),
                                                  (1000, 33, 129, 5, 8), (1024, 120, 2500, 0, 0)])
def test_bf16_weight_gradient_of_few_rows(rh, ctx, rows, k, n, n_top, t_len):
    """Up to 1,024 rows p - q is in two bf16 parts: hi leaves 2^-8 of a value, lo 2^-8 of that, so an
    operand is 2^-16 off and dw has its own rounding (2^-8) and little beside it."""
    d = make(rows, k, n, seed=rows + k, n_top=n_top)
    d = rounded(d, "bf16")
    temp = 2.0 if n_top else 1.0
    ref = definition(d, temp)
    got = grad(rh, ctx, d, "bf16", temp, t_len=t_len)
    check(got, ref, True)
    fpq = ref["fp"] + ref["fq"]
    e = ((128 * U * ref["A"])[:, None] * ref["fp"] + (80 + (rows + 127) // 128) * U * fpq + 2.0 ** -16 * fpq).T @ ref["x"].abs()
    e = e + 2.0 ** -38 * ref["f"].abs().amax() * ref["x"].abs().sum(0)
    err = (got["dw"].double() - ref["dw"]).abs()
    assert not (err > e + BF * (ref["dw"].abs() + e)).any()


@pytest.mark.parametrize("rows,k,n,n_top", [(2, 30, 268, 0), (14_174, 121, 87, 0), (300, 128, 1024, 0), (77, 127, 129, 9),
                                            (5000, 16, 1000, 3)])
def test_bf16_feature_gradient_over_few_classes(rh, ctx, rows, k, n, n_top):
    """Up to 1,024 classes p is in two bf16 parts, 2^-16 off, so da keeps what the mean weight leaves
    over the label's, besides its own rounding."""
    d = rounded(make(rows, k, n, seed=rows + n, n_top=n_top), "bf16")
    temp = 2.0 if n_top else 1.0
    ref = definition(d, temp)
    got = grad(rh, ctx, d, "bf16", temp)
    check(got, ref, True)
    fpq = ref["fp"] + ref["fq"]
    e = ((128 * U * ref["A"])[:, None] * ref["fp"] + (80 + (n + 127) // 128) * U * fpq + 2.0 ** -16 * fpq) @ ref["w"].abs()
    e = e + 2.0 ** -38 * ref["f"].abs().amax() * ref["w"].abs().sum(0)
    err = (got["da"].double() - ref["da"]).abs()
    assert not (err > e + BF * (ref["da"].abs() + e)).any()
