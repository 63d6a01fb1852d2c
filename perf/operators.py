"""The recognition head's training losses: what is measured, and their plain forms.

Two operators over the projection z = x W^T + b of SVTR features onto the CTC vocabulary, both
without keeping the [rows, classes] logits:

  cross entropy   loss_r = lse_r - z[r, target_r], lse_r = log sum_j exp z[r, j]; a row whose
                  target is negative is ignored (loss 0, lse 0, no gradient).
  distillation    from a teacher's top logits: entries (class c_i, teacher logit t_i) per row, an
                  entry with a negative class is absent; q = softmax(t / T) over the row's entries,
                  p = softmax(z / T) over every class, loss_r = T^2 sum_i q_i (log q_i - log p[c_i]);
                  lse_r is of z / T; a row with no entry is ignored.

Each in two directions. "score" is the loss alone on a packed head (int8, compact int8 or FP32
weights, f32 features), what a serving program calls to rate a transcript or a student. "grad" is a
training step's loss, d features, d weight and d bias on plain f32 or bf16 tensors, given d total /
d loss_r for every row.

Sizes are those of the recognition heads (120 features on 18,710 classes; the tiny model's 80 on
6,906) at the line batches of the benchmark configurations; drawn cases spread over the whole range.
"""
import math

import torch

own = False

K, N = 120, 18710            # small recognition head
K_TINY, N_TINY = 80, 6906    # tiny recognition head
LARGEST = 122_880 * K * N    # rows * features * classes of the largest listed case


def _case(name, op, direction, rows, k, n, **more):
    case = {"name": name, "op": op, "dir": direction, "rows": rows, "k": k, "n": n, "t_len": 0, "weights": "int8",
            "dtype": "f32", "n_top": 0, "temperature": 1.0, "ignored": 0.1}
    case.update(more)
    return case


def listed():
    return [
        # one timestep rated by the served int8 head: the smallest call, all latency
        _case("ce score 1", "ce", "score", 1, K, N, ignored=0.0),
        # 64 ragged lines (4,018 timesteps) of one page rated by the FP32 head
        _case("ce score 4018 f32", "ce", "score", 4018, K, N, weights="f32"),
        # a full batch of 1,024 lines x 120 timesteps in the SVTR tail's own [lines, k, T] layout
        _case("ce score 122880 kt", "ce", "score", 122_880, K, N, t_len=120),
        # a fine-tuning step on one line
        _case("ce grad 120", "ce", "grad", 120, K, N),
        # a fine-tuning step on the 64 ragged lines of a page
        _case("ce grad 4018", "ce", "grad", 4018, K, N),
        # a training step on the full batch, f32 master tensors
        _case("ce grad 122880", "ce", "grad", 122_880, K, N),
        # the same in mixed precision, features as the SVTR tail leaves them
        _case("ce grad 122880 bf16 kt", "ce", "grad", 122_880, K, N, dtype="bf16", t_len=120),
        # the compact int8 student rated against a teacher's 8 best classes, 64 ragged lines
        _case("distill score 4018 compact", "distill", "score", 4018, K, N, weights="compact", n_top=8,
              temperature=2.0),
        # distilling into the tiny head: one line, then the full batch in mixed precision
        _case("distill grad 120 tiny", "distill", "grad", 120, K_TINY, N_TINY, n_top=8, temperature=2.0),
        _case("distill grad 122880 tiny bf16", "distill", "grad", 122_880, K_TINY, N_TINY, dtype="bf16", n_top=16,
              temperature=2.0),
        # distilling into the small head: 256 lines x 240 timesteps, f32, and in mixed precision
        _case("distill grad 61440", "distill", "grad", 61_440, K, N, n_top=16, temperature=2.0, t_len=240),
        _case("distill grad 61440 bf16", "distill", "grad", 61_440, K, N, dtype="bf16", n_top=32, temperature=4.0),
    ]


def draw(rng):
    shape = rng.random()
    if shape < 0.4:
        k, n = K, N
    elif shape < 0.6:
        k, n = K_TINY, N_TINY
    else:
        k = rng.randint(8, 128)
        n = int(round(math.exp(rng.uniform(math.log(64), math.log(24_000)))))
    op = rng.choice(["ce", "distill"])
    direction = rng.choice(["score", "grad", "grad"])
    rows = int(round(math.exp(rng.uniform(0.0, math.log(122_880)))))
    t_len = 0
    if rng.random() < 0.4 and rows > 1:
        t_len = rng.randint(1, min(rows, 240))
        rows = rows // t_len * t_len
    while rows * k * n > LARGEST:
        rows = max(1, rows // 2)
        t_len = 0
    return {"op": op, "dir": direction, "rows": rows, "k": k, "n": n, "t_len": t_len,
            "weights": rng.choice(["int8", "compact", "f32"]) if direction == "score" else "int8",
            "dtype": rng.choice(["f32", "bf16"]) if direction == "grad" else "f32",
            "n_top": rng.randint(1, 32) if op == "distill" else 0,
            "temperature": round(rng.uniform(1.0, 4.0), 2) if op == "distill" else 1.0,
            "ignored": round(rng.uniform(0.0, 0.4), 2)}


_F8 = torch.float64


def _inputs(case, seed):
    """Features, weight, bias, targets (or a teacher's top entries) and row weights on the GPU.

    Weights are N(0, 0.05^2) and biases N(0, 0.01^2), the spread of the real head. Over half of the
    rows belong to the blank (class 0), as in CTC training; a row's features are unit noise plus a
    share of its class's weight row, so that its target's logit stands 0 to 16 above the noise:
    undecided rows and confident ones."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, k, n = case["rows"], case["k"], case["n"]

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=g)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    w = 0.05 * randn(n, k)
    bias = 0.01 * randn(n)
    target = (rand(rows) * n).long().clamp_(max=n - 1)
    target[rand(rows) < 0.55] = 0
    wt = w[target]
    x = randn(rows, k) + (16 * rand(rows) / wt.square().sum(1))[:, None] * wt
    keep = rand(rows) >= case["ignored"]
    keep[0] = True
    grad = (0.5 + rand(rows)) / keep.sum()
    s = {"case": case, "w": w, "bias": bias, "row_grad": grad}
    if case["op"] == "ce":
        s["target"] = torch.where(keep, target, -1).to(torch.int32)
    else:
        top = case["n_top"]
        # distinct classes from the target onwards; lists of 1 to n_top entries, the best first
        step = max(1, n // max(top, 1))
        hop = 1 + (rand(rows, top) * step).long().clamp_(max=step - 1)
        hop[:, 0] = 0
        cls = (target[:, None] + hop.cumsum(1)) % n
        logits = 14 - 1.5 * torch.arange(top, device="cuda") + 2 * randn(rows, top)
        there = torch.arange(top, device="cuda") < 1 + (rand(rows, 1) * 2 * top).long()
        s["top_idx"] = torch.where(there & keep[:, None], cls, -1).to(torch.int32)
        s["top_logits"] = logits.float()
    if case["dtype"] == "bf16":
        x, s["w"] = x.bfloat16(), w.bfloat16()
    if case["t_len"]:
        x = x.view(-1, case["t_len"], k).transpose(1, 2).contiguous()
    s["x"] = x
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _own_state(s)
    return s


def _own_state(s):
    """What a program keeps between calls: the packed head (score), the workspace and the outputs."""
    import rust_ppocrv6_b200 as rh

    case = s["case"]
    rows, k, n = case["rows"], case["k"], case["n"]
    ctx = rh.default_context()

    def empty(like_rows, dtype=torch.float32):
        return torch.empty(like_rows, dtype=dtype, device="cuda")

    s["rh"], s["ctx"] = rh, ctx
    s["loss"], s["lse"] = empty(rows), empty(rows)
    if case["dir"] == "score":
        w_t, b = s["w"].cpu().numpy(), s["bias"].cpu().numpy()
        if case["weights"] == "f32":
            s["head"] = rh.Fp32Weight.from_f32_transposed(w_t, ctx=ctx, bias=b)
        else:
            s["head"] = rh.QuantizedWeight.from_f32_transposed(w_t, ctx=ctx, bias=b,
                                                               compact=case["weights"] == "compact")
        s["ws"] = empty(rh.head_loss_workspace_bytes(s["head"], rows), torch.uint8)
    else:
        s["dx"], s["dw"], s["db"] = torch.empty_like(s["x"]), torch.empty_like(s["w"]), torch.empty_like(s["bias"])
        s["ws"] = empty(rh.head_grad_workspace_bytes(ctx, case["dtype"], rows, k, n, case["n_top"]), torch.uint8)


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    rh, case = s["rh"], s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    x, ws = s["x"], s["ws"]
    if case["dir"] == "score":
        out = (s["loss"].data_ptr(), s["lse"].data_ptr(), ws.data_ptr(), ws.numel())
        if case["op"] == "ce":
            rh.head_cross_entropy_device(s["head"], x.data_ptr(), case["rows"], s["target"].data_ptr(), *out,
                                         t_len=case["t_len"], stream=stream)
        else:
            rh.head_distill_device(s["head"], x.data_ptr(), case["rows"], s["top_idx"].data_ptr(),
                                   s["top_logits"].data_ptr(), case["n_top"], case["temperature"], *out,
                                   t_len=case["t_len"], stream=stream)
        return s["loss"], s["lse"]
    head = (s["ctx"], case["dtype"], x.data_ptr(), case["rows"], case["k"], s["w"].data_ptr(), case["n"],
            s["bias"].data_ptr())
    out = (s["row_grad"].data_ptr(), s["loss"].data_ptr(), s["lse"].data_ptr(), s["dx"].data_ptr(),
           s["dw"].data_ptr(), s["db"].data_ptr(), ws.data_ptr(), ws.numel())
    if case["op"] == "ce":
        rh.head_cross_entropy_grad_device(*head, s["target"].data_ptr(), *out, t_len=case["t_len"], stream=stream)
    else:
        rh.head_distill_grad_device(*head, s["top_idx"].data_ptr(), s["top_logits"].data_ptr(), case["n_top"],
                                    case["temperature"], *out, t_len=case["t_len"], stream=stream)
    return s["loss"], s["lse"], s["dx"], s["dw"], s["db"]


# ------------------------------------------------------------------------------ plain forms


def _head_weight(s):
    """The weight that the packed head multiplies by: int8 codes times their class's scale."""
    w = s["w"]
    if s["case"]["dir"] == "grad" or s["case"]["weights"] == "f32":
        return w.float()
    top = w.abs().amax(1, keepdim=True)
    # (divided by a tensor: a scalar divisor may become a product with its rounded inverse)
    scale = torch.where(top > 1e-8, top / torch.full_like(top, 127), torch.ones_like(top))
    v = w * (1 / scale)
    codes = (torch.sign(v) * torch.floor(v.abs() + 0.5)).clamp(-127, 127)
    return codes * scale


def _run_plain(s):
    case = s["case"]
    rows, k, temp = case["rows"], case["k"], case["temperature"]
    x = s["x"].float()
    if case["t_len"]:
        x = x.transpose(1, 2).reshape(rows, k)
    w = _head_weight(s)
    z = x @ w.t()
    z.add_(s["bias"]).div_(temp)
    top = z.amax(1, keepdim=True)
    if case["op"] == "ce":
        cls = s["target"].long()[:, None]
        there = cls >= 0
        q = there.float()
        log_q = torch.zeros_like(q)
    else:
        cls = s["top_idx"].long()
        there = cls >= 0
        t = torch.where(there, s["top_logits"] / temp, -torch.inf)
        t = t - t.amax(1, keepdim=True).clamp(min=torch.finfo(t.dtype).min)
        e = torch.where(there, torch.exp(t), 0.0)
        total = e.sum(1, keepdim=True)
        q = e / total.clamp(min=torch.finfo(t.dtype).tiny)
        log_q = torch.where(there, t - torch.log(total), 0.0)
    cls = cls.clamp(min=0)
    z_cls = z.gather(1, cls)
    p = z.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    valid = there.any(1)
    lse = (top + torch.log(total))[:, 0]
    loss = temp * temp * (q * torch.where(there, log_q - (z_cls - lse[:, None]), 0.0)).sum(1)
    loss, lse = torch.where(valid, loss, 0.0), torch.where(valid, lse, 0.0)
    if case["dir"] == "score":
        return loss, lse
    f = torch.where(valid, temp * s["row_grad"], 0.0)[:, None]
    dz = p.mul_(f / total)
    dz.scatter_add_(1, cls, -f * q)
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    if case["t_len"]:
        dx = dx.view(-1, case["t_len"], k).transpose(1, 2).contiguous()
    return loss, lse, dx.to(s["x"].dtype), dw.to(s["w"].dtype), db


# ----------------------------------------------------------------------- the definition, 64 bits


def exact(case, seed):
    """From the definition in float64, a block of rows at a time."""
    s = _inputs(case, seed)
    rows, k, n, temp = case["rows"], case["k"], case["n"], case["temperature"]
    x = s["x"].to(_F8)
    x = x.permute(0, 2, 1).reshape(rows, k) if case["t_len"] else x
    if case["dir"] == "score" and case["weights"] != "f32":
        # the packed codes and scales are f32 arithmetic by definition; their product is exact here
        big = torch.linalg.vector_norm(s["w"], float("inf"), dim=1)
        scale = torch.where(big > 1e-8, big / torch.full_like(big, 127), torch.ones_like(big))
        v = (s["w"] * (1 / scale)[:, None]).to(_F8)
        w = torch.copysign((v.abs() + 0.5).floor(), v).clamp(-127, 127) * scale.to(_F8)[:, None]
    else:
        w = s["w"].to(_F8)
    b = s["bias"].to(_F8)
    loss, lse = torch.zeros(rows, dtype=_F8, device="cuda"), torch.zeros(rows, dtype=_F8, device="cuda")
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(b)
    block = max(1, (1 << 27) // n)
    for r0 in range(0, rows, block):
        part = slice(r0, min(rows, r0 + block))
        xs = x[part]
        log_p = torch.log_softmax((torch.addmm(b, xs, w.t())) / temp, 1)
        full = torch.logsumexp((torch.addmm(b, xs, w.t())) / temp, 1)
        goal = torch.zeros_like(log_p)  # the distribution that the row is held to
        if case["op"] == "ce":
            t = s["target"][part].long()
            valid = t >= 0
            at = valid.nonzero()[:, 0]
            goal[at, t[at]] = 1.0
            entropy = torch.zeros_like(full)
        else:
            t = s["top_idx"][part].long()
            valid = (t >= 0).any(1)
            u = (s["top_logits"][part].to(_F8) / temp).masked_fill(t < 0, -float("inf"))
            u[~valid] = 0.0
            q = torch.softmax(u, 1).masked_fill(t < 0, 0.0)
            r, c = (t >= 0).nonzero(as_tuple=True)
            goal.index_put_((r, t[r, c]), q[r, c], accumulate=True)
            entropy = torch.special.xlogy(q, q).sum(1)
        loss[part] = torch.where(valid, temp ** 2 * (entropy - torch.where(goal > 0, goal * log_p, 0.0).sum(1)), 0.0)
        lse[part] = torch.where(valid, full, 0.0)
        if case["dir"] == "grad":
            f = temp * s["row_grad"][part].to(_F8) * valid
            d = (log_p.exp() - goal) * f[:, None]
            dx[part] = d @ w
            dw += d.t() @ xs
            db += d.sum(0)
    if case["dir"] == "score":
        return loss, lse
    if case["t_len"]:
        dx = dx.reshape(-1, case["t_len"], k).permute(0, 2, 1).contiguous()
    return loss, lse, dx, dw, db


def work(case):
    """Each input read once, each output written once; one product of rows x classes x features for
    the loss and two more for its gradients."""
    rows, k, n = case["rows"], case["k"], case["n"]
    e = 2 if case["dtype"] == "bf16" else 4
    labels = 4 * rows if case["op"] == "ce" else 8 * rows * case["n_top"]
    if case["dir"] == "score":
        per_class = {"int8": k + 8, "compact": k + 8, "f32": 4 * k + 4}[case["weights"]]
        return {"bytes": 4 * rows * k + per_class * n + labels + 8 * rows, "flops": 2 * rows * n * k}
    read = e * (rows * k + n * k) + 4 * n + labels + 4 * rows
    written = 8 * rows + e * (rows * k + n * k) + 4 * n
    return {"bytes": read + written, "flops": 6 * rows * n * k}
