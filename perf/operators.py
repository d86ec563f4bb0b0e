"""What is timed of three operators that a training step over categories is made of, and their plain forms:

  embedding  table lookup with a scale, and its gradient by sorted tokens;
  fp8        a dense layer in 8-bit floating point with one scale for each block of 128, and its gradients;
  adamw      an AdamW step over many tensors at once, states in 32 or in 8 bits, gradients clipped by their global norm.

``listed()`` and ``draw(rng)`` give cases, ``prepare(case, seed)`` the state a program holds before the call, ``run(state)``
one pass (plain torch where ``own`` is false, ddgani_amd's operators where it is true), ``work(case)`` the bytes and
operations a pass cannot do without and ``exact(case, seed)`` the outputs from the definitions in 64 bits.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
TINY = 2.0 ** -100           # a block whose largest magnitude is below this is stored as zeros
FP8_BLOCK = 128              # elements that share a scale: fp8 operands, along the reduction (weights: 128 x 128)
STATE_BLOCK = 256            # elements that share a scale: 8-bit optimizer states


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # serving: the eight rows of one decoding batch; a launch and a few kilobytes each
        dict(name="embed_serve", op="embed", tokens=8, vocab=32000, dim=4096, table="bf16", out="bf16", scale=64.0),
        # training: a batch of 16 sequences of 4 093 tokens, fp32 master table, 16-bit activations
        dict(name="embed_train", op="embed", tokens=65488, vocab=50021, dim=1024, table="f32", out="bf16", scale=32.0),
        # one minibatch of a table's category codes (a few hundred codes, 176 encoded columns), all in fp32
        dict(name="embed_grad_small", op="embed_grad", tokens=257, vocab=611, dim=176, dy="f32", out="f32", scale=1.0,
             pad=0.0, accumulate=False),
        # a long batch with a padded tail; word-like frequencies: the most common row owns several percent of the tokens
        dict(name="embed_grad_large", op="embed_grad", tokens=262144, vocab=128000, dim=2048, dy="bf16", out="f32",
             scale=45.25, pad=0.1, accumulate=False),
        # serving: one row through a square layer: the weights' bytes are the work
        dict(name="fp8_serve", op="fp8", rows=1, inn=4096, out=4096, x="bf16", bias=False),
        # the sampler's widening layer on a 200 000-row table (176 encoded columns, twice as many hidden)
        dict(name="fp8_sampler", op="fp8", rows=200000, inn=176, out=352, x="f32", bias=True),
        # a training batch through a wide layer: the matrix units are the work
        dict(name="fp8_train", op="fp8", rows=8192, inn=4096, out=8192, x="bf16", bias=False),
        # the gradients of the framework's minibatch of 128 rows
        dict(name="fp8_grad_small", op="fp8_grad", rows=128, inn=176, out=352, x="f32", bias=True),
        # the gradients of a ragged batch through a layer with an odd width
        dict(name="fp8_grad", op="fp8_grad", rows=4001, inn=2048, out=5000, x="bf16", bias=True),
        # the generator of a 176-column table: 15 fp32 tensors, about a quarter of a million elements: launches count
        dict(name="adamw_generator", op="adamw", net="generator", width=176, count=0, p="f32", g="f32", master=False, bits=32,
             max_norm=1.0),
        # 48 odd tensors from 1 to some 300 000 elements, 16-bit parameters, 8-bit states, no clip
        dict(name="adamw_ragged", op="adamw", net="ragged", width=300000, count=48, p="bf16", g="bf16", master=False,
             bits=8, max_norm=0.0),
        # a stack of twelve 4096-wide layers and a table: 332 million elements, fp32 masters behind bf16 parameters
        dict(name="adamw_stack", op="adamw", net="stack", width=4096, count=12, p="bf16", g="bf16", master=True, bits=8,
             max_norm=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case; a drawn case costs no more than the largest listed one of its operator."""
    op = rng.choice(["embed", "embed_grad", "fp8", "fp8_grad", "adamw"])
    dt = lambda: rng.choice(["f32", "bf16", "f16"])
    if op in ("embed", "embed_grad"):
        dim, vocab = _log_int(rng, 1, 4096), _log_int(rng, 1, 128000)
        tokens = _log_int(rng, 1, max(1, min(262144, 262144 * 2048 // dim)))
        if op == "embed":
            return dict(op=op, tokens=min(tokens, max(1, 65488 * 1024 // dim)), vocab=vocab, dim=dim, table=dt(), out=dt(),
                        scale=rng.choice([1.0, math.sqrt(dim), 0.37]))
        return dict(op=op, tokens=tokens, vocab=max(1, min(vocab, 128000 * 2048 // dim)), dim=dim, dy=dt(), out=dt(),
                    scale=rng.choice([1.0, math.sqrt(dim), 0.37]), pad=rng.choice([0.0, 0.1, 0.5]),
                    accumulate=rng.random() < 0.4)
    if op in ("fp8", "fp8_grad"):
        inn, out = _log_int(rng, 1, 8192), _log_int(rng, 1, 8192)
        most = (8192 * 4096 * 8192 if op == "fp8" else 4001 * 2048 * 5000) // (inn * out)
        rows = _log_int(rng, 1, max(1, min(200000, most, 400000000 // (inn + out))))
        return dict(op=op, rows=rows, inn=inn, out=out, x=dt(), bias=rng.random() < 0.5)
    p = dt()
    net = rng.choice(["generator", "ragged", "stack"])
    width = {"generator": _log_int(rng, 8, 512), "ragged": _log_int(rng, 1, 2000000), "stack": _log_int(rng, 64, 3000)}[net]
    return dict(op=op, net=net, width=width, count=_log_int(rng, 1, 12 if net == "stack" else 48), p=p,
                g=rng.choice(["f32", p]), master=p != "f32" and rng.random() < 0.5, bits=rng.choice([8, 32]),
                max_norm=rng.choice([0.0, 1.0, 1e6]))


def _shapes(case):
    """the tensors of an optimizer case: (shape, whether weight decay applies)"""
    w = case["width"]
    if case["net"] == "generator":
        s = []
        for a, b in ((2 * w, w), (w, 2 * w), (2 * w, w), (w, 2 * w)):
            s += [((a, b), True), ((a,), False)] + ([((a,), False), ((a,), False)] if len(s) < 12 else [])
        return s + [((7, w), True)]
    if case["net"] == "stack":
        s = [((32000, w), True)]
        for _ in range(case["count"]):
            s += [((w, w), True), ((w,), False)]
        return s
    # sizes of a low-discrepancy sequence over the logarithm, made odd: 1 ... width
    return [((1 + (int(math.exp(math.log(w) * ((i * 0.6180339887) % 1.0))) // 2) * 2,), i % 3 > 0) for i in range(case["count"])]


def _offsets(shapes):
    """where each tensor's states begin in the flat buffers (whole blocks of STATE_BLOCK), and the buffers' length"""
    offsets, total = [], 0
    for s, _ in shapes:
        offsets.append(total)
        total += -(-math.prod(s) // STATE_BLOCK) * STATE_BLOCK
    return offsets, total


# ------------------------------------------------------------------------------------------ inputs
HYPER = dict(lr=3e-4, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)
START_STEP = 10


def _ids(n, vocab, pad, gen, dev):
    """word-like token numbers: rank v drawn with probability ~ 1/(v + 2.7), ranks scattered over the table"""
    u = torch.rand(n, generator=gen, device=dev, dtype=torch.float64)
    rank = (2.7 * torch.exp(u * math.log((vocab + 2.7) / 2.7)) - 2.7).long().clamp_(0, vocab - 1)
    perm = torch.randperm(vocab, generator=gen, device=dev)
    ids = perm[rank]
    if pad:
        ids[n - int(n * pad):] = -1
    return ids


def _flat(shapes, offsets, total, dev, make):
    out = torch.zeros(total, device=dev)
    for (s, _), o in zip(shapes, offsets):
        out[o:o + math.prod(s)] = make(s).view(-1)
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s, dt=torch.float32, k=1.0: torch.randn(*s, generator=gen, device=dev).mul_(k).to(dt)
    st = dict(case=case)
    op = case["op"]
    if op == "embed":
        st["table"] = rand(case["vocab"], case["dim"], dt=TYPES[case["table"]], k=0.02)
        st["ids"] = _ids(case["tokens"], case["vocab"], 0.0, gen, dev)
    elif op == "embed_grad":
        st["ids"] = _ids(case["tokens"], case["vocab"], case["pad"], gen, dev)
        st["dy"] = rand(case["tokens"], case["dim"], dt=TYPES[case["dy"]], k=1e-2)
        st["grad"] = rand(case["vocab"], case["dim"], dt=TYPES[case["out"]], k=1e-2) if case["accumulate"] else None
    elif op in ("fp8", "fp8_grad"):
        M, K, N, dt = case["rows"], case["inn"], case["out"], TYPES[case["x"]]
        st["x"] = rand(M, K, dt=dt) * rand(K).exp_().to(dt)              # columns of different size, as activations have
        W = rand(N, K, dt=dt, k=1.0 / math.sqrt(K))
        st["bias"] = rand(N) if case["bias"] else None
        if op == "fp8_grad":
            st["dy"] = rand(M, N, dt=dt, k=1e-3)
        if own:
            from ddgani_amd import ops
            st["weight"] = ops.Fp8Weight(W)
        else:
            st["weight"] = _quant_block(W)                               # codes and scales, laid out once
    else:
        shapes = _shapes(case)
        st["offsets"], total = _offsets(shapes)
        st["params"] = [rand(*s, dt=TYPES[case["p"]], k=0.02) for s, _ in shapes]
        st["grads"] = [rand(*s, dt=TYPES[case["g"]], k=1e-3) for s, _ in shapes]
        st["decay"] = [HYPER["weight_decay"] if d else 0.0 for _, d in shapes]
        # the states after some steps, as a program resumes with them: one flat buffer each, a tensor at its offset
        state = dict(exp_avg=_flat(shapes, st["offsets"], total, dev, lambda s: rand(*s, k=1e-3)),
                     exp_avg_sq=_flat(shapes, st["offsets"], total, dev, lambda s: rand(*s, k=1e-3).square_()))
        if case["bits"] == 8:
            m, r = _blocks(state["exp_avg"]), _blocks(state["exp_avg_sq"].sqrt_())
            state = dict(exp_avg=_code(m), exp_avg_sq=_code(r), exp_avg_scale=_scale(m), exp_avg_sq_scale=_scale(r))
        if case["master"]:
            state["masters"] = torch.zeros(total, device=dev)
            for o, p in zip(st["offsets"], st["params"]):            # what a 16-bit parameter is the rounding of
                master = p.float().view(-1) * (1.0 + rand(p.numel(), k=1e-5))
                state["masters"][o:o + p.numel()] = master
                p.copy_(master.view_as(p))
        state["step"] = torch.full((1,), START_STEP, dtype=torch.int64, device=dev)
        if own:
            from ddgani_amd import ops
            st["opt"] = ops.AdamW(st["params"], st["grads"], lr=HYPER["lr"], betas=(HYPER["beta1"], HYPER["beta2"]),
                                  eps=HYPER["eps"], weight_decay=st["decay"], max_norm=case["max_norm"] or None,
                                  state_bits=case["bits"], masters=case["master"])
            st["opt"].load_state_dict(state)
        else:
            st["state"] = state
    return st


# ------------------------------------------------------------------------------------------ plain forms
def _inv(amax):
    return torch.where(amax >= TINY, E4M3_MAX / amax, torch.zeros_like(amax))


def _scale_of(amax):
    return torch.where(amax >= TINY, amax / E4M3_MAX, torch.zeros_like(amax))


def _blocks(t):
    """flat tensor in rows of STATE_BLOCK, the last one filled with zeros"""
    return torch.nn.functional.pad(t, (0, -t.numel() % STATE_BLOCK)).view(-1, STATE_BLOCK)


def _scale(b):
    return _scale_of(b.abs().amax(1))


def _code(b):
    return (b * _inv(b.abs().amax(1, keepdim=True))).to(E4M3).view(-1)


def _code_dithered(b, first, step):
    """codes of non-negative blocks, rounded up where the fraction and the element's dither number pass one: the dither
    runs over (index, step), so that the mean of the codes over steps follows the value; positive stays positive"""
    y = b * _inv(b.amax(1, keepdim=True))
    small = y < 2.0 ** -6
    bits = torch.where(small, y + 2.0 ** -6, y).view(torch.int32).to(torch.int64)
    i = first + torch.arange(b.numel(), device=b.device, dtype=torch.int64).view_as(bits)
    u = ((i * 2654435769 + step * 2246822507) & 0xFFFFFFFF) >> 12
    c = ((bits + u) >> 20) - 960 - 8 * small.long()
    c = torch.where(y > 0, c.clamp(1, 126), torch.zeros_like(c))
    return c.to(torch.uint8).view(E4M3).view(-1)


def _pow2(amax):
    """the smallest power of two that brings amax to 448 or below (1 for what is stored as zeros)"""
    frac, exp = torch.frexp(amax)
    exp = torch.where(amax >= TINY, exp - 9 + (frac > 0.875).int(), torch.zeros_like(exp))
    return ((exp + 127) << 23).view(torch.float32)


def _to_e4m3(x, dims):
    """blocks of x over dims -> codes, scales (powers of two: the division is exact)"""
    amax = x.abs().amax(dims, keepdim=True)
    scale = _pow2(amax)
    return torch.where(amax >= TINY, x / scale, torch.zeros_like(x)).to(E4M3), scale


def _dequant_rows(x):
    """[R, C] -> what its codes stand for in fp32; groups of 128 along a row"""
    R, C = x.shape
    q, s = _to_e4m3(torch.nn.functional.pad(x.float(), (0, -C % FP8_BLOCK)).view(R, -1, FP8_BLOCK), 2)
    return (q.float() * s).flatten(1)[:, :C]


def _quant_block(W):
    """[N, K] -> codes and scales of its 128 x 128 blocks"""
    N, K = W.shape
    w = torch.nn.functional.pad(W.float(), (0, -K % FP8_BLOCK, 0, -N % FP8_BLOCK))
    return *_to_e4m3(w.view(w.shape[0] // FP8_BLOCK, FP8_BLOCK, -1, FP8_BLOCK), (1, 3)), (N, K)


def _dequant_block(weight):
    q, s, (N, K) = weight
    w = q.float() * s
    return w.reshape(w.shape[0] * FP8_BLOCK, -1)[:N, :K]


def run(state):
    case = state["case"]
    return {"embed": _run_embed, "embed_grad": _run_embed_grad, "fp8": _run_fp8, "fp8_grad": _run_fp8_grad,
            "adamw": _run_adamw}[case["op"]](state, case)


def _run_embed(st, case):
    if own:
        from ddgani_amd import ops
        return ops.embedding(st["ids"], st["table"], scale=case["scale"], out_dtype=TYPES[case["out"]])
    return (st["table"][st["ids"]].float() * case["scale"]).to(TYPES[case["out"]])


def _run_embed_grad(st, case):
    if own:
        from ddgani_amd import ops
        return ops.embedding_grad(st["ids"], st["dy"], case["vocab"], scale=case["scale"], out_dtype=TYPES[case["out"]],
                                  out=st["grad"], accumulate=case["accumulate"])
    # (one more row takes the padded tokens; the most common rows are long sums: 64 bits)
    ids = torch.where(st["ids"] < 0, case["vocab"], st["ids"])
    total = torch.zeros(case["vocab"] + 1, case["dim"], dtype=torch.float64, device=ids.device)
    total.index_add_(0, ids, st["dy"].double())
    total = total[:-1] * case["scale"]
    if case["accumulate"]:
        return st["grad"].copy_((st["grad"] + total).to(TYPES[case["out"]]))
    return total.to(TYPES[case["out"]])


def _run_fp8(st, case):
    if own:
        from ddgani_amd import ops
        return ops.linear_fp8(st["x"], st["weight"], bias=st["bias"])
    y = _dequant_rows(st["x"]) @ _dequant_block(st["weight"]).t()
    if st["bias"] is not None:
        y = y + st["bias"]
    return y.to(st["x"].dtype)


def _run_fp8_grad(st, case):
    if own:
        from ddgani_amd import ops
        return ops.linear_fp8_grads(st["dy"], st["x"], st["weight"], want_bias=case["bias"])
    dx = (_dequant_rows(st["dy"]) @ _dequant_block(st["weight"])).to(st["x"].dtype)
    dw = _dequant_rows(st["dy"].t()) @ _dequant_rows(st["x"].t()).t()
    db = st["dy"].sum(0, dtype=torch.float64).float() if case["bias"] else None
    return dx, dw, db


def _run_adamw(st, case):
    if own:
        opt = st["opt"]
        norm = opt.step()
        return dict(opt.state_dict(), params=st["params"], norm=norm)
    h, b1, b2, state = HYPER, HYPER["beta1"], HYPER["beta2"], st["state"]
    norm = clip = None
    if case["max_norm"]:
        total = sum(g.double().square().sum() for g in st["grads"])
        norm = total.sqrt().float().view(1)
        clip = (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    t = state["step"].add_(1)
    step_size = (h["lr"] / (1.0 - b1 ** t.double())).float()
    root2 = (1.0 - b2 ** t.double()).sqrt().float()
    for p, grad, o, decay in zip(st["params"], st["grads"], st["offsets"], st["decay"]):
        n = p.numel()
        g = grad.float().view(-1)
        if clip is not None:
            g = g * clip
        if case["bits"] == 8:
            blocks = slice(o // STATE_BLOCK, -(-(o + n) // STATE_BLOCK))
            value = lambda key: (_blocks(state[key][o:o + n].float()) * state[key + "_scale"][blocks, None]).view(-1)[:n]
            m, r = value("exp_avg"), value("exp_avg_sq")
            v = r * r
        else:
            m, v = state["exp_avg"][o:o + n], state["exp_avg_sq"][o:o + n]
        m = m + (1.0 - b1) * (g - m)
        v = v * b2 + (1.0 - b2) * g * g
        r = v.sqrt()
        w = state["masters"][o:o + n] if case["master"] else p.float().view(-1)
        w = w * (1.0 - h["lr"] * decay) - step_size * (m / (r / root2 + h["eps"]))
        if case["bits"] == 8:
            mb, rb = _blocks(m), _blocks(r)
            state["exp_avg_scale"][blocks] = _scale(mb)
            state["exp_avg_sq_scale"][blocks] = _scale(rb)
            state["exp_avg"][o:o + n] = _code(mb)[:n]
            state["exp_avg_sq"][o:o + n] = _code_dithered(rb, o, t)[:n]
        else:
            state["exp_avg"][o:o + n] = m
            state["exp_avg_sq"][o:o + n] = v
        if case["master"]:
            state["masters"][o:o + n] = w
        p.copy_(w.view_as(p))
    return dict(state, params=st["params"], norm=norm)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "embed":
        n, d = case["tokens"], case["dim"]
        rows = _distinct(n, case["vocab"])
        return {"bytes": 8 * n + rows * d * BYTES[case["table"]] + n * d * BYTES[case["out"]], "flops": n * d}
    if op == "embed_grad":
        n, d = case["tokens"] - int(case["tokens"] * case["pad"]), case["dim"]
        out = 2 * _distinct(n, case["vocab"]) if case["accumulate"] else case["vocab"]
        return {"bytes": 8 * case["tokens"] + n * d * BYTES[case["dy"]] + int(out * d * BYTES[case["out"]]), "flops": n * d}
    if op in ("fp8", "fp8_grad"):
        M, K, N, b = case["rows"], case["inn"], case["out"], BYTES[case["x"]]
        if op == "fp8":
            return {"bytes": M * K * b + N * K + M * N * b, "flops": 2 * M * N * K}
        return {"bytes": M * K * b + N * K + M * N * b + M * K * b + 4 * N * K, "flops": 4 * M * N * K}
    n = sum(math.prod(s) for s, _ in _shapes(case))
    state = 4 * (1 + 4 / STATE_BLOCK) if case["bits"] == 8 else 16
    weight = 8 + BYTES[case["p"]] if case["master"] else 2 * BYTES[case["p"]]
    return {"bytes": int(n * (weight + BYTES[case["g"]] + state)), "flops": 16 * n}


def _distinct(n, vocab):
    """the expected number of different rows that n word-like tokens name: the sum over ranks, in geometric strides"""
    total, lo, z = 0.0, 0, math.log((vocab + 2.7) / 2.7)
    while lo < vocab:
        hi = min(vocab, max(lo + 1, int(lo * 1.02)))
        p = math.log((hi + 2.7) / (lo + 2.7)) / z / (hi - lo)
        total += (hi - lo) * -math.expm1(n * math.log1p(-min(p, 1.0 - 1e-12)))
        lo = hi
    return max(1, int(total))


# ------------------------------------------------------------------------------------------ 64 bits, from the definitions
def _round_e4m3(y):
    """the nearest e4m3 value of |y| <= 448, ties to the even code, in 64 bits: the grid's step is 2^(e - 3), and at least 2^-9"""
    step = torch.exp2(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1].double() - 4.0)
    return torch.round(y / step) * step


def _grid_exact(x, dim_sizes):
    """x [R, C] in 64 bits -> the values its codes stand for; one power-of-two scale for each block of dim_sizes"""
    R, C = x.shape
    a, b = dim_sizes
    rb, cb = -(-R // a), -(-C // b)
    z = torch.zeros(rb * a, cb * b, dtype=torch.float64, device=x.device)
    z[:R, :C] = x
    z = z.view(rb, a, cb, b)
    top = z.abs().amax((1, 3), keepdim=True)
    unit = torch.exp2(torch.ceil(torch.log2(top.clamp(min=TINY) / E4M3_MAX)))
    unit = torch.where(top > unit * E4M3_MAX, unit * 2, torch.where(top <= unit * (E4M3_MAX / 2), unit / 2, unit))
    val = torch.where(top >= TINY, _round_e4m3(z / unit) * unit, torch.zeros_like(z))
    return val.view(rb * a, cb * b)[:R, :C]


def exact(case, seed):
    global own
    saved, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = saved
    op = case["op"]
    if op == "embed":
        return torch.index_select(st["table"], 0, st["ids"]).double() * case["scale"]
    if op == "embed_grad":
        base = st["grad"].double() if case["accumulate"] else torch.zeros(case["vocab"], case["dim"], dtype=torch.float64,
                                                                           device=st["dy"].device)
        keep = (st["ids"] >= 0).nonzero().view(-1)
        for part in keep.split(65536):
            base.index_add_(0, st["ids"][part], st["dy"][part].double(), alpha=case["scale"])
        return base
    if op in ("fp8", "fp8_grad"):
        x = st["x"].double()
        q, s, (N, K) = st["weight"]
        w = (q.double() * s.double()).reshape(q.shape[0] * FP8_BLOCK, -1)[:N, :K]
        if op == "fp8":
            y = torch.mm(_grid_exact(x, (1, FP8_BLOCK)), w.t().contiguous())
            return y if st["bias"] is None else y + st["bias"].double()
        dy = st["dy"].double()
        dx = torch.mm(_grid_exact(dy, (1, FP8_BLOCK)), w.contiguous())
        dw = torch.mm(_grid_exact(dy, (FP8_BLOCK, 1)).t().contiguous(), _grid_exact(x, (FP8_BLOCK, 1)))
        return dx, dw, dy.sum(0) if case["bias"] else None
    return _exact_adamw(st, case)


def _exact_adamw(st, case):
    h, state, t, dev = HYPER, st["state"], START_STEP + 1, st["params"][0].device
    grads = [g.double().view(-1) for g in st["grads"]]
    norm, factor = None, 1.0
    if case["max_norm"]:
        norm = math.sqrt(sum(float((g * g).sum()) for g in grads))
        factor = min(1.0, case["max_norm"] / (norm + 1e-6))
    zeros = lambda n: torch.zeros(n, dtype=torch.float64, device=dev)
    out = {k: zeros(v.numel()) for k, v in state.items() if k != "step"}
    out.update(step=torch.full((1,), t, dtype=torch.int64, device=dev), params=[],
               norm=None if norm is None else torch.full((1,), norm, dtype=torch.float64, device=dev))
    for i, (g, o) in enumerate(zip(grads, st["offsets"])):
        n = g.numel()
        g = g * factor
        m, v = state["exp_avg"][o:o + n].double(), state["exp_avg_sq"][o:o + n].double()
        if case["bits"] == 8:
            first, last = o // STATE_BLOCK, -(-(o + n) // STATE_BLOCK)
            spread = lambda s: s[first:last].double().repeat_interleave(STATE_BLOCK)[:n]
            m, v = m * spread(state["exp_avg_scale"]), (v * spread(state["exp_avg_sq_scale"])) ** 2
        m = h["beta1"] * m + (1.0 - h["beta1"]) * g
        v = h["beta2"] * v + (1.0 - h["beta2"]) * g ** 2
        w = (state["masters"][o:o + n] if case["master"] else st["params"][i].view(-1)).double()
        mean, root = m / (1.0 - h["beta1"] ** t), (v / (1.0 - h["beta2"] ** t)).sqrt()
        w = w - h["lr"] * (st["decay"][i] * w + mean / (root + h["eps"]))
        out["params"].append(w.view_as(st["params"][i]))
        if case["master"]:
            out["masters"][o:o + n] = w
        if case["bits"] == 32:
            out["exp_avg"][o:o + n], out["exp_avg_sq"][o:o + n] = m, v
            continue
        for key, vals in (("exp_avg", m), ("exp_avg_sq", v.sqrt())):
            z = zeros((last - first) * STATE_BLOCK)
            z[:n] = vals
            z = z.view(-1, STATE_BLOCK)
            top = z.abs().amax(1)
            live = top >= TINY
            unit = torch.where(live, top / E4M3_MAX, torch.ones_like(top))
            y = z / unit[:, None]
            if key == "exp_avg":
                code = _round_e4m3(y)
            else:                # down to the grid, up where the fraction in 2^-20ths and the dither number pass one
                grid = torch.exp2(torch.frexp(y.clamp(min=2.0 ** -6))[1].double() - 4.0)
                low = torch.floor(y / grid)
                idx = o + torch.arange(z.numel(), device=dev, dtype=torch.int64).view_as(z)
                dither = ((idx * 2654435769 + t * 2246822507) % 2 ** 32) // 4096
                up = torch.floor((y / grid - low) * 2 ** 20) + dither >= 2 ** 20
                code = ((low + up) * grid).clamp(max=E4M3_MAX)
                code = torch.where(z > 0, code.clamp(min=2.0 ** -9), torch.zeros_like(z))
            out[key][o:o + n] = torch.where(live[:, None], code, torch.zeros_like(z)).view(-1)[:n]
            out[key + "_scale"][first:last] = torch.where(live, top / E4M3_MAX, torch.zeros_like(top))
    return out
