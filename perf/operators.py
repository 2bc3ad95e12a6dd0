"""What is measured of the operators that run a quantized model: linears on
packed weights, rotary positions and the choice of the next token.

``run`` computes one pass in its plain form (elementary torch operations) or,
where ``own`` is true, through the package's public entry points:

* ``linear.packed_matmul(x, weights)``: y = x W^T with W the 1- to 8-bit codes
  of a :class:`packing.PackedLinear`, W[r, c] = (code + qmin - zero) * scale
  with the scale and zero of row r and of column c's group;
* ``rotary.apply_rotary(q, k, positions, plan)``: each pair of the first
  ``rotary_dim`` components of every head turned by position x frequency;
* ``sampling.sample_tokens(logits, u, ...)``: temperature, top-k, top-p and
  min-p, then the inverse of the remaining distribution at u.
"""

import math

import numpy as np
import torch

own = False


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # a 1024 x 1024 linear, one token: a small model's decode step, latency alone
        dict(name="linear 1 token 1024x1024", op="linear", tokens=1, m=1024, n=1024, bits=4,
             group=128, sym=False, act_order=False, dtype="bfloat16"),
        # the widest linear of a 70B block, one token: the decode step that reads most
        dict(name="linear 1 token 28672x8192", op="linear", tokens=1, m=28672, n=8192, bits=4,
             group=128, sym=False, act_order=True, dtype="bfloat16"),
        # a 7B down_proj for a handful of requests decoded together
        dict(name="linear 6 tokens 4096x11008", op="linear", tokens=6, m=4096, n=11008, bits=4,
             group=128, sym=False, act_order=True, dtype="float16"),
        # a 70B k_proj, more requests: few rows, a long sum
        dict(name="linear 17 tokens 1024x8192", op="linear", tokens=17, m=1024, n=8192, bits=4,
             group=128, sym=True, act_order=False, dtype="bfloat16"),
        # 3-bit weights in float32, as a numerics check of a packed layer runs them
        dict(name="linear 37 tokens f32 3-bit", op="linear", tokens=37, m=4096, n=4096, bits=3,
             group=128, sym=False, act_order=True, dtype="float32"),
        # a calibration or perplexity window of 2048 tokens through a 7B gate_proj
        dict(name="linear 2048 tokens 11008x4096", op="linear", tokens=2048, m=11008, n=4096,
             bits=4, group=128, sym=False, act_order=True, dtype="bfloat16"),
        # one decoded token of a 7B block: latency alone
        dict(name="rotary 1 token", op="rotary", batch=1, seq=1, heads=32, kv_heads=32,
             head_dim=128, rotary_dim=128, interleaved=False, scaling="none", factor=1.0,
             start=731, dtype="bfloat16"),
        # four windows of a 70B block with grouped heads, positions scaled by parts
        dict(name="rotary 4x2048 grouped heads", op="rotary", batch=4, seq=2048, heads=64,
             kv_heads=8, head_dim=128, rotary_dim=128, interleaved=False, scaling="yarn",
             factor=4.0, start=0, dtype="bfloat16"),
        # half of an odd-sized head, neighbouring pairs, far positions, float32
        dict(name="rotary part of head, far", op="rotary", batch=3, seq=333, heads=20, kv_heads=5,
             head_dim=96, rotary_dim=48, interleaved=True, scaling="linear", factor=8.0,
             start=1000003, dtype="float32"),
        # one request, the usual settings: latency alone
        dict(name="sample 1 x 32000", op="sample", rows=1, vocab=32000, dtype="float32",
             temperature=0.8, top_k=50, top_p=0.95, min_p=0.0, mixed=False, masked=0.0),
        # requests served together, each with its own settings, some tokens masked out
        dict(name="sample 48 x 128256 mixed", op="sample", rows=48, vocab=128256, dtype="bfloat16",
             temperature=1.0, top_k=0, top_p=0.9, min_p=0.02, mixed=True, masked=0.01),
        # a large batch drawn from the whole distribution
        dict(name="sample 256 x 128256", op="sample", rows=256, vocab=128256, dtype="float32",
             temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False, masked=0.0),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "rotary", "sample"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "linear":
        group = rng.choice([32, 64, 128, 128, 96, 256])
        n = group * max(1, _log_between(rng, 256, 16384) // group)
        m = _log_between(rng, 64, 28672)
        tokens = _log_between(rng, 1, 2048)
        while tokens * m * n > 2048 * 11008 * 4096 or m * n > 28672 * 8192:
            m, tokens = max(1, m // 2), max(1, tokens // 2)
        return dict(op=op, tokens=tokens, m=m, n=n, bits=rng.choice([2, 3, 4, 4, 4, 8]),
                    group=group, sym=rng.random() < 0.3, act_order=rng.random() < 0.6, dtype=dtype)
    if op == "rotary":
        head_dim = rng.choice([32, 64, 80, 96, 128, 128, 256])
        rotary_dim = head_dim if rng.random() < 0.6 else 2 * rng.randrange(4, head_dim // 2)
        kv_heads = rng.choice([1, 2, 4, 5, 8, 32])
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        batch, seq = _log_between(rng, 1, 16), _log_between(rng, 1, 4096)
        while batch * seq * (heads + kv_heads) * head_dim > 4 * 2048 * 72 * 128 // 2:
            batch, seq = max(1, batch // 2), max(1, seq * 2 // 3)
        scaling = rng.choice(["none", "linear", "yarn"])
        return dict(op=op, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                    rotary_dim=rotary_dim, interleaved=rng.random() < 0.4, scaling=scaling,
                    factor=1.0 if scaling == "none" else round(rng.uniform(2.0, 16.0), 2),
                    start=_log_between(rng, 1, 1 << 21), dtype=dtype)
    return dict(op=op, rows=_log_between(rng, 1, 256), vocab=_log_between(rng, 1000, 128256),
                dtype=dtype, temperature=round(rng.uniform(0.3, 1.5), 3),
                top_k=rng.choice([0, 1, 20, 50, 1000]),
                top_p=rng.choice([1.0, 0.95, 0.9, 0.5]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]),
                mixed=rng.random() < 0.4, masked=rng.choice([0.0, 0.01, 0.5]))


# --------------------------------------------------------------- the inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _qmin(bits, sym):
    return 1 - (1 << (bits - 1)) if sym else 0


def _quantized(case, gen):
    """Codes, scales and zeros of N(0, 0.02^2) weights rounded to the nearest,
    and each column's group (a random order of the columns for act-order)."""
    m, n, g, bits = case["m"], case["n"], case["group"], case["bits"]
    order = torch.randperm(n, generator=gen, device="cuda") if case["act_order"] else \
        torch.arange(n, device="cuda")
    w = (torch.randn((m, n // g, g), generator=gen, device="cuda") * 0.02)
    if case["sym"]:
        qmax = (1 << (bits - 1)) - 1
        scales = (w.abs().amax(-1) / qmax).clamp_min(1e-8)
        zeros = torch.zeros_like(scales)
    else:
        qmax = (1 << bits) - 1
        mn, mx = w.amin(-1), w.amax(-1)
        scales = ((mx - mn) / qmax).clamp_min(1e-8)
        zeros = (-mn / scales).round().clamp(0, qmax)
    qmin = _qmin(bits, case["sym"])
    q = (w / scales[..., None] + zeros[..., None]).round().clamp(qmin, qmax) - qmin
    codes = torch.empty((m, n), dtype=torch.uint8, device="cuda")
    codes[:, order] = q.to(torch.uint8).view(m, n)
    g_idx = torch.empty((n,), dtype=torch.int32, device="cuda")
    g_idx[order] = (torch.arange(n, device="cuda") // g).to(torch.int32)
    return codes, scales, zeros, g_idx, order.to(torch.int32)


def _packed_words(codes, bits):
    """Each row's codes as one little-endian bit stream in 32-bit words."""
    m, n = codes.shape
    words = (n * bits + 31) // 32
    bit = torch.arange(n, device="cuda") * bits
    v = codes.long() << (bit % 32)
    out = torch.zeros((m, words + 1), dtype=torch.int64, device="cuda")
    out.index_add_(1, bit // 32, v & 0xffffffff)
    out.index_add_(1, bit // 32 + 1, v >> 32)
    out = out[:, :words]
    return torch.where(out >= 1 << 31, out - (1 << 32), out).to(torch.int32)


def _activations(case, gen):
    """N(0, 1) times a log-normal scale per channel, as calibration inputs are."""
    scale = torch.exp(torch.randn((case["n"],), generator=gen, device="cuda"))
    x = torch.randn((case["tokens"], case["n"]), generator=gen, device="cuda") * scale
    return x.to(getattr(torch, case["dtype"]))


def _frequencies(case):
    """Radians per position of each pair, in float64, and the factor on cos and sin."""
    d, base = case["rotary_dim"], 10000.0
    i = torch.arange(d // 2, dtype=torch.float64)
    inv = base ** (-2.0 * i / d)
    if case["scaling"] == "linear":
        return inv / case["factor"], 1.0
    if case["scaling"] == "yarn":
        # pairs that turn more than 32 times over 4096 positions keep their
        # frequency, those that turn less than once are slowed down, a ramp between
        lo = max(math.floor(d * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(base))), 0)
        hi = min(math.ceil(d * math.log(4096 / (2 * math.pi)) / (2 * math.log(base))), d - 1)
        keep = 1.0 - ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv * keep + inv / case["factor"] * (1 - keep), 0.1 * math.log(case["factor"]) + 1.0
    return inv, 1.0


def _heads(case, gen):
    b, s, d = case["batch"], case["seq"], case["head_dim"]
    dt = getattr(torch, case["dtype"])
    # projections come out [batch, seq, heads * head_dim]; heads are a view of them
    q = torch.randn((b, s, case["heads"], d), generator=gen, device="cuda").to(dt).transpose(1, 2)
    k = torch.randn((b, s, case["kv_heads"], d), generator=gen, device="cuda").to(dt)
    off = torch.randint(0, 50, (b, 1), generator=gen, device="cuda")
    pos = case["start"] + off + torch.arange(s, device="cuda")
    return q, k.transpose(1, 2), pos


def _logits(case, gen):
    b, v = case["rows"], case["vocab"]
    z = torch.randn((b, v), generator=gen, device="cuda") * 2.0
    likely = torch.randint(0, v, (b, 32), generator=gen, device="cuda")
    z.scatter_add_(1, likely, 4.0 + 6.0 * torch.rand((b, 32), generator=gen, device="cuda"))
    if case["masked"]:
        z[torch.rand((b, v), generator=gen, device="cuda") < case["masked"]] = -math.inf
    z = z.to(getattr(torch, case["dtype"]))
    u = torch.rand((b,), generator=gen, device="cuda")
    par = dict(temperature=case["temperature"], top_k=case["top_k"], top_p=case["top_p"],
               min_p=case["min_p"])
    if case["mixed"]:
        r = torch.rand((4, b), generator=gen, device="cuda")
        par = dict(temperature=torch.where(r[0] < 0.1, torch.zeros_like(r[0]), 0.4 + r[0]),
                   top_k=torch.where(r[1] < 0.5, torch.zeros_like(r[1]), 1 + 200 * r[1]).int(),
                   top_p=torch.where(r[2] < 0.3, torch.ones_like(r[2]), 0.3 + 0.7 * r[2]),
                   min_p=torch.where(r[3] < 0.5, torch.zeros_like(r[3]), 0.1 * r[3]))
    return z, u, par


def prepare(case, seed):
    gen = _gen(seed)
    state = dict(case=case)
    if case["op"] == "linear":
        codes, scales, zeros, g_idx, order = _quantized(case, gen)
        state.update(qweight=_packed_words(codes, case["bits"]), scales=scales, zeros=zeros,
                     g_idx=g_idx, x=_activations(case, gen))
        if own:  # the packed layer as it is loaded, laid out once for the products
            from jax_gptq_b200 import linear, packing
            state["weights"] = linear.prepare_linear(packing.PackedLinear(
                state["qweight"], scales, zeros, g_idx, order, case["bits"], case["group"],
                case["sym"], case["n"]))
    elif case["op"] == "rotary":
        q, k, pos = _heads(case, gen)
        inv, factor = _frequencies(case)
        state.update(q=q, k=k, positions=pos, inv=inv.cuda(), factor=factor)
        if own:
            from jax_gptq_b200 import rotary
            scaling = {"none": None, "linear": rotary.LinearScaling(case["factor"]),
                       "yarn": rotary.YarnScaling(case["factor"], 4096)}[case["scaling"]]
            state["plan"] = rotary.rotary_plan(case["head_dim"], theta=10000.0,
                                               rotary_dim=case["rotary_dim"],
                                               interleaved=case["interleaved"], scaling=scaling)
    else:
        state["logits"], state["u"], state["par"] = _logits(case, gen)
    return state


# ------------------------------------------------------------ the operators

def run(state):
    op = state["case"]["op"]
    if not own:
        return {"linear": _linear, "rotary": _rotary, "sample": _sample}[op](state)
    if op == "linear":
        from jax_gptq_b200 import linear
        return linear.packed_matmul(state["x"], state["weights"])
    if op == "rotary":
        from jax_gptq_b200 import rotary
        return rotary.apply_rotary(state["q"], state["k"], state["positions"], state["plan"])
    from jax_gptq_b200 import sampling
    got = sampling.sample_tokens(state["logits"], state["u"], **state["par"])
    return got.tokens, got.logprobs


def _linear(state):
    """Codes out of the bit stream, float32 weights, one float32 product."""
    case, q = state["case"], state["qweight"]
    bits = case["bits"]
    bit = torch.arange(case["n"], device="cuda", dtype=torch.int32) * bits
    word, off = (bit // 32).long(), bit % 32
    code = q[:, word] >> off
    if 32 % bits:  # a code may begin in one word and end in the next
        nxt = q[:, (word + 1).clamp_max(q.shape[1] - 1)] << (32 - off) % 32
        code = torch.where(off + bits > 32, (code & ((1 << (32 - off)) - 1)) | nxt, code)
    code = code & ((1 << bits) - 1)
    g = state["g_idx"].long()
    w = (code.float() + (_qmin(bits, case["sym"]) - state["zeros"])[:, g]) * state["scales"][:, g]
    return (state["x"].float() @ w.T).to(state["x"].dtype)


def _turn(x, cos, sin, rotary_dim, interleaved):
    xf, half = x.float(), rotary_dim // 2
    out = xf.clone()
    if interleaved:
        a, b = xf[..., 0:rotary_dim:2], xf[..., 1:rotary_dim:2]
        out[..., 0:rotary_dim:2], out[..., 1:rotary_dim:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = xf[..., :half], xf[..., half:rotary_dim]
        out[..., :half], out[..., half:rotary_dim] = a * cos - b * sin, b * cos + a * sin
    return out.to(x.dtype)


def _rotary(state):
    case = state["case"]
    angle = state["positions"].double()[:, None, :, None] * state["inv"]  # [B, 1, S, pairs]
    cos = (angle.cos() * state["factor"]).float()
    sin = (angle.sin() * state["factor"]).float()
    return tuple(_turn(x, cos, sin, case["rotary_dim"], case["interleaved"])
                 for x in (state["q"], state["k"]))


def _per_row(v, rows):
    """A setting as float64 [rows, 1]."""
    if isinstance(v, torch.Tensor):
        return v.double()[:, None]
    return torch.full((rows, 1), float(v), dtype=torch.float64, device="cuda")


def _sample(state):
    z = state["logits"].double()
    rows, vocab = z.shape
    t, k, p, mp = (_per_row(state["par"][s], rows) for s in
                   ("temperature", "top_k", "top_p", "min_p"))
    top = z.amax(1, keepdim=True)
    # temperature 0 is the largest logit alone, the first of equal ones
    e = ((z - top) / torch.where(t > 0, t, torch.ones_like(t))).exp()
    k = torch.where(t > 0, torch.where(k > 0, k, torch.full_like(k, vocab)), torch.ones_like(k))
    order = z.sort(dim=1, descending=True, stable=True).indices
    es = e.gather(1, order)
    rank = torch.arange(vocab, device="cuda")[None]
    es = torch.where(rank < k, es, torch.zeros_like(es))
    before = es.cumsum(1) - es
    keep = (rank < k) & ((before < p * es.sum(1, keepdim=True)) | (p >= 1)) & (es >= mp)
    keep[:, 0] = True
    kept = torch.zeros_like(e).scatter_(1, order, torch.where(keep, es, torch.zeros_like(es)))
    cum = kept.cumsum(1)
    total = cum[:, -1:]
    token = (cum <= state["u"].double()[:, None] * total).sum(1)
    last = vocab - 1 - (kept.flip(1) > 0).int().argmax(1)
    token = torch.minimum(token, last)
    logprob = (kept.gather(1, token[:, None]) / total).log()[:, 0]
    return token, logprob.float()


# ----------------------------------------------------- what it cannot do without

def work(case):
    size = {"bfloat16": 2, "float16": 2, "float32": 4}[case["dtype"]]
    if case["op"] == "linear":
        t, m, n = case["tokens"], case["m"], case["n"]
        groups = n // case["group"]
        return {"bytes": m * n * case["bits"] / 8 + 8 * m * groups + 4 * n + size * t * (m + n),
                "flops": 2.0 * t * m * n}
    if case["op"] == "rotary":
        heads = case["heads"] + case["kv_heads"]
        n = case["batch"] * case["seq"] * heads
        return {"bytes": 2.0 * size * n * case["head_dim"] + 8 * case["batch"] * case["seq"],
                "flops": 3.0 * n * case["rotary_dim"]}
    return {"bytes": float(size) * case["rows"] * case["vocab"] + 16 * case["rows"],
            "flops": 4.0 * case["rows"] * case["vocab"]}


# ----------------------------------------------------------------- in 64 bits

def exact(case, seed):
    gen = _gen(seed)
    if case["op"] == "linear":
        codes, scales, zeros, g_idx, _ = _quantized(case, gen)
        x = _activations(case, gen).double()
        out = torch.zeros((case["tokens"], case["m"]), dtype=torch.float64, device="cuda")
        for r in range(0, case["m"], 4096):
            q = codes[r:r + 4096].double() + _qmin(case["bits"], case["sym"])
            s = scales[r:r + 4096].double().index_select(1, g_idx.int())
            z = zeros[r:r + 4096].double().index_select(1, g_idx.int())
            out[:, r:r + 4096] = torch.einsum("tc,rc->tr", x, (q - z) * s)
        return out
    if case["op"] == "rotary":
        q, k, pos = _heads(case, gen)
        inv, factor = _frequencies(case)
        turn = torch.polar(torch.tensor(factor, dtype=torch.float64, device="cuda"),
                           pos.double()[:, None, :, None] * inv.cuda())
        r = case["rotary_dim"]
        both = []
        for x in (q.double(), k.double()):
            head, rest = x[..., :r], x[..., r:]
            if case["interleaved"]:
                c = torch.view_as_complex(head.unflatten(-1, (r // 2, 2)).contiguous()) * turn
                head = torch.view_as_real(c).flatten(-2)
            else:
                c = torch.complex(head[..., :r // 2], head[..., r // 2:]) * turn
                head = torch.cat([c.real, c.imag], -1)
            both.append(torch.cat([head, rest], -1))
        return tuple(both)
    logits, u, par = _logits(case, gen)
    rows, vocab = logits.shape
    z, u = logits.double().cpu().numpy(), u.double().cpu().numpy()
    t, k, p, mp = (_per_row(par[s], rows).cpu().numpy()[:, 0] for s in
                   ("temperature", "top_k", "top_p", "min_p"))
    tokens, logprobs = np.zeros(rows, np.int64), np.zeros(rows)
    for b in range(rows):
        if t[b] <= 0:
            tokens[b] = int(np.argmax(z[b]))
            continue
        order = np.argsort(-z[b], kind="stable")
        if k[b] > 0:
            order = order[:int(k[b])]
        weight = np.exp((z[b][order] - z[b].max()) / t[b])
        if p[b] < 1:
            before = np.concatenate([[0.0], np.cumsum(weight)[:-1]])
            count = max(1, int(np.count_nonzero(before < p[b] * weight.sum())))
            order, weight = order[:count], weight[:count]
        count = max(1, int(np.count_nonzero(weight >= mp[b])))
        order, weight = order[:count], weight[:count]
        by_index = np.argsort(order)
        order, weight = order[by_index], weight[by_index]
        cum = np.cumsum(weight)
        at = min(int(np.searchsorted(cum, u[b] * cum[-1], side="right")), len(order) - 1)
        while weight[at] == 0:
            at -= 1
        tokens[b], logprobs[b] = order[at], math.log(weight[at] / cum[-1])
    return torch.from_numpy(tokens), torch.from_numpy(logprobs)
