"""The 8-bit floating-point operators of the framework, as cases to measure.

A checkpoint that is only partly EXL3 keeps its other linears, and some layers'
routed experts, in e4m3 with one fp32 scale for each 128 x 128 block of a
weight.  Three operators serve it:

  quantize   x -> (e4m3, scales): one scale for each row and 128 columns
             (activations), or for each 128 x 128 block (weights);
  linear     y = x . W^T (+ bias), x quantised by row and 128 columns;
  moe        a routed-expert layer for a few tokens: gate / up, clamped SwiGLU,
             down, sum over the experts with the router's weights.

Definitions, with g a group of 128 columns (or a block of 128 x 128):
  s_g = max(max|x_g| / 448, 2^-126), rounded to fp32; with `pow2` the smallest
        power of two that is not below it
  q   = e4m3(x / s_g), nearest, ties to even
  y[r, n] = sum over k-groups of  s_x[r, g] * s_w[n // 128, g] * sum_k q_x[r, k] * q_w[n, k]
  moe: G = x . Wgate^T, U = x . Wup^T, a = silu(min(G, L)) * clamp(U, -L, L),
       a quantised like x, out[t] = sum over the valid slots of weight * (a . Wdown^T).
"""
import math

import torch

own = False

BLOCK = 128


def listed():
    """Sizes: hidden 4096, expert width 2048 and its shards, 1536 and the row counts are this repository's benchmark configurations."""
    return [
        # a decode batch's activations before two projections share them
        {"name": "quantize 16 rows", "op": "quantize", "rows": 16, "cols": 4096, "blocks": 1, "dtype": "bf16", "pow2": False},
        # a long prompt's activations
        {"name": "quantize 8192 rows", "op": "quantize", "rows": 8192, "cols": 4096, "blocks": 1, "dtype": "bf16", "pow2": True},
        # a weight at load time whose sides end inside a block
        {"name": "quantize a weight", "op": "quantize", "rows": 4000, "cols": 4080, "blocks": 128, "dtype": "bf16", "pow2": False},
        # one token through an attention projection
        {"name": "linear 1 row", "op": "linear", "rows": 1, "n": 4096, "k": 4096, "dtype": "bf16", "out": "bf16", "bias": False, "pow2": False},
        # a small decode batch, a ragged head count in the output
        {"name": "linear 7 rows", "op": "linear", "rows": 7, "n": 1336, "k": 4096, "dtype": "fp16", "out": "fp16", "bias": True, "pow2": False},
        # a large decode batch through the shared expert's down projection
        {"name": "linear 100 rows", "op": "linear", "rows": 100, "n": 4096, "k": 2048, "dtype": "bf16", "out": "bf16", "bias": False, "pow2": True},
        # a prefill chunk
        {"name": "linear 512 rows", "op": "linear", "rows": 512, "n": 4096, "k": 4096, "dtype": "bf16", "out": "bf16", "bias": False, "pow2": False},
        # several prompts of odd length, fp32 logits-like output
        {"name": "linear 2050 rows", "op": "linear", "rows": 2050, "n": 1336, "k": 1552, "dtype": "bf16", "out": "fp32", "bias": True, "pow2": False},
        # a long prompt
        {"name": "linear 8192 rows", "op": "linear", "rows": 8192, "n": 4096, "k": 4096, "dtype": "bf16", "out": "bf16", "bias": False, "pow2": False},
        # one token, an eighth of the experts' width
        {"name": "moe 1 token", "op": "moe", "tokens": 1, "experts": 256, "topk": 8, "hidden": 4096, "inter": 256, "dtype": "bf16", "out": "bf16", "zipf": False, "skip": False, "limit": 10.0},
        # the repository's decode benchmark: four tokens, the experts' whole width
        {"name": "moe 4 tokens", "op": "moe", "tokens": 4, "experts": 256, "topk": 8, "hidden": 4096, "inter": 2048, "dtype": "bf16", "out": "bf16", "zipf": False, "skip": False, "limit": 10.0},
        # a full decode batch, popular experts, some slots on another rank
        {"name": "moe 32 tokens", "op": "moe", "tokens": 32, "experts": 256, "topk": 8, "hidden": 4096, "inter": 512, "dtype": "fp16", "out": "fp16", "zipf": True, "skip": True, "limit": 10.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "moe", "moe"])
    if op == "quantize":
        blocks = rng.choice([1, 1, BLOCK])
        cols = 8 * _log(rng, 8, 1024)
        if rng.random() < 0.2:
            cols += rng.randint(1, 7)
        rows = _log(rng, 1, max(2, min(8192, 8192 * 4096 // cols)))
        return {"op": op, "rows": rows, "cols": cols, "blocks": blocks, "dtype": rng.choice(["bf16", "fp16", "fp32"]) if rows * cols < 2 ** 24 else "bf16", "pow2": rng.random() < 0.5}
    if op == "linear":
        n, k = _log(rng, 64, 8192), 16 * _log(rng, 8, 512)
        rows = _log(rng, 1, max(2, min(8192, 8192 * 4096 * 4096 // (n * k))))
        return {"op": op, "rows": rows, "n": n, "k": k, "dtype": rng.choice(["bf16", "fp16"]), "out": rng.choice(["bf16", "fp16", "fp32"]), "bias": rng.random() < 0.3, "pow2": rng.random() < 0.3}
    tokens, topk = _log(rng, 1, 32), rng.choice([1, 2, 4, 6, 8])
    experts = max(topk, _log(rng, 8, 256))
    hidden, inter = BLOCK * _log(rng, 4, 32), BLOCK * _log(rng, 1, 16)
    while min(experts, tokens * topk) * inter * hidden > 32 * 2048 * 4096 or tokens * topk * inter * hidden > 256 * 512 * 4096:
        inter = max(BLOCK, inter // 2 // BLOCK * BLOCK)
        hidden = max(BLOCK, hidden // 2 // BLOCK * BLOCK) if inter == BLOCK else hidden
    return {"op": op, "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "inter": inter, "dtype": rng.choice(["bf16", "fp16"]), "out": rng.choice(["bf16", "fp16"]), "zipf": rng.random() < 0.5, "skip": rng.random() < 0.5, "limit": 10.0}


_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _groups(n):
    return (n + BLOCK - 1) // BLOCK


# ------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _activations(rows, cols, dtype, g):
    """N(0, 1) with a tenth of the channels 20 times larger, as hidden states have them."""
    x = torch.randn((rows, cols), generator=g, device="cuda")
    loud = torch.rand((cols,), generator=g, device="cuda") < 0.1
    return (x * torch.where(loud, 20.0, 1.0)).to(dtype)


def _weight(shape, g):
    """e4m3 weights as a checkpoint holds them: normal values whose largest of 128 x 128 is near 448, and scales that bring them to about 0.02."""
    q = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    flat = q.view(-1, shape[-1])
    for i in range(0, flat.shape[0], 65536):
        part = torch.randn((min(65536, flat.shape[0] - i), shape[-1]), generator=g, device="cuda")
        flat[i:i + part.shape[0]] = part.mul_(109.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    s = torch.rand((*shape[:-2], _groups(shape[-2]), _groups(shape[-1])), generator=g, device="cuda")
    return q, (0.5 + s) * (0.02 / 109.0)


def prepare(case, seed):
    g = _gen(seed)
    c = dict(case)
    if c["op"] == "quantize":
        c["x"] = _activations(c["rows"], c["cols"], _DT[c["dtype"]], g)
        if c["blocks"] == BLOCK:
            c["x"] = c["x"] * 0.02
        return c
    if c["op"] == "linear":
        c["x"] = _activations(c["rows"], c["k"], _DT[c["dtype"]], g)
        c["w"], c["ws"] = _weight((c["n"], c["k"]), g)
        c["b"] = torch.randn((c["n"],), generator=g, device="cuda").to(_DT[c["out"]]) if c["bias"] else None
    else:
        T, E, H, I = c["tokens"], c["experts"], c["hidden"], c["inter"]
        c["x"] = _activations(T, H, _DT[c["dtype"]], g)
        c["w13"], c["w13s"] = _weight((E, 2 * I, H), g)
        c["w2"], c["w2s"] = _weight((E, H, I), g)
        popular = torch.arange(1, E + 1, device="cuda").float().pow(-1.1) if c["zipf"] else torch.ones(E, device="cuda")
        ids = torch.multinomial(popular.expand(T, E), c["topk"], replacement=False, generator=g)
        if c["skip"]:  # a quarter of the experts live on another rank
            c["map"] = torch.where(torch.arange(E, device="cuda") % 4 == 3, -1, torch.arange(E, device="cuda"))
        else:
            c["map"], ids = None, ids.to(torch.int32)
        c["ids"] = ids
        c["rw"] = torch.softmax(torch.randn((T, c["topk"]), generator=g, device="cuda"), dim=1)
        c["y"] = torch.empty((T, H), dtype=_DT[c["out"]], device="cuda")
    if own:
        _prepare_own(c)
    return c


def _prepare_own(c):
    """What a user's program keeps: the layer's linear, or the MoE layer's state."""
    if c["op"] == "linear":
        from dsv4_carve_b200.linear import LinearFP8

        c["layer"] = LinearFP8(c["w"], c["ws"], bias=c["b"], out_dtype=_DT[c["out"]], pow2_scale=c["pow2"])
    else:
        from dsv4_carve_b200 import moe

        c["state"] = moe.Fp8MoeState(c["w13"], c["w13s"], c["w2"], c["w2s"])


# ------------------------------------------------------------------ the framework's calls
def _run_own(c):
    if c["op"] == "quantize":
        from dsv4_carve_b200 import vllm_exl3_c as ext

        return dict(zip(("q", "scale"), ext.fp8_quantize(c["x"], block_rows=c["blocks"], pow2_scale=c["pow2"])))
    if c["op"] == "linear":
        return c["layer"].forward(c["x"])
    from dsv4_carve_b200 import moe

    return moe.apply_moe(c["x"], c["ids"], c["rw"], c["state"], c["map"], c["limit"], out=c["y"])


# ------------------------------------------------------------------ the plain form
def _round_e4m3(v):
    """fp64 -> the nearest e4m3 value (ties to even), as fp64."""
    _, e = torch.frexp(v)
    step = (torch.clamp(e - 1, min=-6).long() - 3 + 1023 << 52).view(torch.float64)  # 2 to that power, by its bits
    return torch.round(v / step) * step


def _scale_of(amax, pow2):
    """The quotient in 64 bits, rounded once: next to a power of two an error of the last bit would double the scale."""
    s = torch.clamp((amax.double() / 448.0).float(), min=2.0 ** -126)
    if pow2:
        m, e = torch.frexp(s)
        s = (torch.where(m == 0.5, e - 1, e) + 127 << 23).view(torch.float32)
    return s


def _pad(x, r, k):
    """x with zeros up to r rows and k columns."""
    out = x.new_zeros((r, k))
    out[: x.shape[0], : x.shape[1]] = x
    return out


def _quant(x, pow2, rows=1):
    """(values that q stands for in fp32, scales) of a 2-D x; the quotient x / s is taken in 64 bits, next to the borders of e4m3."""
    R, K = x.shape
    p = _pad(x.float(), _groups(R) * BLOCK if rows == BLOCK else R, _groups(K) * BLOCK)
    b = p.view(-1, rows, _groups(K), BLOCK)
    s = _scale_of(b.abs().amax(dim=(1, 3)), pow2)
    q = _round_e4m3(b.double() / s[:, None, :, None].double()).float()
    return q.reshape(p.shape)[:R, :K], s


def _spread(s, n, k):
    """Block scales [..., n / 128, k / 128] -> one for each weight [..., n, k]."""
    return s.repeat_interleave(BLOCK, dim=-2).repeat_interleave(BLOCK, dim=-1)[..., :n, :k]


def _dequant_rows(x, pow2):
    q, s = _quant(x, pow2)
    return q * s.repeat_interleave(BLOCK, dim=1)[:, : x.shape[1]]


def _run_plain(c):
    if c["op"] == "quantize":
        q, s = _quant(c["x"], c["pow2"], c["blocks"])
        return {"q": q.to(torch.float8_e4m3fn), "scale": s}
    if c["op"] == "linear":
        w = c["w"].float() * _spread(c["ws"], c["n"], c["k"])
        y = _dequant_rows(c["x"], c["pow2"]) @ w.t()
        if c["b"] is not None:
            y = y + c["b"].float()
        return y.to(_DT[c["out"]])
    x = _dequant_rows(c["x"], False)
    H, I, L = c["hidden"], c["inter"], c["limit"]
    ids = c["ids"].long() if c["map"] is None else c["map"][c["ids"].long()]
    y = torch.zeros(x.shape, device="cuda")
    for slot in range(c["topk"]):
        valid = ids[:, slot] >= 0
        e = ids[:, slot].clamp(min=0)
        w = c["w13"].view(torch.uint8)[e].view(torch.float8_e4m3fn).float() * _spread(c["w13s"][e], 2 * I, H)
        h = torch.bmm(w, x[:, :, None])[:, :, 0]
        g, u = h[:, :I].clamp(max=L), h[:, I:].clamp(-L, L)
        a = _dequant_rows(g / (1.0 + torch.exp(-g)) * u, False)
        w = c["w2"].view(torch.uint8)[e].view(torch.float8_e4m3fn).float() * _spread(c["w2s"][e], H, I)
        d = torch.bmm(w, a[:, :, None])[:, :, 0] * c["rw"][:, slot, None]
        y = y + torch.where(valid[:, None], d, 0.0)
    return y.to(_DT[c["out"]])


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ the definition in 64 bits
_TABLE = []


def _e4m3_table():
    """The finite non-negative e4m3 values by their codes, in fp64."""
    if not _TABLE:
        v = [m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)]
        _TABLE.append(torch.tensor(v[:127], dtype=torch.float64, device="cuda"))
    return _TABLE[0]


def _nearest(v):
    """The nearest table value, a tie to the even code."""
    t = _e4m3_table()
    a = v.abs().clamp(max=448.0)
    hi = torch.searchsorted(t, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = t[hi] - a, a - t[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.copysign(t[code], v)


def _power_above(s):
    """The smallest of the powers of two that is not below s, found by comparing."""
    powers = torch.tensor([2.0 ** e for e in range(-126, 128)], dtype=torch.float64, device="cuda")
    return powers[torch.searchsorted(powers, s.contiguous())]


def _exact_groups(x, pow2):
    """fp64 rows, a whole number of groups -> (q, s): s is a number of 32 bits by its definition."""
    g = x.reshape(x.shape[0], -1, BLOCK)
    s = (g.abs().amax(dim=2) / 448.0).float().double().clamp(min=2.0 ** -126)
    if pow2:
        s = _power_above(s)
    return _nearest(g / s[:, :, None]), s


def _exact_rows(x, pow2):
    """fp64 rows -> the rows after quantising."""
    K = x.shape[1]
    x = torch.nn.functional.pad(x, (0, -K % BLOCK))
    q, s = _exact_groups(x, pow2)
    return (q * s[:, :, None]).reshape(x.shape)[:, :K]


def _exact_weight(q, s):
    rows = torch.arange(q.shape[-2], device="cuda") // BLOCK
    cols = torch.arange(q.shape[-1], device="cuda") // BLOCK
    return q.double() * s.double()[..., rows, :][..., cols]


def exact(case, seed):
    c = prepare(case, seed)
    x = c["x"].double()
    if c["op"] == "quantize":
        if c["blocks"] == 1:
            K = c["cols"]
            q, s = _exact_groups(torch.nn.functional.pad(x, (0, -K % BLOCK)), c["pow2"])
            return {"q": q.reshape(c["rows"], -1)[:, :K], "scale": s}
        R, K = x.shape
        p = torch.nn.functional.pad(x, (0, -K % BLOCK, 0, -R % BLOCK))
        tiles = p.unfold(0, BLOCK, BLOCK).unfold(1, BLOCK, BLOCK)
        s = (tiles.abs().amax(dim=(2, 3)) / 448.0).float().double().clamp(min=2.0 ** -126)
        if c["pow2"]:
            s = _power_above(s)
        rows, cols = torch.arange(R, device="cuda") // BLOCK, torch.arange(K, device="cuda") // BLOCK
        return {"q": _nearest(x / s[rows][:, cols]), "scale": s}
    if c["op"] == "linear":
        y = _exact_rows(x, c["pow2"]) @ _exact_weight(c["w"], c["ws"]).t()
        return y if c["b"] is None else y + c["b"].double()
    x = _exact_rows(x, False)
    I, L = c["inter"], c["limit"]
    out = torch.zeros_like(x)
    ids = c["ids"].tolist()
    here = c["map"].tolist() if c["map"] is not None else list(range(c["experts"]))
    for e in sorted({here[i] for row in ids for i in row if here[i] >= 0}):
        at = [(t, j) for t, row in enumerate(ids) for j, i in enumerate(row) if here[i] == e]
        t, j = torch.tensor(at, device="cuda").t()
        h = x[t] @ _exact_weight(c["w13"][e], c["w13s"][e]).t()
        g, u = torch.clamp(h[:, :I], max=L), torch.clamp(h[:, I:], min=-L, max=L)
        a = _exact_rows(g * torch.sigmoid(g) * u, False)
        out.index_add_(0, t, a @ _exact_weight(c["w2"][e], c["w2s"][e]).t() * c["rw"][t, j].double()[:, None])
    return out


def work(case):
    c = case
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if c["op"] == "quantize":
        n = c["rows"] * c["cols"]
        groups = (_groups(c["rows"]) if c["blocks"] == BLOCK else c["rows"]) * _groups(c["cols"])
        return {"bytes": n * (size[c["dtype"]] + 1) + 4 * groups, "flops": 0}
    if c["op"] == "linear":
        r, n, k = c["rows"], c["n"], c["k"]
        return {"bytes": r * k * size[c["dtype"]] + n * k + 4 * _groups(n) * _groups(k) + r * n * size[c["out"]] + (n * size[c["out"]] if c["bias"] else 0),
                "flops": 2 * r * n * k}
    T, E, H, I = c["tokens"], c["experts"], c["hidden"], c["inter"]
    share = 0.75 if c["skip"] else 1.0
    pairs = T * c["topk"] * share
    p = [float(i) ** -1.1 for i in range(1, E + 1)] if c["zipf"] else [1.0] * E
    total = sum(p)
    # experts that some token takes, about: each of its topk draws misses expert i with 1 - p_i
    active = min(sum(1 - (1 - min(1.0, v / total)) ** (T * c["topk"]) for v in p) * share, pairs)
    return {"bytes": active * 3 * H * I * (1 + 4 / BLOCK ** 2) + T * H * (size[c["dtype"]] + size[c["out"]]) + T * c["topk"] * 12, "flops": 6 * pairs * H * I}
