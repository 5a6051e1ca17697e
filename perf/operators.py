"""Cases of the score operators: what they are measured on, and their plain forms.

A compressed vector set keeps its rows as 8-bit floating point (e4m3) with one power-of-two scale
for every 128 columns.  Serving a batch from it is four operators, each measured by itself:

  quantize   float rows -> codes and scales (the base once, every batch of queries at its arrival)
  scores     query rows x base rows: out[q][j] = alpha * <query q, row j> + bias[j]
  adjust     penalties for ids already shown, biases on chosen ids, excluded rows
  topk       the k best of every row of scores, equal scores by the lower id

Layout: codes e4m3 [rows][dim rounded up to 16], scales e8m0 [rows][4 * ceil(dim / 512)], the scale
of block b = columns [128 b, 128 b + 128) in column b; what pads either is zero bytes.
"""
import math

import torch

own = False

FLT_MAX = 3.4028234663852886e38
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"


def up(x, m):
    return -(-x // m) * m


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one query arriving at a server: nothing but latency
        {"name": "quantize_query", "op": "quantize", "rows": 1, "dim": 512, "type": "f32", "ld": 512},
        # the 1M x 512 unit-vector base compressed once
        {"name": "quantize_base", "op": "quantize", "rows": 1_000_000, "dim": 512, "type": "f32", "ld": 512},
        # half-precision embeddings of 200 dimensions, a slice of wider rows
        {"name": "quantize_slice", "op": "quantize", "rows": 100_003, "dim": 200, "type": "bf16", "ld": 256},
        # a single query against the whole 1M base
        {"name": "scores_one", "op": "scores", "q": 1, "n": 1_000_000, "dim": 512, "type": "f32", "bias": False},
        # a server's batch, squared-distance order through the rows' bias
        {"name": "scores_batch", "op": "scores", "q": 64, "n": 1_000_000, "dim": 512, "type": "f32", "bias": True},
        # training queries against a shard of 200-dimensional rows, neither side a multiple of a tile
        {"name": "scores_dense", "op": "scores", "q": 4_001, "n": 100_003, "dim": 200, "type": "bf16", "bias": False},
        # hidden states against a wide projection: arithmetic, not memory
        {"name": "scores_wide", "op": "scores", "q": 4_096, "n": 8_192, "dim": 4_096, "type": "bf16", "bias": False},
        # one session over a small catalogue
        {"name": "adjust_one", "op": "adjust", "q": 1, "n": 32_000, "type": "f32", "seen": 200, "biases": 16,
         "masked": 0.0, "shared": False},
        # logits of a decoding batch: long histories, a grammar that leaves a tenth of the vocabulary
        {"name": "adjust_tokens", "op": "adjust", "q": 64, "n": 128_000, "type": "bf16", "seen": 2_000, "biases": 32,
         "masked": 0.9, "shared": False},
        # sessions over a 1M base with a shared set of deleted rows
        {"name": "adjust_items", "op": "adjust", "q": 32, "n": 1_000_000, "type": "f32", "seen": 100, "biases": 0,
         "masked": 0.05, "shared": True},
        # one query's scores over the 1M base
        {"name": "topk_one", "op": "topk", "q": 1, "n": 1_000_000, "type": "f32", "k": 10, "masked": 0.0},
        # a decoding batch's logits under a mask
        {"name": "topk_tokens", "op": "topk", "q": 256, "n": 128_000, "type": "bf16", "k": 100, "masked": 0.5},
    ]


def spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "scores", "adjust", "topk"])
    if op == "quantize":
        dim = spread(rng, 1, 4_096)
        rows = min(spread(rng, 1, 1_000_000), 256_000_000 // dim)
        return {"op": op, "rows": rows, "dim": dim, "type": rng.choice(["f32", "bf16", "f16"]),
                "ld": dim + rng.choice([0, 0, 1, 8, 56])}
    if op == "scores":
        dim = spread(rng, 16, 4_096)
        q = spread(rng, 1, 4_096)
        n = spread(rng, 100, 1_000_000)
        n = max(100, min(n, 200_000_000 // q, 256_000_000 // dim, 65_000_000_000 // (q * dim)))
        return {"op": op, "q": q, "n": n, "dim": dim, "type": rng.choice(["f32", "bf16", "f16"]),
                "bias": rng.random() < 0.5}
    n = spread(rng, 100, 1_000_000)
    if op == "adjust":
        q = min(spread(rng, 1, 256), max(1, 30_000_000 // n))
        return {"op": op, "q": q, "n": n, "type": rng.choice(["f32", "bf16", "f16"]),
                "seen": rng.choice([0, spread(rng, 1, 8_000)]), "biases": rng.choice([0, spread(rng, 1, 300)]),
                "masked": rng.choice([0.0, 0.05, 0.5, 0.98]), "shared": rng.random() < 0.3}
    q = min(spread(rng, 1, 512), max(1, 30_000_000 // n))
    return {"op": op, "q": q, "n": n, "type": rng.choice(["f32", "bf16", "f16"]), "k": spread(rng, 1, 1_000),
            "masked": rng.choice([0.0, 0.05, 0.5, 0.98])}


def work(case):
    op = case["op"]
    if op == "quantize":
        r, d = case["rows"], case["dim"]
        return {"bytes": r * (d * BYTES[case["type"]] + up(d, 16) + 4 * -(-d // 512)), "flops": 3 * r * d}
    if op == "scores":
        q, n, d = case["q"], case["n"], case["dim"]
        moved = (q + n) * (d + -(-d // 128)) + q * n * BYTES[case["type"]] + (4 * n if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * q * n * d}
    q, n, size = case["q"], case["n"], BYTES[case["type"]]
    if op == "adjust":
        mask = 0 if case["masked"] == 0.0 else (1 if case["shared"] else q) * 4 * -(-n // 32)
        # every score is written, those that are not excluded are read
        moved = q * n * size * (2.0 - case["masked"]) + mask + q * (4 * case["seen"] + 8 * case["biases"] + 12)
        return {"bytes": moved, "flops": 4 * q * (case["seen"] + case["biases"])}
    return {"bytes": q * n * size + 8 * q * case["k"], "flops": q * n}


# ----------------------------------------------------------------------------------------- inputs
def unit_rows(gen, rows, dim):
    """Clustered unit vectors around a common direction, as an encoder gives them."""
    centres = torch.randn(64, dim, generator=gen, device=DEV) * 0.5 + 0.3
    x = torch.randn(rows, dim, generator=gen, device=DEV)
    x += centres[torch.randint(0, 64, (rows,), generator=gen, device=DEV)]
    return x.div_(x.norm(dim=1, keepdim=True).clamp_min(1e-20))


def mask_words(gen, rows, n, share):
    """int32 [rows][ceil(n / 32)]: bit j % 32 of word j // 32 set = column j excluded."""
    words = torch.zeros(rows, -(-n // 32), dtype=torch.int32, device=DEV)
    for b in range(32):
        at = torch.rand(words.shape, generator=gen, device=DEV) < share
        words |= at.to(torch.int32) << b
    return words


def bits(words, n):
    """The same as truth values [rows][n]."""
    shifts = torch.arange(32, dtype=torch.int32, device=words.device)
    return ((words[:, :, None] >> shifts) & 1).reshape(words.shape[0], -1)[:, :n] != 0


def data(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, t = case["op"], TYPES[case["type"]]
    if op == "quantize":
        whole = torch.zeros(case["rows"], case["ld"], dtype=t, device=DEV)
        whole[:, :case["dim"]] = unit_rows(gen, case["rows"], case["dim"]).to(t)
        return {"x": whole[:, :case["dim"]]}
    if op == "scores":
        s = {"queries": plain_quantize(unit_rows(gen, case["q"], case["dim"])),
             "base": plain_quantize(unit_rows(gen, case["n"], case["dim"])), "bias": None}
        if case["bias"]:
            s["bias"] = -0.5 * torch.rand(case["n"], generator=gen, device=DEV)
        return s
    q, n = case["q"], case["n"]
    x = torch.randn(q, n, generator=gen, device=DEV) * 2.5 - 1.0
    s = {"scores": x.to(t)}
    if op == "topk":
        if case["masked"]:
            s["scores"][torch.rand(q, n, generator=gen, device=DEV) < case["masked"]] = -math.inf
        return s
    s.update(seen=None, penalties=None, bias_ids=None, bias=None, excluded=None)
    if case["seen"]:
        # histories repeat themselves (a squared uniform favours low ids) and end in padding
        u = torch.rand(q, case["seen"], generator=gen, device=DEV)
        ids = (u * u * n).to(torch.int32).clamp_(max=n - 1)
        kept = torch.randint(case["seen"] // 2, case["seen"] + 1, (q, 1), generator=gen, device=DEV)
        s["seen"] = torch.where(torch.arange(case["seen"], device=DEV) < kept, ids, -1).contiguous()
        s["penalties"] = torch.rand(q, 3, generator=gen, device=DEV) * 0.5 + torch.tensor([1.0, 0.0, 0.0], device=DEV)
    if case["biases"]:
        s["bias_ids"] = torch.randint(0, n, (q, case["biases"]), generator=gen, device=DEV, dtype=torch.int32)
        s["bias"] = torch.randn(q, case["biases"], generator=gen, device=DEV) * 4.0
    if case["masked"]:
        s["excluded"] = mask_words(gen, 1 if case["shared"] else q, n, case["masked"])
    return s


def prepare(case, seed):
    return {"case": case, **data(case, seed)}


# ------------------------------------------------------------------------------------ plain forms
def plain_quantize(x):
    rows, dim = x.shape
    blocks = -(-dim // 128)
    f = torch.zeros(rows, blocks * 128, device=x.device)
    f[:, :dim] = x
    f = f.view(rows, blocks, 128)
    m, e = torch.frexp(f.abs().amax(dim=2))
    e = (e - 9 + (m > 0.875).to(torch.int32)).clamp(-127, 127)      # 448 = 0.875 * 2^9: the least e with amax <= 448 * 2^e
    e = torch.where(m == 0, -127, e)
    codes = torch.ldexp(f, -e[:, :, None]).to(torch.float8_e4m3fn).view(rows, blocks * 128)[:, :up(dim, 16)]
    scales = torch.zeros(rows, 4 * -(-dim // 512), dtype=torch.uint8, device=x.device)
    scales[:, :blocks] = (e + 127).to(torch.uint8)
    return codes.contiguous(), scales.view(torch.float8_e8m0fnu)


def values(rows, dim):
    codes, scales = rows
    s = torch.exp2(scales.view(torch.uint8)[:, :-(-dim // 128)].float() - 127.0)
    return codes[:, :dim].float() * s.repeat_interleave(128, dim=1)[:, :dim]


def plain_scores(s, dim):
    out = values(s["queries"], dim) @ values(s["base"], dim).t()
    return out if s["bias"] is None else out + s["bias"]


def counts(ids, n, weights):
    """[rows][n]: the sum of `weights` at each id; ids below 0 count nowhere."""
    out = torch.zeros(ids.shape[0], n + 1, dtype=weights.dtype, device=ids.device)
    return out.scatter_add_(1, torch.where(ids < 0, n, ids).long(), weights)[:, :n]


def plain_adjust(s, t):
    x = s["scores"].to(t)
    n = x.shape[1]
    if s["seen"] is not None:
        c = counts(s["seen"], n, torch.ones(s["seen"].shape, dtype=t, device=x.device))
        p = s["penalties"].to(t)
        x = torch.where(c > 0, torch.where(x > 0, x / p[:, :1], x * p[:, :1]), x)
        x = x - p[:, 1:2] * c - p[:, 2:3] * (c > 0).to(t)
    if s["bias_ids"] is not None:
        x = x + counts(s["bias_ids"], n, s["bias"].to(t))
    if s["excluded"] is not None:
        x = x.masked_fill(bits(s["excluded"], n), -math.inf)
    return x


def plain_topk(x, k):
    """Unique keys, score first, then the lower id; what is excluded (-inf) is not returned."""
    q, n = x.shape
    u = x.float().add(0.0).view(torch.int32)                          # + 0: one zero
    order = torch.where(u < 0, u ^ 0x7FFFFFFF, u).to(torch.int64)
    key = (order << 32) | (0xFFFFFFFF - torch.arange(n, device=x.device))
    key = torch.topk(key, min(k, n), dim=1).values
    ids = 0xFFFFFFFF - (key & 0xFFFFFFFF)
    got = x.float().gather(1, ids)
    gone = got == -math.inf
    ids = torch.where(gone, -1, ids).to(torch.int32)
    got = torch.where(gone, -FLT_MAX, got)
    if k > n:
        ids = torch.cat([ids, torch.full((q, k - n), -1, dtype=torch.int32, device=x.device)], 1)
        got = torch.cat([got, torch.full((q, k - n), -FLT_MAX, device=x.device)], 1)
    return ids, got


handle = None


def index():
    """The handle that a program keeps."""
    global handle
    if handle is None:
        from coral_b200 import capi
        handle = capi.Index(1, 4, 32, "ip")
    return handle


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        ix = handle or index()
        if op == "quantize":
            return ix.fp8_quantize(state["x"])
        if op == "scores":
            return ix.fp8_scores(state["queries"], state["base"], case["dim"], bias=state["bias"], dtype=TYPES[case["type"]])
        if op == "adjust":
            return ix.adjust_scores(state["scores"], state["seen"], state["penalties"], state["bias_ids"], state["bias"],
                                    state["excluded"])
        return ix.topk_scores(state["scores"], case["k"])
    if op == "quantize":
        return plain_quantize(state["x"])
    if op == "scores":
        return plain_scores(state, case["dim"]).to(TYPES[case["type"]])
    if op == "adjust":
        return plain_adjust(state, torch.float32).to(TYPES[case["type"]])
    return plain_topk(state["scores"], case["k"])


# ----------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = data(case, seed)
    op = case["op"]
    if op == "quantize":
        x = s["x"].double()
        rows, dim = x.shape
        codes = torch.zeros(rows, up(dim, 16), dtype=torch.float64, device=x.device)
        scales = torch.full((rows, 4 * -(-dim // 512)), 2.0 ** -127, dtype=torch.float64, device=x.device)
        for b in range(-(-dim // 128)):
            v = x[:, 128 * b:128 * b + 128]
            top = v.abs().amax(1, keepdim=True)
            e = torch.ceil(torch.log2(top / 448.0)).clamp(-127, 127)
            e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)      # log2 next to a power of two
            e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e).clamp(-127, 127)
            v = v / torch.exp2(e)
            step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3.0)
            codes[:, 128 * b:128 * b + v.shape[1]] = torch.round(v / step) * step      # ties to even
            scales[:, b:b + 1] = torch.exp2(e)
        return codes, scales
    if op == "scores":
        dim = case["dim"]
        parts = []
        for c, e in (s["queries"], s["base"]):
            w = torch.pow(2.0, e.view(torch.uint8).double() - 127.0)
            col = torch.arange(dim, device=c.device) // 128
            parts.append(c.to(torch.float64)[:, :dim] * w[:, col])
        out = torch.mm(parts[0], parts[1].T)
        if s["bias"] is not None:
            out += s["bias"].double()
        return out
    if op == "adjust":
        x = s["scores"].double()
        q, n = x.shape
        if s["seen"] is not None:
            ids = s["seen"].long()
            row = torch.arange(q, device=x.device)[:, None].expand_as(ids)
            there = ids >= 0
            c = torch.zeros(q * n, dtype=torch.float64, device=x.device)
            c += torch.bincount((row * n + ids)[there], minlength=q * n)
            c = c.view(q, n)
            rep, freq, pres = s["penalties"].double().unsqueeze(2).unbind(1)
            hit = c > 0
            x = torch.where(hit & (x > 0), x / rep, torch.where(hit, x * rep, x)) - freq * c - pres * hit
        if s["bias_ids"] is not None:
            ids = s["bias_ids"].long()
            row = torch.arange(q, device=x.device)[:, None].expand_as(ids)
            x = x.index_put((row, ids), s["bias"].double(), accumulate=True)
        if s["excluded"] is not None:
            j = torch.arange(n, device=x.device)
            x[((s["excluded"][:, j // 32] >> (j % 32)) & 1).bool().expand(q, n)] = -math.inf
        return x
    x, k = s["scores"].double(), case["k"]
    best, ids = torch.sort(x, dim=1, descending=True, stable=True)
    best, ids = best[:, :k].clone(), ids[:, :k].to(torch.int32)
    short = k - best.shape[1]
    if short > 0:
        best = torch.nn.functional.pad(best, (0, short), value=-math.inf)
        ids = torch.nn.functional.pad(ids, (0, short), value=-1)
    ids[best == -math.inf] = -1
    best[best == -math.inf] = -FLT_MAX
    return ids, best
