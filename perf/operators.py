"""The 8-bit serving operators of the hot path as measurable cases.

Four operators that together run an attention layer with 8-bit weights,
activations and cache:

``norm8``       residual addition + RMSNorm + e4m3 codes with a scale for every 128 columns
                (``norm`` false: the codes alone, as an attention output or a feed-forward
                activation needs them)
``mm8``         matrix product of e4m3 codes: weights with a scale for every 128 x 128 block,
                activations with one for every token and 128 columns
``attention8``  the attention layer for 1..10 new tokens over a K/V cache held in int8 with a
                scale for every 64 tokens and head, its newest rows in fp16
``cache8``      packing fp16 rows into that cache and reading rows back

``run`` computes a case with elementary torch operations, or, where ``own`` is true, with the
framework's entry points.  The head layout is the model's: 24 query heads and 4 K/V heads of
dimension 256, rotary positions on the first 64 dimensions with base 1e7.
"""
import math

import torch

own = False

NQ, NKV, HD, GROUP = 24, 4, 256, 6
BLOCK = 64                    # tokens that share a scale in the cache
COLS = 128                    # columns that share a scale in e4m3 codes
TAIL = 128                    # fp16 rows beside the packed cache
CONTEXT = 139264
EPS = 1e-6
E4M3_MAX = 448.0

_hot = None


def hot_path():
    """The framework's handle, made once and kept, as a serving program does."""
    global _hot
    if _hot is None:
        from redshift_b200 import HotPath
        _hot = HotPath()
    return _hot


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # one token of a fresh conversation: latency counts, the cache hardly does
        {"name": "attention8 1 token at 777", "op": "attention8", "batch": 1, "position": 777, "packed": 768},
        # a draft of five tokens verified in a long document, the tail two thirds full
        {"name": "attention8 5 at 32767", "op": "attention8", "batch": 5, "position": 32767, "packed": 32704},
        # the longest context, a full verify block: the bench's shape with the cache in 8 bits
        {"name": "attention8 8 at 139256", "op": "attention8", "batch": 8, "position": 139256, "packed": 139200},
        # decode loop: the 64 oldest rows of the fp16 tail leave for the packed cache
        {"name": "cache8 one block", "op": "cache8", "rows": 64, "begin": 0},
        # a prompt of a few thousand tokens, of which rows from an odd one on are read back
        {"name": "cache8 4096 rows", "op": "cache8", "rows": 4096, "begin": 1001},
        # a long document packed whole, and read back to prefill another block behind it
        {"name": "cache8 32768 rows", "op": "cache8", "rows": 32768, "begin": 0},
        # one decoded token's residual stream
        {"name": "norm8 1 x 5120", "op": "norm8", "tokens": 1, "width": 5120, "norm": True},
        # a prefill block's residual stream
        {"name": "norm8 4096 x 5120", "op": "norm8", "tokens": 4096, "width": 5120, "norm": True},
        # a prefill block's feed-forward activation on its way into the down projection
        {"name": "norm8 1999 x 17408 codes", "op": "norm8", "tokens": 1999, "width": 17408, "norm": False},
        # one decoded token through the output projection of an attention layer
        {"name": "mm8 1 x 6144 x 5120", "op": "mm8", "tokens": 1, "width": 6144, "rows": 5120},
        # a verify block through the feed-forward up projection
        {"name": "mm8 8 x 5120 x 17408", "op": "mm8", "tokens": 8, "width": 5120, "rows": 17408},
        # a prefill block of an odd length through the same projection
        {"name": "mm8 4001 x 5120 x 17408", "op": "mm8", "tokens": 4001, "width": 5120, "rows": 17408},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["attention8", "attention8", "cache8", "norm8", "mm8", "mm8"])
    if op == "attention8":
        batch = rng.randint(1, 10)
        position = _log_int(rng, 16, CONTEXT - 10)
        # the packed part ends anywhere the tail still reaches from
        first = max(0, -(-(position + batch - TAIL) // BLOCK))
        packed = BLOCK * rng.randint(first, max(first, position // BLOCK))
        return {"op": op, "batch": batch, "position": position, "packed": packed}
    if op == "cache8":
        rows = BLOCK * _log_int(rng, 1, 32768 // BLOCK)
        return {"op": op, "rows": rows, "begin": rng.randint(0, rows - 1)}
    if op == "norm8":
        return {"op": op, "tokens": _log_int(rng, 1, 2000), "width": _log_int(rng, 100, 17408), "norm": rng.random() < 0.7}
    return {"op": op, "tokens": _log_int(rng, 1, 4000), "width": 16 * _log_int(rng, 8, 320), "rows": _log_int(rng, 64, 17408)}


def work(case):
    op = case["op"]
    if op == "attention8":
        t, n, packed = case["batch"], case["position"] + case["batch"], case["packed"]
        fp16_rows = case["position"] - packed
        cache = 2 * NKV * (packed * HD + packed // BLOCK * 4) + 2 * fp16_rows * NKV * HD * 2
        new = t * (NQ * 2 * HD + 2 * NKV * HD + NQ * HD) * 4 + 2 * t * NKV * HD * 2
        return {"bytes": cache + new, "flops": 4 * t * NQ * HD * n}
    if op == "cache8":
        rows, back = case["rows"], case["rows"] - case["begin"]
        codes = 2 * NKV * (rows * HD + rows // BLOCK * 4)
        return {"bytes": 2 * rows * NKV * HD * 2 + codes + 2 * back * NKV * HD * 3, "flops": 4 * rows * NKV * HD}
    if op == "norm8":
        t, w = case["tokens"], case["width"]
        blocks = -(-w // COLS)
        return {"bytes": t * (w * ((12 if case["norm"] else 4) + 1) + 4 * blocks) + (4 * w if case["norm"] else 0), "flops": 6 * t * w}
    t, w, r = case["tokens"], case["width"], case["rows"]
    blocks = -(-w // COLS)
    return {"bytes": r * w + t * w + 4 * t * r + 4 * blocks * (t + -(-r // COLS)), "flops": 2 * t * w * r}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _pack_blocks(rows):
    """int8 codes [blocks][4][64][256] and scales [blocks][4] of fp16 rows [64 n][4][256]."""
    x = rows.view(-1, BLOCK, NKV, HD).transpose(1, 2)
    amax = x.abs().amax(dim=(2, 3)).float()
    scales = amax / 127
    codes = torch.zeros(x.shape, dtype=torch.int8, device=rows.device)
    torch.round(x.double() / torch.where(scales > 0, scales, torch.ones_like(scales)).double()[:, :, None, None], out=(q := torch.empty(x.shape, dtype=torch.float64, device=rows.device)))
    codes.copy_(q)
    return codes, scales


def prepare(case, seed):
    g = _generator(seed)
    dev = torch.device("cuda")

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    s = dict(case)
    if case["op"] == "attention8":
        t, position, packed = case["batch"], case["position"], case["packed"]
        blocks = packed // BLOCK
        # keys as they leave the key norm and values of unit size: rows of N(0, 1); codes of such rows
        # spread over a block's range as 127 / 4.3 times a normal variable does
        for name in ("key", "value"):
            s[name + "_codes"] = (normal(max(blocks, 1), NKV, BLOCK, HD) * 29.5).round_().clamp_(-127, 127).to(torch.int8)[:blocks]
            s[name + "_scales"] = (4.3 / 127) * (0.9 + 0.2 * torch.rand((blocks, NKV), generator=g, device=dev))
            s[name + "_tail"] = normal(TAIL, NKV, HD).half()
        s["q_gate"] = normal(t, NQ, 2 * HD)
        s["key"], s["value"] = normal(t, NKV, HD), normal(t, NKV, HD)
        s["q_norm"], s["k_norm"] = 1 + 0.1 * normal(HD), 1 + 0.1 * normal(HD)
        s["out"] = torch.empty((t, NQ, HD), device=dev)
    elif case["op"] == "cache8":
        rows, back = case["rows"], case["rows"] - case["begin"]
        # some channels of a key are far larger than the others, as behind a norm's weights
        gain = 1 + 4 * (torch.rand(HD, generator=g, device=dev) > 0.97)
        s["key_rows"], s["value_rows"] = (normal(rows, NKV, HD) * gain).half(), normal(rows, NKV, HD).half()
        for name in ("key", "value"):
            s[name + "_codes"] = torch.empty((rows // BLOCK, NKV, BLOCK, HD), dtype=torch.int8, device=dev)
            s[name + "_scales"] = torch.empty((rows // BLOCK, NKV), device=dev)
            s[name + "_back"] = torch.empty((back, NKV, HD), dtype=torch.float16, device=dev)
    elif case["op"] == "norm8":
        t, w = case["tokens"], case["width"]
        # a residual stream grows over the layers and has a few large channels
        s["x"] = normal(t, w)
        if case["norm"]:
            s["residual"] = 4 * normal(t, w) * (1 + 20 * (torch.rand(w, generator=g, device=dev) > 0.995))
            s["weights"] = 1 + 0.2 * normal(w)
            s["residual_out"] = torch.empty((t, w), device=dev)
        s["codes"] = torch.empty((t, w), dtype=torch.float8_e4m3fn, device=dev)
        s["scales"] = torch.empty((-(-w // COLS), t), device=dev)
    else:
        t, w, r = case["tokens"], case["width"], case["rows"]
        # weights as a checkpoint holds them, activations as norm8 leaves them: codes that fill e4m3's range
        s["weights"] = (normal(r, w) * 105).clamp_(-448, 448).to(torch.float8_e4m3fn)
        s["weight_scales"] = 2e-4 * (0.5 + torch.rand((-(-r // COLS), -(-w // COLS)), generator=g, device=dev))
        s["codes"] = (normal(t, w) * 150).clamp_(-448, 448).to(torch.float8_e4m3fn)
        s["scales"] = 6e-3 * (0.5 + torch.rand((-(-w // COLS), t), generator=g, device=dev))
        s["out"] = torch.empty((t, r), device=dev)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return {"attention8": _attention8, "cache8": _cache8, "norm8": _norm8, "mm8": _mm8}[s["op"]](s)


def _normed_rotated(x, weight, position):
    """RMSNorm over the last axis and the rotary embedding of dimensions [0, 64), in 64 bits."""
    x = x.double()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.double()
    pos = torch.arange(position, position + x.shape[0], device=x.device, dtype=torch.float64)
    angle = pos[:, None, None] * 1e7 ** (-torch.arange(32, device=x.device, dtype=torch.float64) / 32)
    a, b = x[..., :32], x[..., 32:64]
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., 64:]], -1)


def _attention8(s):
    t, position, packed = s["batch"], s["position"], s["packed"]
    if own:
        hot_path().attention8(s["out"], s["key_codes"], s["key_scales"], s["value_codes"], s["value_scales"], packed,
                              s["key_tail"], s["value_tail"], s["q_gate"], s["key"], s["value"], s["q_norm"],
                              s["k_norm"], t, position, EPS)
        return {"out": s["out"], "key_tail": s["key_tail"], "value_tail": s["value_tail"]}
    dev, n = s["q_gate"].device, position + t
    q = _normed_rotated(s["q_gate"][..., :HD], s["q_norm"], position).float()
    new = torch.arange(position, n, device=dev) % TAIL
    s["key_tail"][new] = _normed_rotated(s["key"], s["k_norm"], position).half()
    s["value_tail"][new] = s["value"].half()
    tail = torch.arange(packed, n, device=dev) % TAIL

    def rows(name):
        old = (s[name + "_codes"].float() * s[name + "_scales"][:, :, None, None]).transpose(1, 2).reshape(-1, NKV, HD)
        return torch.cat([old, s[name + "_tail"][tail].float()])

    keys, values = rows("key").permute(1, 2, 0), rows("value").transpose(0, 1)
    scores = torch.matmul(q.view(t, NKV, GROUP, HD).transpose(0, 1).reshape(NKV, t * GROUP, HD), keys) / 16
    scores = scores.view(NKV, t, GROUP, n)
    seen = torch.arange(n, device=dev) <= torch.arange(position, n, device=dev)[:, None]
    scores = scores.masked_fill(~seen[None, :, None, :], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(NKV, t * GROUP, n)
    o = torch.matmul(p, values).view(NKV, t, GROUP, HD).transpose(0, 1).reshape(t, NQ, HD)
    return {"out": o / (1 + torch.exp(-s["q_gate"][..., HD:])), "key_tail": s["key_tail"], "value_tail": s["value_tail"]}


def _cache8(s):
    rows, begin = s["rows"], s["begin"]
    if own:
        hot = hot_path()
        hot.cache8_pack(s["key_codes"], s["key_scales"], s["value_codes"], s["value_scales"], s["key_rows"], s["value_rows"],
                        0, rows)
        hot.cache8_unpack(s["key_back"], s["value_back"], s["key_codes"], s["key_scales"], s["value_codes"],
                          s["value_scales"], begin, rows, origin=begin)
        return {"key": s["key_back"], "value": s["value_back"], "key_scales": s["key_scales"], "value_scales": s["value_scales"]}
    (kc, ks), (vc, vs) = _pack_blocks(s["key_rows"]), _pack_blocks(s["value_rows"])

    def back(codes, scales):
        return (codes.float() * scales[:, :, None, None]).transpose(1, 2).reshape(rows, NKV, HD)[begin:].half()

    return {"key": back(kc, ks), "value": back(vc, vs), "key_scales": ks, "value_scales": vs}


def _norm8(s):
    t, w = s["tokens"], s["width"]
    if own:
        if s["norm"]:
            hot_path().norm8(s["codes"], s["scales"], s["x"], s["weights"], residual=s["residual"], residual_out=s["residual_out"], epsilon=EPS)
            return {"codes": s["codes"], "scales": s["scales"], "residual_out": s["residual_out"]}
        hot_path().quantize8(s["codes"], s["scales"], s["x"])
        return {"codes": s["codes"], "scales": s["scales"]}
    out = {}
    y = s["x"]
    if s["norm"]:
        out["residual_out"] = y = y + s["residual"]
    y = y.double()
    if s["norm"]:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * s["weights"].double()
    padded = torch.zeros((t, -(-w // COLS) * COLS), dtype=torch.float64, device=y.device)
    padded[:, :w] = y
    scales = (padded.view(t, -1, COLS).abs().amax(-1) / E4M3_MAX).float()
    per_column = scales.repeat_interleave(COLS, 1)[:, :w].double()
    out["codes"] = (y / torch.where(per_column > 0, per_column, torch.ones_like(per_column))).float().clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    out["scales"] = scales.t().contiguous()
    return out


def _mm8(s):
    t, w, r = s["tokens"], s["width"], s["rows"]
    if own:
        hot_path().mm8(s["out"], s["weights"], s["weight_scales"], s["codes"], s["scales"])
        return {"out": s["out"]}
    weights = s["weights"].float() * s["weight_scales"].repeat_interleave(COLS, 0)[:r].repeat_interleave(COLS, 1)[:, :w]
    x = s["codes"].float() * s["scales"].t().repeat_interleave(COLS, 1)[:, :w]
    return {"out": torch.matmul(x, weights.t())}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    return {"attention8": _exact_attention8, "cache8": _exact_cache8, "norm8": _exact_norm8, "mm8": _exact_mm8}[case["op"]](prepare(case, seed))


def _exact_attention8(s):
    t, position, packed = s["batch"], s["position"], s["packed"]
    q_raw, gate = s["q_gate"].double().split(HD, -1)
    out = torch.empty((t, NQ, HD), dtype=torch.float64, device=q_raw.device)
    key_tail, value_tail = s["key_tail"].clone(), s["value_tail"].clone()

    def prepared(row, weight, pos):
        y = row / torch.sqrt(row.square().mean(-1, keepdim=True) + EPS) * weight.double()
        z = y.clone()
        for i in range(32):
            angle = pos * 10000000.0 ** (-i / 32)
            c, sn = math.cos(angle), math.sin(angle)
            z[..., i] = y[..., i] * c - y[..., i + 32] * sn
            z[..., i + 32] = y[..., i + 32] * c + y[..., i] * sn
        return z

    for i in range(t):
        key_tail[(position + i) % TAIL] = prepared(s["key"][i].double(), s["k_norm"], position + i).half()
        value_tail[(position + i) % TAIL] = s["value"][i].half()
    for h in range(NKV):
        def whole(codes, scales, tail):
            old = (codes[:, h].double() * scales[:, h].double()[:, None, None]).reshape(packed, HD)
            return torch.cat([old] + [tail[r % TAIL, h].double()[None] for r in range(packed, position + t)])
        k, v = whole(s["key_codes"], s["key_scales"], key_tail), whole(s["value_codes"], s["value_scales"], value_tail)
        for i in range(t):
            n = position + i + 1
            for j in range(h * GROUP, (h + 1) * GROUP):
                logits = k[:n] @ prepared(q_raw[i, j], s["q_norm"], position + i) / 16
                e = torch.exp(logits - logits.max())
                out[i, j] = (e @ v[:n]) / e.sum() * torch.sigmoid(gate[i, j])
    return {"out": out, "key_tail": key_tail.double(), "value_tail": value_tail.double()}


def _exact_cache8(s):
    begin, found = s["begin"], {}
    for name in ("key", "value"):
        x = s[name + "_rows"].double()
        back, scales = torch.empty_like(x), []
        for b in range(s["rows"] // BLOCK):
            block = x[b * BLOCK:(b + 1) * BLOCK]
            scale = block.abs().amax(dim=(0, 2)) / 127
            scales.append(scale)
            held = scale.float().double()[None, :, None].clamp_min(1e-300)
            back[b * BLOCK:(b + 1) * BLOCK] = torch.round(block / held) * held
        found[name], found[name + "_scales"] = back[begin:], torch.stack(scales)
    return found


def _exact_norm8(s):
    w, found = s["width"], {}
    y = s["x"].double()
    if s["norm"]:
        found["residual_out"] = y + s["residual"].double()
        y = found["residual_out"].float().double()
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / w + EPS) * s["weights"].double()
    codes, scales = torch.empty_like(y), []
    for c in range(0, w, COLS):
        part = y[:, c:c + COLS]
        scale = part.abs().amax(-1) / E4M3_MAX
        scales.append(scale)
        z = part / scale.float().double().clamp_min(1e-300)[:, None]
        # e4m3: steps of 2^(e - 3) in the binade [2^e, 2^(e + 1)), no finer than 2^-9
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -20))).clamp_min(-6) - 3)
        codes[:, c:c + COLS] = (torch.round(z / step) * step).clamp(-E4M3_MAX, E4M3_MAX)
    found["codes"], found["scales"] = codes, torch.stack(scales)
    return found


def _exact_mm8(s):
    w, r = s["width"], s["rows"]
    out = torch.zeros((s["tokens"], r), dtype=torch.float64, device=s["codes"].device)
    for k, c in enumerate(range(0, w, COLS)):
        part = s["codes"][:, c:c + COLS].double() @ s["weights"][:, c:c + COLS].double().t()
        per_row = s["weight_scales"][:, k].double()[torch.arange(r, device=out.device) // COLS]
        out += part * s["scales"][k].double()[:, None] * per_row
    return {"out": out}
