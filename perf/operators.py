"""Cases of the few-bit inference operators: RMS norm into int8 rows, products with 4-bit weights,
the paged int8 key/value cache, and attention over it.

`run` computes a case either in its plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with `own` true, through libsdq's entry points.  `exact` gives the same
results from the definitions in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2, "i8": 3}   # SDQ_F32, SDQ_BF16, SDQ_F16, SDQ_I8
SIZES = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1}

_lib = None


def lib():
    """The framework's library object, bound to GPU 0 as a user's program does it once."""
    global _lib
    if _lib is None:
        from __graft_entry__ import load_package
        _lib = load_package().Sdq(0)
    return _lib


# ---------------------------------------------------------------- cases
def listed():
    return [
        # the norm in front of a projection while one token is generated
        {"name": "norm_one_token", "op": "norm", "M": 1, "K": 4096, "type": "bf16", "residual": True, "weight": True},
        # all tokens of a 720p video clip, fp32 residual stream
        {"name": "norm_video_rows", "op": "norm", "M": 27280, "K": 4096, "type": "f32", "residual": True, "weight": True},
        # one token through a square projection
        {"name": "w4_one_token", "op": "w4", "M": 1, "K": 4096, "N": 4096, "type": "bf16", "out": "bf16",
         "group": 128, "scale": "bf16", "bias": False, "gelu": False},
        # a few int8 rows, as the norm leaves them, through a wide first FFN linear with bias and GELU
        {"name": "w4_int8_rows_wide", "op": "w4", "M": 3, "K": 4096, "N": 28672, "type": "i8", "out": "f32",
         "group": 64, "scale": "f16", "bias": True, "gelu": True},
        # a small batch of fp32 rows through a second FFN linear with an odd output width
        {"name": "w4_batch_fp32", "op": "w4", "M": 24, "K": 14336, "N": 5003, "type": "f32", "out": "f32",
         "group": 32, "scale": "f32", "bias": True, "gelu": False},
        # one new token of each of 48 sequences goes into the cache
        {"name": "cache_append_tokens", "op": "append", "batch": 48, "rows": 48, "context": 2000, "heads": 8, "dim": 128,
         "page": 16, "type": "bf16"},
        # chunks of five sequences of uneven lengths, fp32 keys and values of many small heads
        {"name": "cache_append_chunks", "op": "append", "batch": 5, "rows": 8001, "context": 700, "heads": 24, "dim": 64,
         "page": 64, "type": "f32"},
        # whole sequences read back dense
        {"name": "cache_read_back", "op": "read", "batch": 6, "rows": 100003, "context": 0, "heads": 8, "dim": 128,
         "page": 32, "type": "bf16"},
        # one token over one long cache: latency and bandwidth of a single sequence
        {"name": "attend_one_long", "op": "attend", "batch": 1, "rows": 1, "context": 32768, "heads": 8, "group": 4, "dim": 128,
         "page": 64, "type": "bf16", "causal": True},
        # one token of each of 64 sequences of uneven lengths
        {"name": "attend_batch", "op": "attend", "batch": 64, "rows": 64, "context": 4096, "heads": 8, "group": 4, "dim": 128,
         "page": 16, "type": "f16", "causal": True},
        # fp32 chunks (the framework's own activation type) with a key head for each query head
        {"name": "attend_chunk_fp32", "op": "attend", "batch": 2, "rows": 1000, "context": 8000, "heads": 24, "group": 1, "dim": 128,
         "page": 64, "type": "f32", "causal": False},
        # ragged causal chunks with shared key heads over a long cache
        {"name": "attend_chunk_long", "op": "attend", "batch": 3, "rows": 1537, "context": 16000, "heads": 8, "group": 4, "dim": 128,
         "page": 64, "type": "bf16", "causal": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "w4", "append", "read", "attend", "attend"])
    t = rng.choice(["f32", "bf16", "f16"])
    if op == "norm":
        K = _log(rng, 64, 16384)
        return {"op": "norm", "M": _log(rng, 1, min(27280, (64 << 20) // K)), "K": K, "type": t,
                "residual": rng.random() < 0.7, "weight": rng.random() < 0.8}
    if op == "w4":
        return {"op": "w4", "M": _log(rng, 1, 32), "K": _log(rng, 64, 14336), "N": _log(rng, 8, 20000),
                "type": rng.choice(["f32", "bf16", "f16", "i8"]), "out": rng.choice(["f32", "bf16", "f16"]),
                "group": rng.choice([32, 64, 128]), "scale": rng.choice(["f32", "bf16", "f16"]),
                "bias": rng.random() < 0.5, "gelu": rng.random() < 0.3}
    c = {"op": op, "batch": _log(rng, 1, 64), "heads": rng.choice([1, 2, 4, 8, 24]), "dim": rng.choice([32, 64, 80, 112, 128]),
         "page": rng.choice([16, 32, 48, 64, 128]), "type": t}
    if op == "append":
        c.update(rows=max(c["batch"], _log(rng, 1, 8000)), context=_log(rng, 1, 2000))
    elif op == "read":
        c.update(rows=max(c["batch"], _log(rng, 1, 60000)), context=0)
    else:
        c.update(group=rng.choice([1, 2, 4, 8]), causal=rng.random() < 0.6)
        c["rows"] = c["batch"] if rng.random() < 0.5 else max(c["batch"], _log(rng, 1, 1200))
        heads = c["heads"] * c["group"]      # bounded by what the largest chunk computes, and by its plain scores
        most = min(20000, 400000 // c["batch"], 2 ** 28 // (c["rows"] * heads), 2 ** 27 // (c["rows"] * c["group"]))
        c["context"] = _log(rng, 1, max(16, most))
    return c


def _lengths(case):
    """(new rows, keys) of each sequence: uneven, fixed by the case alone."""
    B, rows, context = case["batch"], case["rows"], case["context"]
    share = [0.25 + (b + 1) * 0.6180339887 % 1.0 for b in range(B)]
    new = [1 + int((rows - B) * s / sum(share)) for s in share]
    new[0] += rows - sum(new)
    old = [context if b == 0 else int(context * (0.3 + 0.7 * ((b + 1) * 0.7548776662 % 1.0))) for b in range(B)]
    return new, [n + o for n, o in zip(new, old)]


def work(case):
    if case["op"] == "norm":
        M, K, t = case["M"], case["K"], SIZES[case["type"]]
        streams = 3 if case["residual"] else 1
        return {"bytes": M * K * (t * streams + 1) + 4 * M + (4 * K if case["weight"] else 0), "flops": 8 * M * K}
    if case["op"] == "w4":
        M, K, N = case["M"], case["K"], case["N"]
        weights = N * ((K + 1) // 2 + -(-K // case["group"]) * SIZES[case["scale"]])
        return {"bytes": weights + M * K * SIZES[case["type"]] + M * N * SIZES[case["out"]] + (4 * N if case["bias"] else 0)
                + (4 * M if case["type"] == "i8" else 0), "flops": 2 * M * K * N}
    new, keys = _lengths(case)
    H, D, t = case["heads"], case["dim"], SIZES[case["type"]]
    if case["op"] == "attend":
        pairs = sum(n * (k - n) + n * (n + 1) // 2 if case["causal"] else n * k for n, k in zip(new, keys))
        return {"bytes": sum(keys) * H * 2 * (D + 4) + 2 * sum(new) * H * case["group"] * D * t,
                "flops": 4 * D * H * case["group"] * pairs}
    both = 2 if case["op"] == "append" else 1     # an append is read back: the rows' codes cross once, their values twice
    return {"bytes": 2 * sum(new) * H * (D + 4 + both * D * t), "flops": 4 * sum(new) * H * D}


# ---------------------------------------------------------------- inputs
def _quantized(x, most, step=1.0):
    """(codes, scale) of the last axis in `most` steps each way."""
    scale = x.abs().amax(-1).clamp_min(1e-8) * (step / most)
    return torch.round(x / scale[..., None]).clamp_(-most, most).to(torch.int8), scale


class Weight:
    """A 4-bit weight as a user's program keeps it: the library's handle, released with the object."""

    def __init__(self, q, scale, case):
        self.handle = lib().w4_upload(q.data_ptr(), scale.data_ptr(), CODES[case["scale"]], case["N"], case["K"], case["group"])

    def __del__(self):
        try:
            lib().weight_release(self.handle)
        except Exception:
            pass


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    s = {"case": case}
    if case["op"] == "norm":
        M, K, dt = case["M"], case["K"], DTYPES[case["type"]]
        s["x"] = (randn(M, K) * 0.7).to(dt)
        s["residual"] = (randn(M, K) * (1.0 + 4.0 * (torch.arange(K, device="cuda") % 97 == 0))).to(dt) if case["residual"] else None
        s["weight"] = 1.0 + 0.2 * randn(K) if case["weight"] else None
        s["eps"] = 1e-6
        s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
        s["aq"] = torch.empty(M, K, device="cuda", dtype=torch.int8)
        s["scale"] = torch.empty(M, device="cuda")
        s["values"] = torch.empty(M, K, device="cuda")
        return s
    if case["op"] == "w4":
        M, K, N, G = case["M"], case["K"], case["N"], case["group"]
        groups = -(-K // G)
        w = torch.nn.functional.pad(randn(N, K) * 0.02, (0, groups * G - K)).view(N, groups, G)
        scale = (w.abs().amax(-1).clamp_min(1e-6) / 7).to(DTYPES[case["scale"]])
        codes = torch.round(w / scale.float()[..., None]).clamp_(-7, 7).view(N, groups * G)[:, :K].to(torch.int32) + 8
        codes = torch.nn.functional.pad(codes, (0, K % 2), value=8)
        s["q"] = (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8).contiguous()
        s["scale"] = scale.contiguous()
        x = randn(M, K) * (0.3 + torch.rand(K, device="cuda", generator=g))
        s["x"], s["x_scale"] = _quantized(x, 127) if case["type"] == "i8" else (x.to(DTYPES[case["type"]]), None)
        s["bias"] = 0.1 * randn(N) if case["bias"] else None
        s["out"] = torch.empty(M, N, device="cuda", dtype=DTYPES[case["out"]])
        if own:
            s["w"] = Weight(s["q"], s["scale"], case)
        return s
    new, keys = _lengths(case)
    B, H, D, P = case["batch"], case["heads"], case["dim"], case["page"]
    counts = [-(-k // P) for k in keys]
    wide, total = max(counts), sum(counts)
    order = list(range(total + 3))                     # a pool a little larger than what is used
    random.Random(seed).shuffle(order)
    table, at = [], 0
    for n in counts:
        table += order[at:at + n] + [0] * (wide - n)
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s["row_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(keys, dtype=torch.int32, device="cuda")
    s["table"] = torch.tensor(table, dtype=torch.int32, device="cuda").view(B, wide)
    rows, dt = case["rows"], DTYPES[case["type"]]
    pool = (total + 3, H, P, D)
    for n in ("k", "v"):
        if case["op"] == "append":
            s["pool_" + n] = torch.zeros(pool, dtype=torch.int8, device="cuda")
            s["pool_%s_scale" % n] = torch.zeros(pool[:3], device="cuda")
            s[n] = (randn(rows, H, D) * (0.5 + torch.rand(rows, H, 1, device="cuda", generator=g))).to(dt)
        else:
            x = randn(*pool) * (0.5 + torch.rand(*pool[:3], 1, device="cuda", generator=g))
            s["pool_" + n], s["pool_%s_scale" % n] = _quantized(x, 127)
            del x
    if case["op"] == "attend":
        s["q"] = (1.5 * randn(rows, H * case["group"], D)).to(dt)
        s["out"] = torch.empty_like(s["q"])
    else:
        s["out_k"], s["out_v"] = (torch.empty(rows, H, D, dtype=dt, device="cuda") for _ in range(2))
    if own:
        s["cache"] = lib().kv_cache(s["pool_k"].data_ptr(), s["pool_v"].data_ptr(), s["pool_k_scale"].data_ptr(),
                                    s["pool_v_scale"].data_ptr(), pool[0], H, P, D)
        s["seqs"] = lib().kv_seqs(s["row_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), B, wide)
    return s


# ---------------------------------------------------------------- the plain forms and the calls
def run(s):
    op = s["case"]["op"]
    return {"norm": _norm, "w4": _w4, "append": _append, "read": _read, "attend": _attend}[op](s)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _norm(s):
    case = s["case"]
    if own:
        M, K = case["M"], case["K"]
        f = lib()
        f.rmsnorm_quantize(_ptr(s["x"]), CODES[case["type"]], M, K, _ptr(s["aq"]), _ptr(s["scale"]), weight_ptr=_ptr(s["weight"]),
                           eps=s["eps"], residual_ptr=_ptr(s["residual"]), sum_ptr=_ptr(s["sum"]))
        f.dequant_rows_device(_ptr(s["aq"]), _ptr(s["scale"]), M, K, _ptr(s["values"]))
        total, scale, values = s["sum"], s["scale"], s["values"]
    else:
        total = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
        x = total.float()
        eps = float(torch.tensor(s["eps"], dtype=torch.float32))
        r = (1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps)).float()
        h = x * r
        if s["weight"] is not None:
            h = h * s["weight"]
        scale = h.abs().amax(-1) / 127.0
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        q = torch.round(h * (1.0 / scale)[:, None]).clamp_(-127, 127)
        values = q * scale[:, None]
    return {"sum": total if s["residual"] is not None else None, "scale": scale, "values": values}


def _gelu(y):
    return 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))


def _w4(s):
    case = s["case"]
    if own:
        f = lib()
        f.w4_matmul(s["w"].handle, _ptr(s["x"]), CODES[case["type"]], case["M"], _ptr(s["out"]), CODES[case["out"]],
                    a_scale_ptr=_ptr(s["x_scale"]), bias_ptr=_ptr(s["bias"]), gelu=case["gelu"])
        return s["out"]
    K = case["K"]
    q = s["q"].to(torch.int32)
    w = torch.stack((q & 15, q >> 4), -1).flatten(1)[:, :K].float() - 8.0
    w *= s["scale"].float().repeat_interleave(case["group"], 1)[:, :K]
    y = torch.matmul(s["x"].float(), w.t())
    if s["x_scale"] is not None:
        y = y * s["x_scale"][:, None]
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["gelu"]:
        y = _gelu(y)
    return y.to(s["out"].dtype)


def _slots(s):
    """(page, offset in it) of every row."""
    start, P = s["row_start"].long(), s["case"]["page"]
    row = torch.arange(s["case"]["rows"], device="cuda")
    seq = torch.bucketize(row, start[1:], right=True)
    at = s["kv_len"].long()[seq] - start[seq + 1] + row
    return s["table"].long()[seq, at // P], at % P


def _append(s):
    case = s["case"]
    if own:
        f, t = lib(), CODES[case["type"]]
        f.kv_append(s["cache"], s["seqs"], _ptr(s["k"]), _ptr(s["v"]), t, case["rows"])
        f.kv_read(s["cache"], s["seqs"], _ptr(s["out_k"]), _ptr(s["out_v"]), t, case["rows"])
        return {"k": s["out_k"], "v": s["out_v"], "k_scale": s["pool_k_scale"], "v_scale": s["pool_v_scale"]}
    page, off = _slots(s)
    for n in ("k", "v"):
        x = s[n].float()
        scale = x.abs().amax(-1) / 127.0
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        s["pool_" + n][page, :, off] = torch.round(x * (1.0 / scale)[..., None]).clamp_(-127, 127).to(torch.int8)
        s["pool_%s_scale" % n][page, :, off] = scale
    return {**_read(s), "k_scale": s["pool_k_scale"], "v_scale": s["pool_v_scale"]}


def _read(s):
    case = s["case"]
    if own:
        lib().kv_read(s["cache"], s["seqs"], _ptr(s["out_k"]), _ptr(s["out_v"]), CODES[case["type"]], case["rows"])
        return {"k": s["out_k"], "v": s["out_v"]}
    page, off = _slots(s)
    return {n: (s["pool_" + n][page, :, off].float() * s["pool_%s_scale" % n][page, :, off][..., None]).to(DTYPES[case["type"]])
            for n in ("k", "v")}


def _attend(s):
    case = s["case"]
    H, G, D, B = case["heads"], case["group"], case["dim"], case["batch"]
    if own:
        lib().kv_attention(s["cache"], s["seqs"], _ptr(s["q"]), CODES[case["type"]], case["rows"], H * G, _ptr(s["out"]),
                           causal=case["causal"])
        return s["out"]
    # all sequences padded to the longest: keys [B, H, L, D], rows [B, H, n, G, D]
    new, keys = _lengths(case)
    n, L = max(new), max(keys)
    k, v = ((s["pool_" + x][s["table"].long()].float() * s["pool_%s_scale" % x][s["table"].long()][..., None])
            .permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :L] for x in ("k", "v"))
    start, length = s["row_start"].long(), s["kv_len"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(n, device="cuda")
    there = i < count[:, None]                                                     # [B, n]
    q = s["q"].float()[(start[:-1, None] + i).clamp_max(case["rows"] - 1)]          # [B, n, H*G, D]
    q = q.view(B, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, n * G, D)
    scores = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(D))
    last = (length - count)[:, None] + i if case["causal"] else (length - 1)[:, None].expand(B, n)
    seen = torch.arange(L, device="cuda") <= last[..., None]                        # [B, n, L]
    scores = scores.masked_fill_(~seen.repeat_interleave(G, 1)[:, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    out = out.view(B, H, n, G, D).permute(0, 2, 1, 3, 4).reshape(B, n, H * G, D)
    return out[there].to(s["q"].dtype)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        total = None
        if s["residual"] is not None:
            total = x + s["residual"].double()
            x = total.to(s["x"].dtype).double()         # the stream is kept in its type: that is what is normalised
        h = x * (x.pow(2).sum(1, keepdim=True) / case["K"] + s["eps"]).pow(-0.5)
        if s["weight"] is not None:
            h *= s["weight"].double()
        # the int8 values are decided in fp32: no 64-bit counterpart
        return {"sum": total, "scale": h.abs().max(1).values / 127, "values": None}
    if case["op"] == "w4":
        G, K, out = case["group"], case["K"], 0
        x = s["x"].double() * (1.0 if s["x_scale"] is None else s["x_scale"].double()[:, None])
        w = torch.empty(case["N"], K + K % 2, device="cuda", dtype=torch.float64)
        w[:, 0::2], w[:, 1::2] = (s["q"] % 16).double() - 8, torch.div(s["q"], 16, rounding_mode="floor").double() - 8
        for j in range(s["scale"].shape[1]):
            cols = slice(j * G, min(K, (j + 1) * G))
            out = out + torch.einsum("mk,nk,n->mn", x[:, cols], w[:, cols], s["scale"][:, j].double())
        if s["bias"] is not None:
            out += s["bias"].double()
        if case["gelu"]:
            out = 0.5 * out * (1 + torch.tanh(math.sqrt(2 / math.pi) * (out + 0.044715 * out ** 3)))
        return out
    new, keys = _lengths(case)
    P, D, table = case["page"], case["dim"], s["table"].tolist()

    def dense(n, b, first):
        """Values of positions first.. of sequence b, [tokens, H, D]."""
        pages = table[b][first // P:-(-keys[b] // P)]
        x = s["pool_" + n][pages].double() * s["pool_%s_scale" % n][pages].double()[..., None]
        return x.transpose(1, 2).flatten(0, 1)[first % P:][:keys[b] - first]

    if case["op"] == "append":
        out = {}
        where = [(table[b][p // P], p % P) for b in range(case["batch"]) for p in range(keys[b] - new[b], keys[b])]
        page, off = torch.tensor(where, device="cuda").t()
        for n in ("k", "v"):
            x = s[n].double()
            step = x.abs().max(-1).values / 127
            out[n + "_scale"] = torch.zeros(s["pool_%s_scale" % n].shape, dtype=torch.float64, device="cuda")
            out[n + "_scale"][page, :, off] = step
            # which code an fp32 value takes is decided in fp32: no 64-bit counterpart
            out[n] = None if case["type"] == "f32" else torch.round(x / step[..., None]) * step[..., None]
        return out
    if case["op"] == "read":
        return {n: torch.cat([dense(n, b, keys[b] - new[b]) for b in range(case["batch"])]) for n in ("k", "v")}
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for b in range(case["batch"]):
        k, v = dense("k", b, 0), dense("v", b, 0)
        for h in range(case["heads"]):
            hs = slice(h * case["group"], (h + 1) * case["group"])
            for i in range(0, new[b], 512):
                q = s["q"][at + i:at + min(i + 512, new[b]), hs].double()
                z = torch.einsum("ngd,ld->ngl", q, k[:, h]) / math.sqrt(D)
                if case["causal"]:
                    pos = keys[b] - new[b] + i + torch.arange(q.shape[0], device="cuda")
                    z.masked_fill_(torch.arange(keys[b], device="cuda")[None, None] > pos[:, None, None], -math.inf)
                out[at + i:at + i + q.shape[0], hs] = torch.softmax(z, -1) @ v[:, h]
        at += new[b]
    return out
