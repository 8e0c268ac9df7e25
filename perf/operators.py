"""What a layer with capped, biased or range-limited attention needs around the paged cache, as a program that serves a
model calls it: three operators, each with its plain form.

  attend   paged attention whose scores are changed before the softmax: capped by a tanh, lowered in proportion to the
           distance between query and key (one slope per head), and limited to a range of keys per token (the token's own
           document in a packed sequence; a prefix that every token of it sees whole).  Over all the cache's formats
  project  what stands in front of the cache: the norm of every query and key head, the rotary embedding of its first
           channels and the split of the layer's output gate, from packed projection rows
  read     cached rows taken out again as 16-bit values (a prefix handed to another process or another layer format)

`run` computes them with elementary torch operations where `own` is false, and calls the library where it is true.  Rows of
the cache: TQ4 is two halves of {fp16 d; 64 bytes of codes}, an element is d x centroid in a rotated basis (sign diagonal,
256-point Walsh-Hadamard transform); FP8 is 256 e4m3 codes and two fp32 scales; Q8 is four blocks of {fp32 d; 64 int8}; BF16 is
256 values.  A (page, head) holds 16 rows.
"""
import math

import numpy as np
import torch

own = False

D = 256
PAGE = 16
SM_SCALE = 1.0 / 16.0
THETA, EPS = 1.0e6, 1e-6
ROW_BYTES = {"tq4": 132, "fp8": 264, "q8": 272, "bf16": 512}

CENTROID_BITS = (0xbe2d79ec, 0xbe03ac9f, 0xbdce3ac1, 0xbda0412c, 0xbd709113, 0xbd27ba58, 0xbcc640ea, 0xbc03358e,
                 0x3c03358e, 0x3cc640ea, 0x3d27ba58, 0x3d709113, 0x3da0412c, 0x3dce3ac1, 0x3e03ac9f, 0x3e2d79ec)
SIGN_WORDS = (0x29e1d357, 0x48974752, 0xeebc0de4, 0xf1297e2a, 0xba639274, 0xe2eb25d0, 0xfde0ee14, 0x36b5bda1)
CENTROIDS = np.array(CENTROID_BITS, np.uint32).view(np.float32)
SIGNS = np.array([1 - 2 * ((SIGN_WORDS[i >> 5] >> (i & 31)) & 1) for i in range(D)], np.float32)


def attend(name, kv_format, q_heads, kv_heads, batch, ctx_lo, ctx_hi, new=1, new_lo=None, cap=0.0, slopes=False, window=0, doc=0, prefix=0):
    return {"name": name, "kind": "attend", "kv": kv_format, "q_heads": q_heads, "kv_heads": kv_heads, "batch": batch, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "new": new, "new_lo": new if new_lo is None else new_lo, "cap": cap, "slopes": slopes, "window": window,
            "doc": doc, "prefix": prefix}


def project(name, dtype, q_heads, kv_heads, tokens, rotary, planes, gate):
    return {"name": name, "kind": "project", "dtype": dtype, "q_heads": q_heads, "kv_heads": kv_heads, "tokens": tokens, "rotary": rotary,
            "planes": planes, "gate": gate}


def read(name, kv_format, kv_heads, batch, ctx_lo, ctx_hi):
    return {"name": name, "kind": "read", "kv": kv_format, "kv_heads": kv_heads, "batch": batch, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi}


def listed():
    return [
        # one user, a short conversation on a model that caps its scores: latency and launches
        attend("attend_1_short", "tq4", 24, 4, 1, 317, 317, cap=30.0),
        # the serving batch of the decode benchmark, with capped scores
        attend("attend_64_capped", "tq4", 24, 4, 64, 8192, 32768, cap=30.0),
        # a batch on a model without position embeddings, its boundary layers in 8 bits: scores fall off with distance
        attend("attend_16_distance_fp8", "fp8", 24, 4, 16, 1024, 8192, slopes=True),
        # drafted tokens verified on an uncompressed cache: a capped layer with a sliding window
        attend("attend_verify_window", "bf16", 16, 4, 16, 1000, 8192, new=4, cap=50.0, window=2500),
        # ragged prompts of packed documents, padding tokens among them
        attend("attend_documents_q8", "q8", 16, 4, 5, 0, 2053, new=899, new_lo=37, slopes=True, doc=211),
        # prompts whose first part (an image, an instruction) every token of it sees whole, on an uncompressed cache
        attend("attend_prefix_bf16", "bf16", 24, 4, 4, 2048, 2048, new=2048, cap=50.0, prefix=3000),
        # long prompts in 2048-token chunks, half way through, capped
        attend("attend_8x2048", "tq4", 16, 4, 8, 8192, 8192, new=2048, cap=30.0),
        # the projection rows of one decoded token, output gate between the query heads
        project("project_1", "fp16", 24, 4, 1, 64, 3, True),
        # one prompt's rows, the whole head rotated
        project("project_2053", "bf16", 16, 4, 2053, 256, 1, False),
        # a prefill batch's rows, with gate and three position planes
        project("project_32k", "fp16", 24, 4, 32768, 64, 3, True),
        # the last pages of one sequence, for a layer kept in 8 bits
        read("read_tail_fp8", "fp8", 4, 1, 37, 37),
        # cached prefixes of a few sequences on their way out of the pool
        read("read_32k", "tq4", 4, 5, 1025, 13001),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "project", "read"))
    kv_heads = rng.choice((1, 2, 4, 4))
    q_heads = kv_heads * rng.choice((1, 3, 4, 6))
    kv_format = rng.choice(("tq4", "tq4", "fp8", "q8", "bf16", "bf16"))
    if kind == "project":
        case = project("", rng.choice(("fp16", "bf16")), q_heads, kv_heads, _log_int(rng, 1, 32768), rng.choice((16, 64, 128, 192, 256)),
                       rng.choice((1, 3)), rng.random() < 0.5)
    elif kind == "read":
        batch = _log_int(rng, 1, 32)
        hi = _log_int(rng, 1, 65536 // batch)
        case = read("", kv_format, kv_heads, batch, max(1, hi // rng.choice((1, 3))), hi)
    else:
        what = rng.choice(("decode", "decode", "verify", "chunk", "chunk"))
        if what == "chunk":
            batch = _log_int(rng, 1, 8)
            new = _log_int(rng, 7, 2048)
            hi = rng.choice((0, _log_int(rng, 5, 8192)))
            case = attend("", kv_format, q_heads, kv_heads, batch, hi // rng.choice((1, 3)), hi, new=new, new_lo=max(1, new // rng.choice((1, 5))))
        else:
            batch = _log_int(rng, 1, 96)
            hi = _log_int(rng, 1, min(200000, 1000000 // batch))
            case = attend("", kv_format, q_heads, kv_heads, batch, hi // rng.choice((1, 4)), hi, new=1 if what == "decode" else rng.randint(2, 5))
        changes = rng.choice(("cap", "cap", "distance", "documents", "prefix", "all"))
        if changes in ("cap", "prefix", "all"):
            case["cap"] = rng.choice((20.0, 30.0, 50.0))
        if changes in ("distance", "documents", "all"):
            case["slopes"] = True
        if changes in ("documents", "all"):
            case["doc"] = _log_int(rng, 3, 5000)
        if changes == "prefix":
            case["prefix"] = _log_int(rng, 1, 4096)
        if changes == "cap" and rng.random() < 0.5:
            case["window"] = _log_int(rng, 1, 8192)
    case.pop("name", None)
    return case


# ---- what a case holds, from its numbers alone -------------------------------------------------------------------------
def _spread(lo, hi, n):
    return [hi] if n == 1 else [hi - (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(case):
    """Cached and new tokens of every sequence.  Long prompts go with short prefixes."""
    n = case["batch"]
    return _spread(case["ctx_lo"], case["ctx_hi"], n), _spread(case.get("new_lo", 0), case.get("new", 0), n)[::-1]


def _visible(case):
    """Per request: (begin, end, key_begin, key_end) of its new tokens, as arrays of positions.  begin / end are the keys a token sees,
    window and causality included; key_begin / key_end what the call is given (None: not given)."""
    res = []
    for c, n in zip(*_lens(case)):
        pos = c + np.arange(n)
        begin, end, kb, ke = np.zeros(n, np.int64), pos + 1, None, None
        if case["window"]:
            begin = np.maximum(0, pos - case["window"] + 1)
        if case["doc"]:      # the token's own document, aligned from the sequence's start; every 97th position is padding
            kb = pos // case["doc"] * case["doc"]
            ke = pos + 1
            kb = np.where(pos % 97 == 96, ke, kb)
        if case["prefix"]:
            ke = np.maximum(pos + 1, case["prefix"])
        if kb is not None:
            begin = np.maximum(begin, kb)
        if ke is not None:
            end = np.minimum(ke, c + n)
        res.append((begin, end, kb, ke))
    return res


def _axes(rotary, planes):
    """Position plane of every frequency: interleaved thirds for three planes."""
    half = rotary // 2
    s1, s2 = (half + 1) // 3, half // 3
    axis = np.zeros(half, np.int64)
    if planes == 3:
        i = np.arange(half)
        axis[(i % 3 == 1) & (i < 3 * s1)] = 1
        axis[(i % 3 == 2) & (i < 3 * s2)] = 2
    return axis, (half - s1 - s2, s1, s2)


def work(case):
    if case["kind"] == "project":
        n, rows = case["tokens"], case["q_heads"] + case["kv_heads"]
        moved = 2 * rows * D * 2 + (2 * case["q_heads"] * D * 2 if case["gate"] else 0)
        return {"bytes": n * (moved + 4 * case["planes"]), "flops": n * rows * (4 * D + 3 * case["rotary"])}
    if case["kind"] == "read":
        n = sum(_lens(case)[0])
        rotation = 8 * D if case["kv"] == "tq4" else 0
        return {"bytes": 2 * n * case["kv_heads"] * (ROW_BYTES[case["kv"]] + 2 * D), "flops": 2 * n * case["kv_heads"] * (D + rotation)}
    keys = pairs = 0
    for begin, end, _, _ in _visible(case):
        seen = end > begin
        pairs += int((end - begin)[seen].sum())
        keys += int(end[seen].max() - begin[seen].min()) if seen.any() else 0
    rows = sum(_lens(case)[1]) * case["q_heads"]
    return {"bytes": keys * case["kv_heads"] * 2 * ROW_BYTES[case["kv"]] + 2 * rows * D * 2, "flops": 4 * D * pairs * case["q_heads"]}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _code_bytes():
    """65536 uniform numbers -> bytes of two 4-bit codes with the frequencies they have in rotated rows."""
    mid = torch.tensor((CENTROIDS[1:] + CENTROIDS[:-1]) / 2)
    z = torch.special.ndtri((torch.arange(256, dtype=torch.float64) + 0.5) / 256) / 16
    code = torch.bucketize(z.float(), mid)
    return (code[None, :] + 16 * code[:, None]).reshape(-1).to(torch.uint8).cuda()


def _rows(fmt, n, gen):
    """n cached rows as bytes, [n, row bytes]: elements of about unit variance, row magnitudes that differ."""
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    if fmt == "bf16":
        return (rand(n, D) * torch.exp(0.25 * rand(n, 1))).to(torch.bfloat16).view(torch.uint8).view(n, 512)
    if fmt == "tq4":
        d = (16.0 * torch.exp(0.25 * rand(n, 2))).to(torch.float16).view(torch.uint8).view(n, 2, 2)
        u = torch.randint(0, 65536, (n, 2, 64), generator=gen, device="cuda", dtype=torch.int32)
        return torch.cat([d, _code_bytes()[u]], 2).view(n, 132)
    if fmt == "fp8":
        codes = (rand(n, D) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        return torch.cat([codes, (torch.exp(0.25 * rand(n, 2)) / 100).view(torch.uint8).view(n, 8)], 1)
    codes = torch.round(rand(n, 4, 64) * 40).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return torch.cat([(torch.exp(0.25 * rand(n, 4, 1)) / 40).view(torch.uint8).view(n, 4, 4), codes], 2).view(n, 272)


def _slab(fmt, pages, heads, gen):
    out = torch.empty(pages, heads, PAGE, ROW_BYTES[fmt], dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 19) // (heads * PAGE))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        out[p:p + n] = _rows(fmt, n * heads * PAGE, gen).view(n, heads, PAGE, ROW_BYTES[fmt])
    return out


def _cache(case, seed, new):
    """Pages of every sequence from a shuffled pool, page 0 kept free: slabs, page table, positions of the rows."""
    ctx = _lens(case)[0]
    total = [c + n for c, n in zip(ctx, new)]
    need = [(t + PAGE - 1) // PAGE for t in total]
    rng = np.random.RandomState(seed % (1 << 32))
    order = 1 + rng.permutation(sum(need) + 3)
    table = np.zeros((len(need), max(max(need), 1)), np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    gen = _generator(seed)
    pages = len(order) + 1
    return _slab(case["kv"], pages, case["kv_heads"], gen), _slab(case["kv"], pages, case["kv_heads"], gen), table, total, gen


def _own_layer(case, k, v):
    from warp34_b200 import ffi, kv
    rotated, plain = ffi.KV_TRANSFORM_RADEMACHER_WHT256, ffi.KV_TRANSFORM_IDENTITY
    f, t = {"tq4": (ffi.KV_FORMAT_TQ4, rotated), "fp8": (ffi.KV_FORMAT_FP8_E4M3, plain), "q8": (ffi.KV_FORMAT_Q8_0, plain),
            "bf16": (ffi.KV_FORMAT_BF16, plain)}[case["kv"]]
    layer = kv.KvLayer(k.shape[0], case["kv_heads"], formats=(f, f, t, t))
    layer.k.copy_(k.view(-1))
    layer.v.copy_(v.view(-1))
    return layer


def _dtype(case):
    if "dtype" in case:
        return torch.float16 if case["dtype"] == "fp16" else torch.bfloat16
    return torch.bfloat16 if case["kv"] == "bf16" else torch.float16


def prepare(case, seed):
    return {"attend": _prepare_attend, "project": _prepare_project, "read": _prepare_read}[case["kind"]](case, seed)


def _prepare_attend(case, seed):
    ctx, new = _lens(case)
    k, v, table, total, gen = _cache(case, seed, new)
    n, hq = sum(new), case["q_heads"]
    q = (torch.randn(n, hq, D, generator=gen, device="cuda") * 4).to(_dtype(case))
    seen = _visible(case)
    ranges = [None, None]
    for i in range(2):
        if seen[0][2 + i] is not None:
            ranges[i] = torch.from_numpy(np.concatenate([s[2 + i] for s in seen]).astype(np.int32)).cuda()
    slopes = None
    if case["slopes"]:
        slopes = (2.0 ** (-8.0 * torch.arange(1, hq + 1, dtype=torch.float64) / hq)).float().cuda()
    s = {"kind": "attend", "case": case, "q": q, "key_begin": ranges[0], "key_end": ranges[1], "slopes": slopes, "ctx": ctx, "new": new,
         "total": total, "table": torch.from_numpy(table.astype(np.int64)).cuda()}
    if not own:
        s.update(k=k, v=v)
        return s
    from warp34_b200 import kv
    starts = np.concatenate([[0], np.cumsum(new)])
    slots = np.concatenate([table[r, np.arange(c, t) // PAGE] * PAGE + np.arange(c, t) % PAGE for r, (c, t) in enumerate(zip(ctx, total))])
    s.update(layer=_own_layer(case, k, v), ex=kv.Executor(), out=torch.zeros_like(q),
             batch=kv.StepBatch(starts, ctx, total, table, slots, table.shape[1], SM_SCALE, sliding_window=case["window"]))
    return s


def _prepare_project(case, seed):
    gen = _generator(seed)
    n, hq, hkv, dt = case["tokens"], case["q_heads"], case["kv_heads"], _dtype(case)
    width = 2 * D if case["gate"] else D
    packed = torch.randn(n, hq * width + 2 * hkv * D, generator=gen, device="cuda")      # rows [queries (and gates) | keys | values]
    packed = (packed * torch.exp(0.5 * torch.randn(n, 1, generator=gen, device="cuda"))).to(dt)
    weights = [(torch.randn(D, generator=gen, device="cuda") * 0.2).to(dt) for _ in range(2)]
    first = torch.randint(0, 262144 - n + 1, (1,), generator=gen, device="cuda", dtype=torch.int32)
    pos = torch.arange(n, dtype=torch.int32, device="cuda") + first
    if case["planes"] == 3:      # text tokens hold the same position in all planes, an image's rows and columns differ
        pos = torch.stack([pos, pos - pos % 5, pos - pos % 3])
    inv_freq = (THETA ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64) / case["rotary"])).float().cuda()
    new = lambda h: torch.zeros(n, h, D, dtype=dt, device="cuda")  # noqa: E731
    s = {"kind": "project", "case": case, "q": packed[:, :hq * width].view(n, hq, width), "k": packed[:, hq * width:(hq * width + hkv * D)].view(n, hkv, D),
         "weights": weights, "pos": pos, "inv_freq": inv_freq}
    if own:
        from warp34_b200 import kv
        s.update(ex=kv.Executor(1 << 16), q_out=new(hq), k_out=new(hkv), gate_out=new(hq) if case["gate"] else None,
                 sections=_axes(case["rotary"], 3)[1] if case["planes"] == 3 else None)
    return s


def _prepare_read(case, seed):
    ctx = _lens(case)[0]
    k, v, table, total, _ = _cache(case, seed, [0] * len(ctx))
    s = {"kind": "read", "case": case, "total": total, "table": torch.from_numpy(table.astype(np.int64)).cuda()}
    if not own:
        s.update(k=k, v=v)
        return s
    from warp34_b200 import kv
    starts = np.concatenate([[0], np.cumsum(total)])
    slots = np.concatenate([table[r, np.arange(t) // PAGE] * PAGE + np.arange(t) % PAGE for r, t in enumerate(total)])
    out = lambda: torch.zeros(int(starts[-1]), case["kv_heads"] * D, dtype=_dtype(case), device="cuda")  # noqa: E731
    s.update(layer=_own_layer(case, k, v), ex=kv.Executor(1 << 16), k_out=out(), v_out=out(),
             batch=kv.StepBatch(starts, np.zeros(len(total)), total, table, slots, table.shape[1], SM_SCALE))
    return s


def run(state):
    return {"attend": _own_attend if own else _plain_attend, "project": _own_project if own else _plain_project,
            "read": _own_read if own else _plain_read}[state["kind"]](state)


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _own_attend(s):
    from warp34_b200 import kv
    kv.paged_attention_scored(s["ex"], s["layer"], s["batch"], s["q"], s["out"], s["case"]["q_heads"], softcap=s["case"]["cap"],
                              slopes=s["slopes"], key_begin=s["key_begin"], key_end=s["key_end"])
    return s["out"]


def _own_project(s):
    from warp34_b200 import kv
    kv.qk_norm_rope(s["ex"], s["q"], s["k"], s["weights"][0], s["weights"][1], s["pos"], s["inv_freq"], s["q_out"], s["k_out"],
                    gate_out=s["gate_out"], sections=s["sections"], eps=EPS, weight_offset=1.0)
    return [s["q_out"], s["k_out"], s["gate_out"]] if s["case"]["gate"] else [s["q_out"], s["k_out"]]


def _own_read(s):
    from warp34_b200 import kv
    kv.kv_cache_read(s["ex"], s["layer"], s["batch"], s["k_out"], s["v_out"])
    return [s["k_out"], s["v_out"]]


# ---- plain forms, in 32 bits -------------------------------------------------------------------------------------------
_hadamard = None


def _rotation():
    """The 256-point Walsh-Hadamard matrix / 16, times the sign diagonal on its right."""
    global _hadamard
    if _hadamard is None:
        h = torch.ones(1, 1)
        for _ in range(8):
            h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
        _hadamard = (h / 16 * torch.from_numpy(SIGNS)).cuda()
    return _hadamard


def _values(rows, fmt):
    """Bytes [..., row bytes] -> fp32 [..., 256]."""
    lead = rows.shape[:-1]
    if fmt == "bf16":
        return rows.contiguous().view(torch.bfloat16).float()
    if fmt == "tq4":
        halves = rows.reshape(*lead, 2, 66)
        d = halves[..., :2].contiguous().view(torch.float16).float()
        codes = halves[..., 2:]
        codes = torch.stack([codes & 15, codes >> 4], -1).view(*lead, 2, 128).int()
        return (torch.from_numpy(CENTROIDS).cuda()[codes] * d).view(*lead, D) @ _rotation()
    if fmt == "fp8":
        codes = rows[..., :D].contiguous().view(torch.float8_e4m3fn).float().view(*lead, 2, 128)
        return (codes * rows[..., D:].contiguous().view(torch.float32).unsqueeze(-1)).view(*lead, D)
    blocks = rows.reshape(*lead, 4, 68)
    return (blocks[..., 4:].contiguous().view(torch.int8).float() * blocks[..., :4].contiguous().view(torch.float32)).view(*lead, D)


def _sequence(slab, table, r, total, fmt):
    """The cached rows of one sequence: [heads, tokens, 256] in fp32."""
    pages = slab[table[r, :(total + PAGE - 1) // PAGE]]
    rows = pages.transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :total]
    return _values(rows, fmt)


def _plain_attend(s):
    case, q = s["case"], s["q"]
    hq, hkv = case["q_heads"], case["kv_heads"]
    g = hq // hkv
    out = torch.empty_like(q)
    at = 0
    for r, (c, n, total) in enumerate(zip(s["ctx"], s["new"], s["total"])):
        k = _sequence(s["k"], s["table"], r, total, case["kv"])
        v = _sequence(s["v"], s["table"], r, total, case["kv"])
        rows = q[at:at + n].float().view(n, hkv, g, D).permute(1, 2, 0, 3).reshape(hkv, g * n, D)
        sc = (rows @ k.transpose(1, 2)).view(hkv, g, n, total) * SM_SCALE
        if case["cap"] > 0:
            sc = case["cap"] * torch.tanh(sc / case["cap"])
        pos = torch.arange(c, c + n, device=q.device)
        key = torch.arange(total, device=q.device)
        distance = (pos[:, None] - key[None, :])
        if s["slopes"] is not None:
            sc = sc - s["slopes"].view(hkv, g, 1, 1) * distance.abs().float()
        first = torch.zeros_like(pos) if s["key_begin"] is None else s["key_begin"][at:at + n].long()
        end = pos + 1 if s["key_end"] is None else s["key_end"][at:at + n].long()
        seen = (key >= first[:, None]) & (key < end[:, None])
        if case["window"]:
            seen &= distance < case["window"]
        sc = sc.masked_fill(~seen, -math.inf)
        top = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        mass = p.sum(-1, keepdim=True)
        o = (p.view(hkv, g * n, total) @ v).view(hkv, g, n, D) / torch.where(mass > 0, mass, torch.ones_like(mass))
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, hq, D).to(q.dtype)
        at += n
    return out


def _plain_project(s):
    case = s["case"]
    half = case["rotary"] // 2
    pos = s["pos"].double()
    if case["planes"] == 3:
        pos = pos[torch.from_numpy(_axes(case["rotary"], 3)[0]).cuda()].T      # [tokens, frequencies]
    else:
        pos = pos[:, None]
    angle = pos * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    res = []
    for x, w in ((s["q"][..., :D], s["weights"][0]), (s["k"], s["weights"][1])):
        f = x.float()
        f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * (1.0 + w.float())
        a, b = f[..., :half], f[..., half:2 * half]
        res.append(torch.cat([a * cos - b * sin, b * cos + a * sin, f[..., 2 * half:]], -1).to(x.dtype))
    return res + [s["q"][..., D:].contiguous()] if case["gate"] else res


def _plain_read(s):
    fmt, dt = s["case"]["kv"], _dtype(s["case"])
    res = []
    for slab in (s["k"], s["v"]):
        parts = [_sequence(slab, s["table"], r, t, fmt).transpose(0, 1).reshape(t, -1).to(dt) for r, t in enumerate(s["total"])]
        res.append(torch.cat(parts))
    return res


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _elements64(rows, fmt):
    """Stored elements (TQ4: in the rotated basis) of byte rows [n, row bytes], fp64."""
    n = rows.shape[0]
    if fmt == "bf16":
        return (rows.contiguous().view(torch.int16).to(torch.int32) << 16).view(torch.float32).double()
    if fmt == "tq4":
        parts = []
        for h in range(2):
            d = rows[:, 66 * h:66 * h + 2].contiguous().view(torch.float16).double()
            b = rows[:, 66 * h + 2:66 * h + 66].long()
            c = torch.empty(n, 128, dtype=torch.int64, device=rows.device)
            c[:, 0::2], c[:, 1::2] = b % 16, b // 16
            parts.append(torch.tensor(CENTROIDS, device=rows.device).double()[c] * d)
        return torch.cat(parts, 1)
    if fmt == "fp8":
        b = rows[:, :D].int()
        mantissa, exponent = (b & 7).double(), ((b >> 3) & 15)
        x = torch.where(exponent == 0, mantissa / 512, (8 + mantissa) * torch.exp2(exponent.double() - 10))
        x = torch.where(b >= 128, -x, x)
        d = rows[:, D:].contiguous().view(torch.float32).double()
        return x * d.repeat_interleave(128, 1)
    parts = []
    for b in range(4):
        d = rows[:, 68 * b:68 * b + 4].contiguous().view(torch.float32).double()
        c = rows[:, 68 * b + 4:68 * b + 68].double()
        parts.append(torch.where(c >= 128, c - 256, c) * d)
    return torch.cat(parts, 1)


def _transform64(x):
    """256-point Walsh-Hadamard transform / 16 along the last axis, by butterflies."""
    lead = x.shape[:-1]
    for bit in range(8):
        y = x.reshape(*lead, D >> (bit + 1), 2, 1 << bit)
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], -2).reshape(*lead, D)
    return x / 16


def _head_rows(slab, table, r, total, head):
    key = torch.arange(total, device=slab.device)
    return slab[table[r, key // PAGE], head, key % PAGE]


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return {"attend": _exact_attend, "project": _exact_project, "read": _exact_read}[case["kind"]](s)


def _exact_attend(s):
    case = s["case"]
    hq, hkv, fmt = case["q_heads"], case["kv_heads"], case["kv"]
    signs = torch.tensor(SIGNS, device="cuda").double()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for r, (begin, end, _, _) in enumerate(_visible(case)):
        c, n, total = s["ctx"][r], s["new"][r], s["total"][r]
        lo, hi = torch.from_numpy(begin).cuda()[:, None], torch.from_numpy(end).cuda()[:, None]
        key = torch.arange(total, device="cuda")[None]
        hidden = (key < lo) | (key >= hi)
        away = (torch.arange(c, c + n, device="cuda")[:, None] - key).abs().double()
        for kv_head in range(hkv):
            k = _elements64(_head_rows(s["k"], s["table"], r, total, kv_head), fmt)
            v = _elements64(_head_rows(s["v"], s["table"], r, total, kv_head), fmt)
            for head in range(kv_head * hq // hkv, (kv_head + 1) * hq // hkv):
                q = s["q"][at:at + n, head].double()
                if fmt == "tq4":
                    q = _transform64(q * signs)
                t = q @ k.T / 16
                if case["cap"] > 0:
                    t = torch.tanh(t / case["cap"]) * case["cap"]
                if case["slopes"]:
                    t = t - float(s["slopes"][head]) * away
                t[hidden] = -math.inf
                p = torch.softmax(t, 1)
                p = torch.where(hidden.all(1, keepdim=True), torch.zeros_like(p), p)
                o = p @ v
                out[at:at + n, head] = _transform64(o) * signs if fmt == "tq4" else o
        at += n
    return out


def _exact_project(s):
    case = s["case"]
    rot, half = case["rotary"], case["rotary"] // 2
    axis = _axes(rot, case["planes"])[0]
    planes = s["pos"] if case["planes"] == 3 else s["pos"][None]
    turn = torch.stack([planes[int(a)].double() * float(f) for a, f in zip(axis, s["inv_freq"].cpu().double())], 1)
    spin = torch.polar(torch.ones_like(turn), turn)[:, None]
    res = []
    for x, w in ((s["q"][..., :D], s["weights"][0]), (s["k"], s["weights"][1])):
        y = x.double()
        y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / D + EPS) * (w.double() + 1)
        z = torch.complex(y[..., :half], y[..., half:rot]) * spin
        y[..., :half], y[..., half:rot] = z.real, z.imag
        res.append(y)
    return res + [s["q"][..., D:].double()] if case["gate"] else res


def _exact_read(s):
    fmt, hkv = s["case"]["kv"], s["case"]["kv_heads"]
    signs = torch.tensor(SIGNS, device="cuda").double()
    res = []
    for slab in (s["k"], s["v"]):
        parts = []
        for r, total in enumerate(s["total"]):
            heads = []
            for h in range(hkv):
                x = _elements64(_head_rows(slab, s["table"], r, total, h), fmt)
                heads.append(_transform64(x) * signs if fmt == "tq4" else x)
            parts.append(torch.cat(heads, 1))
        res.append(torch.cat(parts))
    return res
