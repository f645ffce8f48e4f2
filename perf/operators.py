"""The cache, attention and scoring operators, as measurable cases.

The sizes are those of the repository's own configurations (a 27B-class layer of
48 query and 8 KV heads of 128, a vocabulary of 151936) and generic ones around
them. The operations are the ones a decoder needs between its projections and
behind its output head:

    append     write new tokens' K and V into a quantised paged cache, and
               read what it now holds for them
    read       read tokens of the cache back (a session's export, a copy)
    attention  attention of new queries over the cache: one token a sequence,
               the few of a speculative verification, whole prompts
    logprobs   log probabilities of given tokens, the entropy, the top alternatives

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) cache bytes, queries, logits, output buffers
    run(state)          one pass: the plain form, or nuclis_amd.Backend where `own`
    work(case)          bytes and flops the pass cannot do without
    exact(case, seed)   what run returns, in float64

The cache's bytes (both forms read the same ones) are [pages][kv heads][tiles of
16 tokens]; a tile of head dimension D and b bits is D * (4 b + 2) bytes: K codes,
K scales, V codes, V scales. Values come in groups of 32 along D with one f16
scale. Codes are stored with an offset (8 or 128):
    K codes   [unit][token 16][quarter 4][chunk], the chunk holding for each
              group of the unit the 8 dimensions 8 * quarter ..: at 4 bits one
              32-bit word, dimension 2 p at bit 4 p and 2 p + 1 at bit 16 + 4 p;
              at 8 bits 8 bytes in order
    K scales  [token 16][group]
    V codes   [unit][quad 4][column 16][token of the quad 4][dimensions of the column]
    V scales  [quad 4][group][token of the quad 4]
A unit is 128 dimensions at 4 bits (64 where D is 64) and 64 at 8 bits.
"""
from __future__ import annotations

import math

import torch

own = False

Q_HEADS, KV_HEADS, HEAD_DIM, VOCAB = 48, 8, 128, 151936
DTYPES = {"f32": torch.float32, "f16": torch.float16}
OFFSET = {4: 8, 8: 128}


def listed():
    layer = {"kv_heads": KV_HEADS, "head_dim": HEAD_DIM, "bits": 4, "page": 64}
    attend = dict(layer, op="attention", q_heads=Q_HEADS, ragged=False, window=0)
    return [
        # One decoded token's keys and values of a layer: latency and launches.
        dict(layer, name="append_token", op="append", tokens=1, dtype="f32"),
        # A prompt chunk's keys and values.
        dict(layer, name="append_prompt", op="append", tokens=4096, dtype="f16"),
        # A short session read back, odd count, 8 bits.
        {"name": "read_333_8bit", "op": "read", "kv_heads": 2, "head_dim": 64, "bits": 8, "page": 32, "tokens": 333,
         "dtype": "f32"},
        # A long session's export in f16.
        dict(layer, name="read_session", op="read", tokens=32768, dtype="f16"),
        # One token early in a chat: latency.
        dict(attend, name="decode_300", batch=1, tokens=1, length=300, dtype="f32"),
        # One token far into a long context: the cache's bytes.
        dict(attend, name="decode_32k", batch=1, tokens=1, length=32768, dtype="f32"),
        # A serving batch whose sequences have many different lengths.
        dict(attend, name="decode_batch32", batch=32, tokens=1, length=16384, dtype="f16", ragged=True),
        # Verification of seven drafted tokens, four sequences, 8-bit cache.
        dict(attend, name="verify_8bit", batch=4, tokens=8, length=8191, dtype="f32", bits=8, ragged=True),
        # A whole prompt.
        dict(attend, name="prompt_4096", batch=1, tokens=4096, length=4096, dtype="f16"),
        # Two prompt chunks far into their contexts, wide heads, a sliding window.
        dict(attend, name="chunk_window", batch=2, tokens=1000, length=10000, dtype="f16", q_heads=16, kv_heads=4,
             head_dim=256, page=16, window=4096, ragged=True),
        # One decoded token with twenty alternatives.
        {"name": "logprobs_token", "op": "logprobs", "rows": 1, "count": VOCAB, "top": 20, "dtype": "f32"},
        # A prompt scored after its output head: every token's log probability and five alternatives.
        {"name": "logprobs_prompt", "op": "logprobs", "rows": 1024, "count": VOCAB, "top": 5, "dtype": "f32"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "read", "attention", "attention", "attention", "logprobs"])
    if kind == "logprobs":
        count = rng.choice([VOCAB, 248320, _log(rng, 1000, 262144)])
        return {"op": kind, "rows": min(_log(rng, 1, 1024), (1024 * VOCAB) // count), "count": count,
                "top": rng.choice([0, 1, 5, 20, rng.randint(1, 32)]), "dtype": rng.choice(["f32", "f32", "f16"])}
    head_dim = rng.choice([64, 128, 128, 128, 256])
    case = {"op": kind, "kv_heads": rng.choice([1, 2, 4, 8, 8]), "head_dim": head_dim, "bits": rng.choice([4, 4, 8]),
            "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["f32", "f16"])}
    if kind == "append":
        return dict(case, tokens=_log(rng, 1, 4096))
    if kind == "read":
        return dict(case, tokens=_log(rng, 1, 32768))
    case["q_heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 6, 6, 8])
    case["window"] = rng.choice([0, 0, 0, _log(rng, 64, 4096)])
    form = rng.choice(["decode", "decode", "verify", "prompt"])
    case["batch"] = {"decode": _log(rng, 1, 32), "verify": _log(rng, 1, 8), "prompt": rng.randint(1, 2)}[form]
    case["tokens"] = {"decode": 1, "verify": rng.randint(2, 8), "prompt": _log(rng, 9, 4096)}[form]
    most = {"decode": 32768, "verify": 16384, "prompt": 4096}[form]
    # no more cache than the largest listed batch, nor more products than the largest prompt has
    case["length"] = max(case["tokens"], _log(rng, 16, min(most, 16 * 16384 // case["batch"])))
    if case["tokens"] * case["batch"] * case["q_heads"] * case["length"] * head_dim > 4096 * 4096 * Q_HEADS * HEAD_DIM:
        case["q_heads"] = case["kv_heads"]
        case["tokens"] = min(case["tokens"], 2048)
        case["length"] = min(case["length"], 4096)
    case["ragged"] = case["batch"] > 1 and rng.random() < 0.7
    return case


def _lengths(case):
    """Tokens the sequences hold and bring: spread down to an eighth and to a half where ragged."""
    b, most, new = case["batch"], case["length"], case["tokens"]
    if not case["ragged"] or b == 1:
        return [most] * b, [new] * b
    held = [most - i * (most - most // 8) // (b - 1) for i in range(b)]
    brought = [max(1, new - i * (new // 2) // (b - 1)) for i in range(b)]
    return [max(n, t) for n, t in zip(held, brought)], brought


# -- the cache's format: values, codes and bytes ---------------------------------


def _geometry(case):
    d, bits = case["head_dim"], case["bits"]
    chunk = min(16, d * bits // 32)
    return d, bits, chunk, d * bits // (32 * chunk), 2 * d * bits, d * (4 * bits + 2)


def _tiles(case, cache):
    return cache.view(-1, case["kv_heads"], case["page"] // 16, _geometry(case)[5])


def _planes(case, tiles):
    """Views of the tiles' four parts; `tiles` ends in a tile's bytes."""
    d, bits, chunk, units, codes, _ = _geometry(case)
    half = codes + d
    return (tiles[..., :codes].unflatten(-1, (units, 16, 4, chunk)),
            tiles[..., codes:half].view(torch.float16).unflatten(-1, (16, d // 32)),
            tiles[..., half:half + codes].unflatten(-1, (units, 4, 16, 4, chunk // 4)),
            tiles[..., half + codes:].view(torch.float16).unflatten(-1, (4, d // 32, 4)))


def _quantise(bits, x):
    """x [..., D] in float32 -> codes (with their offset, uint8) and f16 scales."""
    g = x.unflatten(-1, (-1, 32))
    high, low = g.amax(-1), g.amin(-1)
    if bits == 4:
        most = torch.where(high >= -low, high, low)
        d = (most * -0.125).clamp(-2720, 2720).to(torch.bfloat16).to(torch.float16)
    else:
        step = torch.maximum(high, -low) / 127
        step = ((step.view(torch.int32) + 0xfffff) & ~0xfffff).view(torch.float32)  # up to 4 significant bits
        d = step.clamp(max=56).to(torch.float16)
    wide = d.float().unsqueeze(-1)
    q = torch.where(wide == 0, 0, torch.round(g / torch.where(wide == 0, 1, wide)))
    q = q.clamp(-8, 7) if bits == 4 else q.clamp(-127, 127)
    return (q + OFFSET[bits]).to(torch.uint8).flatten(-2), d


def _pack_k(case, q):
    """Codes [..., D] -> [..., unit, quarter, chunk bytes]."""
    _, bits, chunk, units, _, _ = _geometry(case)
    q = q.unflatten(-1, (units, -1, 4, 8)).transpose(-3, -2)  # unit, quarter, group, 8
    if bits == 4:
        q = q.unflatten(-1, (4, 2)).transpose(-2, -1)          # the even ones low, the odd ones high
        q = q.unflatten(-1, (2, 2))
        q = q[..., 0] | q[..., 1] << 4
        return q.flatten(-3)
    return q.flatten(-2)


def _unpack_k(case, b):
    _, bits, _, _, _, _ = _geometry(case)
    if bits == 4:
        b = b.unflatten(-1, (-1, 2, 2))                        # group, even or odd, two bytes
        b = torch.stack([b & 15, b >> 4], -1).flatten(-2)      # .., 4 of a kind
        b = b.transpose(-2, -1).flatten(-2)                    # .., group, 8
    else:
        b = b.unflatten(-1, (-1, 8))
    return b.transpose(-3, -2).flatten(-4)


def _pack_v(case, q):
    """Codes [..., D] -> [..., unit, column, bytes]."""
    _, bits, _, units, _, _ = _geometry(case)
    q = q.unflatten(-1, (units, 16, -1))
    if bits == 4:
        q = q.unflatten(-1, (-1, 2))
        q = q[..., 0] | q[..., 1] << 4
    return q


def _unpack_v(case, b):
    if case["bits"] == 4:
        b = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    return b.flatten(-3)


def _values(bits, codes, scales):
    return ((codes.float() - OFFSET[bits]).unflatten(-1, (-1, 32)) * scales.float().unsqueeze(-1)).flatten(-2)


def _write(case, cache, k, v, slots):
    page, tile, token = slots // case["page"], slots % case["page"] // 16, slots % 16
    kc, ks, vc, vs = _planes(case, _tiles(case, cache))
    codes, scales = _quantise(case["bits"], k.float())
    kc[page, :, tile, :, token] = _pack_k(case, codes)
    ks[page, :, tile, token] = scales
    codes, scales = _quantise(case["bits"], v.float())
    vc[page, :, tile, :, token // 4, :, token % 4] = _pack_v(case, codes)
    vs[page, :, tile, token // 4, :, token % 4] = scales


def _read(case, cache, slots):
    page, tile, token = slots // case["page"], slots % case["page"] // 16, slots % 16
    kc, ks, vc, vs = _planes(case, _tiles(case, cache))
    k = _values(case["bits"], _unpack_k(case, kc[page, :, tile, :, token]), ks[page, :, tile, token])
    v = _values(case["bits"], _unpack_v(case, vc[page, :, tile, :, token // 4, :, token % 4]),
                vs[page, :, tile, token // 4, :, token % 4])
    return k, v


# -- what a user has in hand -------------------------------------------------------


def _projected(case, tokens, gen):
    """Keys and values as projections give them: a few channels larger, heads of different sizes."""
    shape = (tokens, case["kv_heads"], case["head_dim"])
    x = torch.randn(2, *shape, device="cuda", generator=gen)
    x *= torch.exp(0.4 * torch.randn(2, 1, *shape[1:], device="cuda", generator=gen))
    return x[0], x[1]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        rows, count, top = case["rows"], case["count"], case["top"]
        logits = torch.randn(rows, count, device="cuda", generator=gen) * 2.5
        peak = torch.randint(count, (rows, 8), device="cuda", generator=gen)
        logits.scatter_add_(1, peak, 8 + 2 * torch.randn(rows, 8, device="cuda", generator=gen))
        logits[:, torch.randint(count, (count // 100,), device="cuda", generator=gen)] = -math.inf  # not allowed here
        targets = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.7, peak[:, 0],
                              torch.randint(count, (rows,), device="cuda", generator=gen)).int()
        return {"case": case, "logits": logits.to(dtype), "targets": targets,
                "logprobs": torch.empty(rows, device="cuda"), "entropy": torch.empty(rows, device="cuda"),
                "top_ids": torch.empty(rows, top, dtype=torch.int32, device="cuda"),
                "top_logprobs": torch.empty(rows, top, device="cuda")}
    page, tile_bytes = case["page"], _geometry(case)[5]
    held, brought = _lengths(case) if case["op"] == "attention" else ([case["tokens"]], [0])
    # a read starts in the middle of a page, as after a shared prefix
    first = 0 if case["op"] == "attention" else 5
    need = [-(-(n + first) // page) for n in held]
    pages = sum(need) + 3
    order = torch.randperm(pages, device="cuda", generator=gen)
    cache = torch.zeros(pages * case["kv_heads"] * (page // 16) * tile_bytes, dtype=torch.uint8, device="cuda")
    state = {"case": case, "cache": cache, "pages": pages}
    for piece in torch.arange(pages * page, device="cuda").split(16384):
        _write(case, cache, *_projected(case, len(piece), gen), piece)
    if case["op"] != "attention":
        at = torch.arange(first, first + case["tokens"], device="cuda")
        state["slots"] = order[at // page] * page + at % page
        if case["op"] == "append":
            state["k"], state["v"] = (t.to(dtype) for t in _projected(case, case["tokens"], gen))
        shape = (case["tokens"], case["kv_heads"], case["head_dim"])
        out = torch.float32 if case["op"] == "append" else dtype
        state["k_out"], state["v_out"] = (torch.empty(shape, dtype=out, device="cuda") for _ in range(2))
        return state
    table = torch.zeros(len(held), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0] + brought).cumsum(0).int().cuda()
    q = torch.randn(sum(brought), case["q_heads"], case["head_dim"], device="cuda", generator=gen) * 1.5
    return dict(state, table=table, lengths=torch.tensor(held, dtype=torch.int32).cuda(), starts=starts,
                q=q.to(dtype), out=torch.empty(q.shape, dtype=dtype, device="cuda"), total=sum(brought),
                max_tokens=max(brought), max_length=max(held))


# -- the plain forms ---------------------------------------------------------------


def _plain_attention(s):
    case, table, lengths, starts = s["case"], s["table"], s["lengths"].long(), s["starts"].long()
    batch, heads, kv, d = len(lengths), case["q_heads"], case["kv_heads"], case["head_dim"]
    tiles = _tiles(case, s["cache"])[table.long()].transpose(1, 2).flatten(2, 3)  # batch, kv head, tile, bytes
    kc, ks, vc, vs = _planes(case, tiles)
    # one token a row: [batch, kv, tile, 16, ...]
    k = _values(case["bits"], _unpack_k(case, kc.transpose(3, 4)), ks).flatten(2, 3)
    v = _values(case["bits"], _unpack_v(case, vc.permute(0, 1, 2, 4, 6, 3, 5, 7).flatten(3, 4)),
                vs.transpose(-2, -1).flatten(3, 4)).flatten(2, 3)
    k, v = k[:, :, :s["max_length"]], v[:, :, :s["max_length"]]
    new = starts[1:] - starts[:-1]
    row = torch.arange(s["max_tokens"], device="cuda")
    at = torch.minimum(starts[:-1, None] + row, starts[1:, None] - 1)
    q = s["q"].float()[at].unflatten(2, (kv, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # batch, kv, row x group, d
    scores = torch.matmul(q, k.transpose(-2, -1).contiguous()) * d ** -0.5
    position = (lengths - new)[:, None] + row
    j = torch.arange(k.shape[2], device="cuda")
    seen = j <= position[..., None]
    if case["window"]:
        seen &= j > position[..., None] - case["window"]
    seen = seen.repeat_interleave(heads // kv, 1).unsqueeze(1)  # batch, 1, row x group, token
    scores = torch.where(seen, scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
    o = o.unflatten(2, (s["max_tokens"], -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # batch, row, head, d
    sequence = torch.repeat_interleave(torch.arange(batch, device="cuda"), new, output_size=s["total"])
    return o[sequence, torch.arange(s["total"], device="cuda") - starts[sequence]].to(s["q"].dtype)


def _plain_logprobs(s):
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    shifted = x - m
    e = torch.exp(shifted)
    z = e.sum(-1)
    entropy = torch.log(z) - torch.where(e > 0, e * shifted, 0).sum(-1) / z
    lse = torch.log(z).unsqueeze(-1) + m
    values, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    top = s["case"]["top"]
    return {"logprobs": (x.gather(1, s["targets"].long()[:, None]) - lse)[:, 0], "entropy": entropy,
            "top_ids": ids[:, :top].int(), "top_logprobs": values[:, :top] - lse}


_handle = None


def _own(s):
    global _handle
    import nuclis_amd as nq
    if _handle is None:
        _handle = nq.Backend(0)
    case, b = s["case"], _handle
    if case["op"] == "logprobs":
        b.logprobs(s["logits"], s["targets"], s["logprobs"], s["entropy"], s["top_ids"], s["top_logprobs"])
        return {n: s[n] for n in ("logprobs", "entropy", "top_ids", "top_logprobs")}
    cache = nq.KVCache(case["bits"], s["pages"], case["page"], case["kv_heads"], case["head_dim"], s["cache"])
    if case["op"] == "attention":
        b.cache_attention(cache, s["q"], s["out"], s["table"], s["lengths"],
                          starts=s["starts"] if case["ragged"] else None, window=case["window"],
                          max_tokens=s["max_tokens"], max_length=s["max_length"])
        return s["out"]
    if case["op"] == "append":
        b.cache_write(cache, s["k"], s["v"], s["slots"])
    b.cache_read(cache, s["slots"], s["k_out"], s["v_out"])
    return {"k": s["k_out"], "v": s["v_out"]}


def run(s):
    if own:
        return _own(s)
    op = s["case"]["op"]
    if op == "attention":
        return _plain_attention(s)
    if op == "logprobs":
        return _plain_logprobs(s)
    if op == "append":
        _write(s["case"], s["cache"], s["k"], s["v"], s["slots"])
    k, v = _read(s["case"], s["cache"], s["slots"])
    return {"k": k.to(s["k_out"].dtype), "v": v.to(s["v_out"].dtype)}


# -- what a pass needs, and what it should give --------------------------------------


def work(case):
    size = 2 if case["dtype"] == "f16" else 4
    if case["op"] == "logprobs":
        rows, count = case["rows"], case["count"]
        return {"bytes": rows * (count * size + 4 + 8 + 8 * case["top"]), "flops": 6 * rows * count}
    d, heads = case["head_dim"], case["kv_heads"]
    token = heads * d * (4 * case["bits"] + 2) // 16
    if case["op"] != "attention":
        values = 2 * heads * d * case["tokens"]
        if case["op"] == "read":
            return {"bytes": case["tokens"] * (token + 8) + values * size, "flops": values}
        return {"bytes": case["tokens"] * (2 * token + 8) + values * (size + 4), "flops": 5 * values}
    held, brought = _lengths(case)
    window = case["window"] or max(held)
    cached = pairs = 0
    for n, new in zip(held, brought):
        cached += min(n, new - 1 + window)
        # rows see min(position + 1, window) tokens
        full = max(0, min(new, n - window + 1))
        rest = new - full
        pairs += full * window + rest * (n - new) + rest * (rest + 1) // 2
    return {"bytes": cached * token + 2 * sum(brought) * case["q_heads"] * d * size,
            "flops": 4 * pairs * case["q_heads"] * d}


def _places(case):
    """Where a tile holds each (token, dimension): byte, bit and scale of K, and of V."""
    d, bits, chunk, units, codes, _ = _geometry(case)
    t, c = torch.arange(16)[:, None], torch.arange(d)[None, :]
    wide = d // units
    u, g, h, e = c // wide, c % wide // 32, c % 32 // 8, c % 8
    base = ((u * 16 + t) * 4 + h) * chunk + g * bits
    k = (base + (e % 2 * 2 + e // 4 if bits == 4 else e), e // 2 % 2 * 4 if bits == 4 else 0 * e,
         codes + 2 * (t * (d // 32) + c // 32))
    per = wide // 16
    n, j = c % wide // per, c % per
    base = (((u * 4 + t // 4) * 16 + n) * 4 + t % 4) * (chunk // 4)
    half = codes + d
    v = (half + base + (j // 2 if bits == 4 else j), j % 2 * 4 if bits == 4 else 0 * j,
         half + codes + 2 * ((t // 4 * (d // 32) + c // 32) * 4 + t % 4))
    return [[(x + 0 * (t + c)).cuda() for x in p] for p in (k, v)]


def _decoded(case, tiles, place):
    """float64 values [..., 16, D] of tiles [..., bytes]."""
    byte, bit, scale = place
    code = tiles[..., byte].int() >> bit & (15 if case["bits"] == 4 else 255)
    raw = tiles[..., scale].int() | tiles[..., scale + 1].int() << 8
    sign, exponent, fraction = raw >> 15, raw >> 10 & 31, (raw & 1023).double()
    size = torch.where(exponent == 0, fraction * 2.0 ** -24,
                       (1024 + fraction) * torch.exp2((exponent - 25).double()))
    return (code - OFFSET[case["bits"]]) * torch.where(sign == 1, -size, size)


def _exact_values(bits, x):
    """What a cache stands for after x [..., D] was written, in float64."""
    g = x.double().unflatten(-1, (-1, 32))
    if bits == 4:
        first = g.amax(-1)
        first = torch.where(first >= -g.amin(-1), first, g.amin(-1)) / -8
        fraction, exponent = torch.frexp(first.clamp(-2720, 2720))
        d = torch.round(fraction * 256) * torch.exp2((exponent - 8).double())
        low, high = -8, 7
    else:
        fraction, exponent = torch.frexp(g.abs().amax(-1) / 127)
        d = (torch.ceil(fraction * 16) * torch.exp2((exponent - 4).double())).clamp(max=56)
        low, high = -127, 127
    d = torch.where(d.abs() < 2.0 ** -14, torch.round(d * 2.0 ** 24) * 2.0 ** -24, d).unsqueeze(-1)
    return (torch.where(d == 0, 0, torch.round(g / torch.where(d == 0, 1, d)).clamp(low, high)) * d).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        x = s["logits"].double()
        p = torch.log_softmax(x, -1)
        entropy = -(torch.exp(p) * p.clamp(min=-1e4)).sum(-1)
        values = p.topk(case["top"], -1).values if case["top"] else p[:, :0]
        return {"logprobs": p.gather(1, s["targets"].long()[:, None])[:, 0], "entropy": entropy, "top_ids": None,
                "top_logprobs": values}
    if case["op"] == "append":
        return {"k": _exact_values(case["bits"], s["k"]), "v": _exact_values(case["bits"], s["v"])}
    tiles = _tiles(case, s["cache"])
    k_place, v_place = _places(case)
    if case["op"] == "read":
        page, tile, token = s["slots"] // case["page"], s["slots"] % case["page"] // 16, s["slots"] % 16
        rows = torch.arange(len(token), device="cuda")
        picked = tiles[page, :, tile]
        parts = {"k": [], "v": []}
        for r in rows.split(2048):
            for name, place in (("k", k_place), ("v", v_place)):
                whole = _decoded(case, picked[r], place)
                parts[name].append(whole[torch.arange(len(r), device="cuda"), :, token[r]])
        return {name: torch.cat(x) for name, x in parts.items()}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["q_heads"] // case["kv_heads"]
    held, brought = _lengths(case)
    at = 0
    for b, (n, new) in enumerate(zip(held, brought)):
        mine = tiles[s["table"][b].long()]
        position = torch.arange(n - new, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")[None, :]
        seen = (j <= position) & (j > position - (case["window"] or n + 1))
        for head in range(case["kv_heads"]):
            k = _decoded(case, mine[:, head], k_place).flatten(0, 2)[:n]
            v = _decoded(case, mine[:, head], v_place).flatten(0, 2)[:n]
            kt = k.t().contiguous()
            for h in range(head * group, (head + 1) * group):
                x = s["q"][at:at + new, h].double() @ kt / math.sqrt(case["head_dim"])
                out[at:at + new, h] = torch.softmax(x.masked_fill(~seen, -math.inf), -1) @ v
        at += new
    return out
