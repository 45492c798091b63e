"""The cases that the paged-serving operators are measured on, and their plain forms.

Three operators that a continuous-batching server runs around a 4-bit key/value cache with pages:

* append: rotate the queries and keys of new tokens by their positions and append keys and values to the paged cache (and
  read back, in 16 bits, what the cache then holds for the tokens that the call changed);
* attend: one query token per sequence over the paged cache, every sequence with a length of its own;
* prompt: causal attention of whole prompts (or chunks of them), packed one behind the other, with grouped heads.

The cache.  Of a sequence of L tokens the first `sink` ones and the last `recent` to `recent + 31` ones are held in 16 bits
in the sequence's slot (a ring of `recent + 32` rows behind the sink's rows); the tokens between them, in tiles of 32, are
held in 4 bits: symmetric codes -7..7 (stored with 8 added), one scale in the model's type per token and 32 channels for
keys, per channel and 32 tokens for values.  A scale is the group's largest magnitude divided by 7; a group that holds a
value that is not finite has a NaN for a scale.  A tile of one head is one block of 4608 bytes:

    keys' codes    32-bit words [j 4][i 8][l 4][g 4]; nibble n: token 8j + i, channel 32g + 8l + n
    keys' scales   [i 8][j 4][g 4]
    values' codes  32-bit words [p 4][i 8][l 4][m 2][h 2]; nibble n: channel 16i + 4p + 2m + h, token 8(n % 4) + 2l + n // 4
    values' scales [channel 128]

and `pages` is [pages, heads, tiles of a page, 4608] bytes; a row of `table` names a sequence's pages in order.
"""
import math

import numpy as np
import torch

own = False

D, TILE, BLOCK = 128, 32, 4608
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------- cases ---
def listed():
    return [
        # one request decodes alone: the append of a token is latency (4-bit cache, sink 32, window 96; 32 / 8 heads)
        {"name": "append_step_b1", "op": "append", "b": 1, "lo": 4095, "hi": 4095, "new": 1, "mix": 1, "hq": 32, "hkv": 8,
         "dtype": "fp16", "page": 64, "sink": 32, "recent": 96, "interleaved": False},
        # a full decode batch of mixed lengths, 64 / 8 heads (the 70B attention shape)
        {"name": "append_step_b128", "op": "append", "b": 128, "lo": 100, "hi": 9000, "new": 1, "mix": 2, "hq": 64, "hkv": 8,
         "dtype": "bf16", "page": 64, "sink": 32, "recent": 96, "interleaved": False},
        # the prompts of a scheduling step, ragged and odd, quantized as they come
        {"name": "append_prompts", "op": "append", "b": 13, "lo": 37, "hi": 4000, "new": 0, "mix": 3, "hq": 32, "hkv": 8,
         "dtype": "fp16", "page": 128, "sink": 32, "recent": 96, "interleaved": False},
        # one long prompt of a model that rotates neighbouring channels, without a sink
        {"name": "append_prompt_16k", "op": "append", "b": 1, "lo": 16384, "hi": 16384, "new": 0, "mix": 4, "hq": 40, "hkv": 8,
         "dtype": "bf16", "page": 64, "sink": 0, "recent": 32, "interleaved": True},
        # the smallest decode call: one sequence of a few thousand tokens
        {"name": "attend_b1_4k", "op": "attend", "b": 1, "lo": 4096, "hi": 4096, "mix": 5, "hq": 32, "hkv": 8, "dtype": "fp16",
         "page": 64, "sink": 32, "recent": 96},
        # one long sequence: the work is split over its tokens
        {"name": "attend_b1_32k", "op": "attend", "b": 1, "lo": 32768, "hi": 32768, "mix": 6, "hq": 32, "hkv": 8, "dtype": "fp16",
         "page": 64, "sink": 32, "recent": 96},
        # a serving batch of every length from one token on, five query heads to a key head
        {"name": "attend_ragged_b96", "op": "attend", "b": 96, "lo": 1, "hi": 20000, "mix": 7, "hq": 40, "hkv": 8, "dtype": "bf16",
         "page": 32, "sink": 32, "recent": 64},
        # the batch of 32 at 32768 tokens that the framework's benchmark decodes
        {"name": "attend_b32_32k", "op": "attend", "b": 32, "lo": 32768, "hi": 32768, "mix": 8, "hq": 32, "hkv": 8, "dtype": "fp16",
         "page": 64, "sink": 32, "recent": 96},
        # long contexts of the 70B attention shape, eight query heads to a key head
        {"name": "attend_b8_128k", "op": "attend", "b": 8, "lo": 131072, "hi": 131072, "mix": 9, "hq": 64, "hkv": 8, "dtype": "bf16",
         "page": 128, "sink": 0, "recent": 32},
        # short requests, some of a single token: latency
        {"name": "prompt_short", "op": "prompt", "b": 16, "lo": 1, "hi": 300, "past": 0, "mix": 10, "hq": 32, "hkv": 8, "dtype": "fp16",
         "causal": True},
        # one prompt of 8192 tokens, the context of the benchmark's full decode step
        {"name": "prompt_8k", "op": "prompt", "b": 1, "lo": 8192, "hi": 8192, "past": 0, "mix": 11, "hq": 32, "hkv": 8, "dtype": "bf16",
         "causal": True},
        # chunks of long prompts over the keys that came before them, odd lengths, eight query heads to a key head
        {"name": "prompt_chunks", "op": "prompt", "b": 3, "lo": 2000, "hi": 2999, "past": 8111, "mix": 12, "hq": 64, "hkv": 8,
         "dtype": "fp16", "causal": True},
    ]


def draw(rng):
    spread = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    hkv = rng.choice([1, 2, 4, 8])
    c = {"op": rng.choice(["append", "attend", "prompt"]), "mix": rng.randrange(1 << 30), "hkv": hkv,
         "hq": hkv * rng.choice([1, 2, 3, 4, 5, 7, 8]), "dtype": rng.choice(["fp16", "bf16"])}
    if c["op"] == "prompt":
        hi = spread(1, 6000)
        c |= {"b": max(1, min(spread(1, 24), 9000 // hi)), "lo": max(1, spread(1, hi)), "hi": hi, "causal": rng.random() < 0.85,
              "past": rng.choice([0, spread(1, 3000)])}
        return c
    c |= {"page": rng.choice([32, 64, 128, 256]), "sink": rng.choice([0, 32, 64]), "recent": rng.choice([0, 32, 96])}
    if c["op"] == "attend":
        hi = spread(1, 100000)
        c |= {"b": max(1, min(spread(1, 128), 1000000 // hi)), "lo": spread(1, hi), "hi": hi}
    elif rng.random() < 0.5:
        hi = spread(1, 20000)
        c |= {"b": spread(1, 128), "lo": spread(1, hi), "hi": hi, "new": 1, "interleaved": rng.random() < 0.3}
    else:
        hi = spread(1, 16000)
        c |= {"b": max(1, min(spread(1, 32), 24000 // hi)), "lo": spread(1, hi), "hi": hi, "new": 0,
              "interleaved": rng.random() < 0.3}
    return c


def lengths(case):
    """The sequences' lengths: spread over their logarithm from lo to hi, the longest among them."""
    r = np.random.RandomState(case["mix"] % (1 << 31))
    n = np.exp(r.uniform(math.log(case["lo"]), math.log(case["hi"] + 0.999), case["b"])).astype(np.int64)
    n[-1] = case["hi"]
    return n


def packed(n, case):
    """How many tokens of a sequence of n are held in 4 bits."""
    return np.maximum(0, n - case["sink"] - case["recent"]) // TILE * TILE


def spans(case):
    """append: lengths before, tokens that come, first token and number of tokens read back."""
    n = lengths(case)
    if case["new"]:  # a decode step: one token each; the window it changed is read back
        first = np.maximum(0, n + 1 - (case["recent"] + TILE))
        return n, np.ones_like(n), first, n + 1 - first
    return np.zeros_like(n), n, np.zeros_like(n), n  # prompts: all is read back


def work(case):
    hq, hkv, n = case["hq"], case["hkv"], lengths(case)
    if case["op"] == "prompt":
        q, k = n, n + case["past"]
        pairs = (q * case["past"] + q * (q + 1) // 2).sum() if case["causal"] else (q * k).sum()
        return {"bytes": float(4 * D * (q.sum() * hq + k.sum() * hkv)), "flops": float(4 * D * hq * pairs)}
    block = BLOCK // TILE
    if case["op"] == "attend":
        low = packed(n, case)
        return {"bytes": float((low * hkv * block + (n - low) * hkv * 4 * D).sum() + 4 * D * hq * case["b"]),
                "flops": float(4 * D * hq * n.sum())}
    was, new, _, count = spans(case)
    low = packed(was + new, case) - packed(was, case)  # tokens that the call quantizes
    t = int(new.sum())
    again = 0 if case["new"] == 0 else int(low.sum())  # those of them that come out of the ring
    moved = 4 * D * (hq + hkv) * t + 2 * D * hkv * t  # q and k in and out, v in
    moved += hkv * block * int(low.sum()) + 4 * D * hkv * (int(new.sum() - low.sum()) + 2 * again)
    moved += hkv * (4 * D) * int(count.sum()) + 4 * D * t  # read back; cosines and sines
    return {"bytes": float(moved), "flops": float(6 * D * (hq + hkv) * t + 8 * D * hkv * int(low.sum()))}


# ---------------------------------------------------------------- the cache ---
def quantize(x, dim):
    """Codes and scales of x [..., groups of 32 along dim]: scale = amax / 7 and code = x / scale, each rounded to x's type."""
    f = x.float()
    top = f.abs().amax(dim, keepdim=True)
    scale = (top / torch.full_like(top, 7.0)).to(x.dtype)  # a divisor in a tensor: a true division
    ratio = (f.abs() / scale.float()).to(x.dtype).float()
    code = torch.nan_to_num(ratio, nan=0.0, posinf=7.0).clamp(0, 7).round() * f.sign()
    good = torch.isfinite(top)
    return torch.where(good, code, 0.0), torch.where(good, scale, float("nan"))


def pack(k, v):
    """Tiles k, v [..., 32 tokens, 128] to blocks [..., 4608] bytes."""
    at = k.shape[:-2]
    r = len(at)
    lead = list(range(r))
    shift = 4 * torch.arange(8, device=k.device)
    kc, ks = quantize(k.reshape(*at, 32, 4, 32), r + 2)  # token, g, channel of the group
    w = (kc + 8).long().reshape(*at, 4, 8, 4, 4, 8)  # j i g l n
    w = (w << shift).sum(-1).permute(*lead, r, r + 1, r + 3, r + 2).reshape(*at, 512)
    ks = ks.reshape(*at, 4, 8, 4).transpose(r, r + 1).reshape(*at, 128)
    vc, vs = quantize(v, r)
    u = (vc + 8).long().reshape(*at, 4, 4, 2, 8, 4, 2, 2)  # token: n%4, l, n//4; channel: i p m h
    u = u.permute(*lead, r + 4, r + 3, r + 1, r + 5, r + 6, r + 2, r)  # p i l m h | n//4 n%4
    u = (u.reshape(*at, 4, 8, 4, 2, 2, 8) << shift).sum(-1).reshape(*at, 512)
    whole = lambda x: torch.where(x >= 1 << 31, x - (1 << 32), x).int().contiguous().view(torch.uint8)  # noqa: E731
    return torch.cat([whole(w), ks.contiguous().view(torch.uint8), whole(u), vs.reshape(*at, D).contiguous().view(torch.uint8)], -1)


def unpack(blocks, dtype):
    """Blocks [..., 4608] to the values they stand for, in 32 bits: k, v [..., 32, 128]."""
    at = blocks.shape[:-1]
    r = len(at)
    lead = list(range(r))
    shift = 4 * torch.arange(8, device=blocks.device, dtype=torch.int32)
    part = lambda lo, n, t: blocks[..., lo:lo + n].contiguous().view(t)  # noqa: E731
    nib = lambda x: (((x.unsqueeze(-1) >> shift) & 15) - 8).float()  # noqa: E731
    k = nib(part(0, 2048, torch.int32)).reshape(*at, 4, 8, 4, 4, 8)  # j i l g n
    k = k.transpose(r + 2, r + 3).reshape(*at, 32, 4, 32)
    ks = part(2048, 256, dtype).float().reshape(*at, 8, 4, 4).transpose(r, r + 1).reshape(*at, 32, 4, 1)
    v = nib(part(2304, 2048, torch.int32)).reshape(*at, 4, 8, 4, 2, 2, 2, 4)  # p i l m h n//4 n%4
    v = v.permute(*lead, r + 6, r + 2, r + 5, r + 1, r, r + 3, r + 4).reshape(*at, 32, D)
    vs = part(4352, 256, dtype).float().reshape(*at, 1, D)
    return (k * ks).reshape(*at, 32, D), v * vs


def cache(case, n, r, gen, grow):
    """The cache of sequences of n tokens with room for `grow` more each: keys have channels of very different size."""
    dt, h, b, page = TYPES[case["dtype"]], case["hkv"], case["b"], case["page"]
    ring = case["recent"] + TILE
    need = -(-packed(n + grow, case) // page)
    width = max(1, int(need.max()))
    total = max(1, int(need.sum()))
    pages = torch.empty((total, h, page // TILE, BLOCK), dtype=torch.uint8, device="cuda")
    size = torch.exp(torch.randn((h, 1, D), generator=gen, device="cuda"))
    if packed(n, case).any():
        some = max(1, (1 << 28) // (h * page * D))
        for at in range(0, total, some):
            shape = (min(some, total - at), h, page // TILE, TILE, D)
            k = torch.randn(shape, generator=gen, device="cuda") * size[:, None]
            v = torch.randn(shape, generator=gen, device="cuda")
            pages[at:at + some] = pack(k.to(dt), v.to(dt))
    else:
        pages.zero_()
    table = np.full((b, width), -1, np.int32)
    table[np.arange(width)[None] < need[:, None]] = r.permutation(total)[:int(need.sum())]
    dense = (b + 3, h, case["sink"] + ring, D)  # more slots than sequences, as a server has
    return {"pages": pages, "dense_k": (torch.randn(dense, generator=gen, device="cuda") * size).to(dt),
            "dense_v": torch.randn(dense, generator=gen, device="cuda").to(dt), "size": size, "sink": case["sink"],
            "recent": case["recent"], "table": torch.from_numpy(table).cuda(),
            "slots": torch.from_numpy(r.permutation(b + 3)[:b].astype(np.int32)).cuda()}


def starts_of(n):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).cuda()


def prepare(case, seed):
    r = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, hq, hkv = TYPES[case["dtype"]], case["hq"], case["hkv"]
    n = lengths(case)
    if case["op"] == "prompt":
        k_n = n + case["past"]
        q = torch.randn((int(n.sum()), hq, D), generator=gen, device="cuda")
        kv = torch.randn((2, int(k_n.sum()), hkv, D), generator=gen, device="cuda")
        return {"op": "prompt", "q": q.to(dt), "k": kv[0].to(dt), "v": kv[1].to(dt), "cu_q": starts_of(n), "cu_k": starts_of(k_n),
                "causal": case["causal"], "most_q": int(n.max()), "most_k": int(k_n.max())}
    if case["op"] == "attend":
        s = cache(case, n, r, gen, 0)
        return s | {"op": "attend", "lens": torch.from_numpy(n.astype(np.int32)).cuda(), "most": int(n.max()),
                    "q": torch.randn((case["b"], hq, D), generator=gen, device="cuda").to(dt)}
    was, new, first, count = spans(case)
    s = cache(case, was, r, gen, new)
    # the projection's output, q, k and v side by side, and the rotation's table
    qkv = torch.randn((int(new.sum()), hq + 2 * hkv, D), generator=gen, device="cuda")
    qkv[:, hq:hq + hkv] *= s["size"].transpose(0, 1)
    qkv = qkv.to(dt)
    angle = torch.arange(int((was + new).max()), device="cuda").double()[:, None] * 500000.0 ** -(
        torch.arange(0, D, 2, device="cuda").double() / D)
    return s | {"op": "append", "q": qkv[:, :hq], "k": qkv[:, hq:hq + hkv], "v": qkv[:, hq + hkv:], "cos": angle.cos().float(),
                "sin": angle.sin().float(), "interleaved": case["interleaved"], "lens": torch.from_numpy(was.astype(np.int32)).cuda(),
                "after": torch.from_numpy((was + new).astype(np.int32)).cuda(), "cu": starts_of(new), "one": bool(case["new"]),
                "first": torch.from_numpy(first.astype(np.int32)).cuda(), "cu_read": starts_of(count), "n_read": int(count.sum())}


# ---------------------------------------------------------- the plain forms ---
def low_of(n, s):
    return (n - s["sink"] - s["recent"]).clamp(min=0) // TILE * TILE


def owner(cu, total):
    """Which sequence each of `total` packed tokens belongs to, and its place there."""
    at = torch.arange(total, device=cu.device)
    b = torch.searchsorted(cu.long(), at, right=True) - 1
    return b, at - cu.long()[b]


def row_of(pos, s):
    """The row of a sequence's slot that holds the token at `pos`."""
    return torch.where(pos < s["sink"], pos, s["sink"] + (pos - s["sink"]) % (s["recent"] + TILE))


def plain_read(s, b, pos, n):
    """What the cache holds for the tokens at `pos` of the sequences `b`, which are n tokens long, in 32 bits: k, v [tokens, heads, 128]."""
    slot, u = s["slots"].long()[b], (pos - s["sink"]).clamp(min=0)
    k, v = (s[x][slot, :, row_of(pos, s)].float() for x in ("dense_k", "dense_v"))
    held = (pos >= s["sink"]) & (pos < s["sink"] + low_of(n, s)[b])
    of = s["pages"].shape[2] * TILE
    page = s["table"].long()[b, (u // of).clamp(max=s["table"].shape[1] - 1)]
    tile = torch.where(held, page * s["pages"].shape[2] + u % of // TILE, -1)
    which, back = torch.unique(tile, return_inverse=True)  # each tile is unpacked once
    blocks = s["pages"][which.clamp(min=0) // s["pages"].shape[2], :, which.clamp(min=0) % s["pages"].shape[2]]
    lk, lv = unpack(blocks, s["dense_k"].dtype)
    held = held[:, None, None]
    return torch.where(held, lk[back, :, u % TILE], k), torch.where(held, lv[back, :, u % TILE], v)


def plain_rotate(x, c, s, interleaved):
    x = x.float()
    c, s = c[:, None], s[:, None]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :D // 2], x[..., D // 2:])
    a, b = a * c - b * s, b * c + a * s
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def plain_append(s):
    dt, k, v = s["q"].dtype, s["k"], s["v"]
    b, i = owner(s["cu"], k.shape[0])
    was, now = s["lens"].long(), s["after"].long()
    pos = was[b] + i
    cos, sin = s["cos"][pos], s["sin"][pos]
    q = plain_rotate(s["q"], cos, sin, s["interleaved"]).to(dt)
    k = plain_rotate(k, cos, sin, s["interleaved"]).to(dt)
    # the tiles that leave the window: their tokens are new, or come out of the ring
    lo, hi = low_of(was, s), low_of(now, s)
    count = (hi - lo) // TILE
    tb, ti = owner(torch.cat([count.new_zeros(1), count.cumsum(0)]), int(count.sum()))
    u = lo[tb] + ti * TILE
    at = (s["sink"] + u)[:, None] + torch.arange(TILE, device=u.device)
    fresh = (at >= was[tb][:, None])[:, None, :, None]
    src = (s["cu"].long()[tb][:, None] + at - was[tb][:, None]).clamp(min=0, max=k.shape[0] - 1)
    slot, row = s["slots"].long()[tb][:, None], row_of(at, s)
    tk = torch.where(fresh, k[src].transpose(1, 2), s["dense_k"][slot, :, row].transpose(1, 2))
    tv = torch.where(fresh, v[src].transpose(1, 2), s["dense_v"][slot, :, row].transpose(1, 2))
    of = s["pages"].shape[2]
    s["pages"][s["table"].long()[tb, u // (of * TILE)], :, u // TILE % of] = pack(tk, tv)
    # the sink's and the window's tokens
    keep = (pos < s["sink"]) | (pos >= s["sink"] + hi[b])
    slot, row = s["slots"].long()[b[keep]], row_of(pos[keep], s)
    s["dense_k"][slot, :, row] = k[keep]
    s["dense_v"][slot, :, row] = v[keep]
    rb, ri = owner(s["cu_read"], s["n_read"])
    rk, rv = plain_read(s, rb, s["first"].long()[rb] + ri, now)
    return {"q": q, "k": k, "cached_k": rk.to(dt), "cached_v": rv.to(dt)}


def plain_attend(s):
    q, n = s["q"].float(), s["lens"].long()
    bsz, hq, hkv, most, sink = q.shape[0], q.shape[1], s["dense_k"].shape[1], s["most"], s["sink"]
    of = s["pages"].shape[2]
    # the 4-bit tokens of all sequences, padded to the longest, then those of the slots
    blocks = s["pages"][s["table"].long().clamp(min=0)].transpose(1, 2).reshape(bsz, hkv, -1, BLOCK)
    tiles = max(0, most - sink - s["recent"]) // TILE
    lk, lv = unpack(blocks[:, :, :tiles], s["dense_k"].dtype)
    lk, lv = lk.reshape(bsz, hkv, -1, D), lv.reshape(bsz, hkv, -1, D)
    slot = s["slots"].long()
    dk, dv = s["dense_k"][slot].float(), s["dense_v"][slot].float()
    rows = torch.arange(dk.shape[2], device=q.device)
    low = low_of(n, s)
    ring = s["recent"] + TILE
    base = sink + low  # the first token of the window
    token = torch.where(rows < sink, rows, base[:, None] + (rows - sink - low[:, None]) % ring)
    seen = torch.cat([torch.arange(lk.shape[2], device=q.device) < low[:, None], token < n[:, None]], 1)
    q = q.reshape(bsz, hkv, hq // hkv, D)
    score = torch.cat([q @ lk.transpose(-1, -2), q @ dk.transpose(-1, -2)], -1) / math.sqrt(D)
    score = score.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    dv = torch.where((token < n[:, None])[:, None, :, None], dv, 0.0)
    out = p[..., :lk.shape[2]] @ lv + p[..., lk.shape[2]:] @ dv
    return {"out": out.reshape(bsz, hq, D).to(s["q"].dtype)}


def plain_prompt(s):
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"].long(), s["cu_k"].long()
    hq, hkv, dev = q.shape[1], k.shape[1], q.device
    nq, nk = cu_q.diff(), cu_k.diff()
    iq, ik = torch.arange(s["most_q"], device=dev), torch.arange(s["most_k"], device=dev)
    in_q, in_k = iq < nq[:, None], ik < nk[:, None]
    at_q = (cu_q[:-1, None] + iq).clamp(max=q.shape[0] - 1)
    at_k = (cu_k[:-1, None] + ik).clamp(max=k.shape[0] - 1)
    qp = q[at_q].float().reshape(len(nq), -1, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4)
    kp = k[at_k].float().permute(0, 2, 3, 1)[:, :, None]
    vp = torch.where(in_k[:, :, None, None], v[at_k].float(), 0.0).permute(0, 2, 1, 3)[:, :, None]
    seen = in_k[:, None] & torch.ones_like(in_q)[:, :, None]
    if s["causal"]:  # the last query sees the last key
        seen = seen & (ik <= (iq + (nk - nq)[:, None])[..., None])
    score = (qp @ kp).mul_(1.0 / math.sqrt(D)).masked_fill_(~seen[:, None, None], float("-inf"))
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    out = (p @ vp).permute(0, 3, 1, 2, 4).reshape(len(nq), -1, hq, D)
    return {"out": out[in_q].to(q.dtype)}


# ----------------------------------------------------------------- one pass ---
def run(s):
    if not own:
        return {"append": plain_append, "attend": plain_attend, "prompt": plain_prompt}[s["op"]](s)
    from innerq_b200.paged import PagedCache
    from innerq_b200.prompt import prompt_attention
    if s["op"] == "prompt":
        return {"out": prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["causal"])}
    c = PagedCache(s["pages"], s["dense_k"], s["dense_v"], s["sink"], s["recent"])
    if s["op"] == "attend":
        return {"out": c.attend(s["q"], s["table"], s["slots"], s["lens"])}
    q, k = c.append(s["q"], s["k"], s["v"], s["table"], s["slots"], s["lens"], None if s["one"] else s["cu"], cos=s["cos"],
                    sin=s["sin"], interleaved=s["interleaved"], return_k=True)
    rk, rv = c.read(s["table"], s["slots"], s["after"], s["first"], s["cu_read"], s["n_read"])
    return {"q": q, "k": k, "cached_k": rk, "cached_v": rv}


# ------------------------------------------------------------- in 64 bits ---
def exact(case, seed):
    s = prepare(case, seed)
    dt = s["q"].dtype
    dev = "cuda"

    if s["op"] == "prompt":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        out = torch.zeros_like(q)
        cq, ck, group = s["cu_q"].tolist(), s["cu_k"].tolist(), q.shape[1] // k.shape[1]
        for b in range(len(cq) - 1):
            nq, nk = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
            for h in range(q.shape[1]):
                kk, vv = k[ck[b]:ck[b + 1], h // group], v[ck[b]:ck[b + 1], h // group]
                for lo in range(0, nq, 2048):
                    hi = min(nq, lo + 2048)
                    logit = torch.einsum("id,jd->ij", q[cq[b] + lo:cq[b] + hi, h], kk) * D ** -0.5
                    if s["causal"]:
                        logit += torch.full((hi - lo, nk), float("-inf"), dtype=torch.float64, device=dev).triu(nk - nq + lo + 1)
                    out[cq[b] + lo:cq[b] + hi, h] = torch.softmax(logit, 1) @ vv
        return {"out": out}

    def decode(block):
        """The tokens of tiles block [..., 4608], token by token as the format's table says, in 64 bits."""
        t = torch.arange(32, device=dev)[:, None]
        d = torch.arange(D, device=dev)[None]
        byte = block.long()
        j, i, g, l, n = t // 8, t % 8, d // 32, d // 8 % 4, d % 8
        word = ((j * 8 + i) * 4 + l) * 4 + g
        kq = (byte[..., word * 4 + n // 2] >> (4 * (n % 2))) % 16 - 8
        number = lambda x: x.contiguous().view(dt).double()  # noqa: E731
        ks = number(block[..., 2048:2304])[..., (i * 4 + j) * 4 + g]
        i, p, m, h, l, n = d // 16, d // 4 % 4, d // 2 % 2, d % 2, t % 8 // 2, t // 8 + 4 * (t % 2)
        word = ((((p * 8 + i) * 4 + l) * 2 + m) * 2 + h)
        vq = (byte[..., 2304 + word * 4 + n // 2] >> (4 * (n % 2))) % 16 - 8
        return kq * ks, vq * number(block[..., 4352:])[..., None, :].expand(vq.shape)

    of, sink, ring = s["pages"].shape[2], s["sink"], s["recent"] + 32
    table, slots = s["table"].cpu().numpy(), s["slots"].tolist()

    if s["op"] == "attend":
        q = s["q"].double()
        hkv = s["dense_k"].shape[1]
        out = torch.zeros_like(q)
        for b, n in enumerate(s["lens"].tolist()):
            low = max(0, n - sink - s["recent"]) // 32 * 32
            tokens = list(range(min(n, sink))) + list(range(sink + low, n))
            rows = [t if t < sink else sink + (t - sink) % ring for t in tokens]
            pages = torch.from_numpy(table[b, :-(-low // (32 * of))].astype(np.int64)).to(dev)
            for h in range(hkv):
                kk, vv = s["dense_k"][slots[b], h, rows].double(), s["dense_v"][slots[b], h, rows].double()
                if low:
                    lk, lv = decode(s["pages"][pages, h].reshape(-1, BLOCK)[:low // 32])
                    kk, vv = torch.cat([lk.reshape(-1, D), kk]), torch.cat([lv.reshape(-1, D), vv])
                hs = slice(h * q.shape[1] // hkv, (h + 1) * q.shape[1] // hkv)
                out[b, hs] = torch.softmax(q[b, hs] @ kk.T / D ** 0.5, -1) @ vv
        return {"out": out}

    # append: the rotation in 64 bits, the cache's tokens from it by the definition
    def turned(x, pos):
        c, w = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
        z = torch.complex(x[..., 0::2].double(), x[..., 1::2].double()) if s["interleaved"] else torch.complex(
            x[..., :64].double(), x[..., 64:].double())
        z = z * torch.complex(c, w)
        return torch.view_as_real(z).flatten(-2) if s["interleaved"] else torch.cat([z.real, z.imag], -1)

    def held(x, axis):
        """What 4 bits leave of tile x, whose groups of 32 run along `axis`."""
        y = x.double().unflatten(axis, (-1, 32))
        step = (y.abs().amax(axis + 1, keepdim=True) / 7).to(dt).double()
        c = torch.round((y.abs() / step).to(dt).double().clamp(max=7))
        return (torch.where(step > 0, c, 0.0) * step * y.sign()).flatten(axis, axis + 1)

    q64, k64, read_k, read_v = [], [], [], []
    lens, cu, first = s["lens"].tolist(), s["cu"].tolist(), s["first"].tolist()
    for b, n in enumerate(lens):
        sl = slice(cu[b], cu[b + 1])
        now = n + cu[b + 1] - cu[b]
        pos = torch.arange(n, now, device=dev)
        q64.append(turned(s["q"][sl], pos))
        k64.append(turned(s["k"][sl], pos))
        new_k, new_v = k64[-1].to(dt), s["v"][sl]
        low, before = (max(0, m - sink - s["recent"]) // 32 * 32 for m in (now, n))
        dk, dv = s["dense_k"][slots[b]].transpose(0, 1), s["dense_v"][slots[b]].transpose(0, 1)
        # the tokens from `base` on, whole tiles, as they were before quantization
        base = first[b] if first[b] < sink else sink + (first[b] - sink) // 32 * 32
        old = torch.arange(base, n, device=dev)
        row = torch.where(old < sink, old, sink + (old - sink) % ring)
        kk, vv = torch.cat([dk[row], new_k]), torch.cat([dv[row], new_v])
        got_k, got_v = kk.double(), vv.double()
        a = max(base, sink)
        done = sink + before  # tiles that were quantized before the call come from the pages
        if done > a:
            u = (a - sink) // 32
            at = torch.arange(u, before // 32, device=dev)
            pg = torch.from_numpy(table[b].astype(np.int64)).to(dev)[at // of]
            lk, lv = decode(s["pages"][pg, :, at % of])
            got_k[a - base:done - base] = lk.transpose(1, 2).flatten(0, 1)
            got_v[a - base:done - base] = lv.transpose(1, 2).flatten(0, 1)
        a = max(a, done)
        if sink + low > a:
            at = slice(a - base, sink + low - base)
            got_k[at], got_v[at] = held(kk[at], 2), held(vv[at], 0)
        read_k.append(got_k[first[b] - base:])
        read_v.append(got_v[first[b] - base:])
    return {"q": torch.cat(q64), "k": torch.cat(k64), "cached_k": torch.cat(read_k), "cached_v": torch.cat(read_v)}
