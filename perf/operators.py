"""The operators of an attention layer that serves a model, as cases that can be timed and checked:

  rope       norms of queries and keys for each head with the position rotation, one pass
  cache      keys and values written into a paged cache and read back as packed rows, in 8 bits or 16
  attention  whole prompts, packed, causal, grouped heads
  paged      new tokens (one for each sequence, or chunks) over a paged cache in 8 bits or 16

`run` computes a case from elementary torch operations in 32 bits, or, where `own` is true, through the
framework's operators.  Sizes go from a call that is all latency to a prompt of 8192 tokens; lengths are
ragged, and follow from the case alone.
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
F8 = torch.float8_e4m3fn
F8_MOST = 448.0       # the largest finite e4m3 value
LEAST_AMAX = 2.0**-100  # rows smaller than this share its scale, so that neither it nor its inverse leaves the floats
EPS = 1e-6


def _rope(dtype, tokens, heads, kv_heads, dim, rotary, interleaved, norm=True):
    return {"op": "rope", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rotary": rotary, "interleaved": interleaved, "norm": norm}


def _cache(dtype, cache, seqs, longest, chunk, kv_heads, dim, page):
    return {"op": "cache", "dtype": dtype, "cache": cache, "seqs": seqs, "longest": longest, "chunk": chunk,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def _attention(dtype, seqs, longest, heads, kv_heads, dim):
    return {"op": "attention", "dtype": dtype, "seqs": seqs, "longest": longest, "heads": heads, "kv_heads": kv_heads,
            "dim": dim}


def _paged(dtype, cache, seqs, longest, chunk, heads, kv_heads, dim, page):
    return {"op": "paged", "dtype": dtype, "cache": cache, "seqs": seqs, "longest": longest, "chunk": chunk,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page}


def listed():
    return [
        # one step of generation for 16 sequences: a call that is all latency
        dict(_rope("bf16", 16, 32, 8, 128, 128, False), name="rope_decode16"),
        # a packed prompt of 8192 tokens, bound by reading and writing it
        dict(_rope("bf16", 8192, 32, 8, 128, 128, False), name="rope_prompt"),
        # an odd number of tokens, neighbouring pairs, half of each head turned, no norm
        dict(_rope("fp16", 4099, 16, 16, 64, 32, True, False), name="rope_interleaved_odd"),
        # one new token for each of 16 short sequences, into 8 bits, and their contexts back
        dict(_cache("bf16", "fp8", 16, 200, 1, 8, 128, 16), name="cache_fp8_decode16"),
        # chunks of 512 tokens into 8 bits under long contexts, and the contexts back
        dict(_cache("fp16", "fp8", 8, 8191, 512, 8, 128, 64), name="cache_fp8_chunks"),
        # a prompt's small packed sequences: many short rows, tiles mostly cut
        dict(_attention("fp16", 24, 333, 16, 16, 64), name="attention_fp16_short"),
        # a packed batch of prompts of different lengths, grouped heads
        dict(_attention("bf16", 6, 3001, 32, 8, 128), name="attention_bf16_packed"),
        # one long prompt, the largest: bound by the matrix cores
        dict(_attention("bf16", 1, 8192, 32, 8, 128), name="attention_bf16_8192"),
        # generation for a few short sequences: latency
        dict(_paged("fp16", "fp16", 4, 500, 1, 32, 8, 128, 16), name="paged_decode4_fp16"),
        # generation for 64 sequences of different lengths: bound by reading the cache
        dict(_paged("bf16", "bf16", 64, 8192, 1, 32, 8, 128, 64), name="paged_decode64_bf16"),
        # generation for one long sequence from 8 bits: work split over its length
        dict(_paged("bf16", "fp8", 1, 65537, 1, 32, 8, 128, 64), name="paged_decode1_fp8_long"),
        # chunks of up to 512 new tokens, ragged, over 8 bits
        dict(_paged("bf16", "fp8", 4, 8100, 512, 32, 8, 128, 64), name="paged_chunks_fp8"),
    ]


def _size(rng, lo, hi):
    """A whole number from lo to hi, uniform over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    while True:
        op = rng.choice(["rope", "rope", "cache", "cache", "attention", "attention", "paged", "paged", "paged"])
        dtype = rng.choice(["fp16", "bf16"])
        dim = rng.choice([64, 128, 128, 128])
        kv_heads = rng.choice([2, 4, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 8])
        page = rng.choice([16, 32, 64])
        held = rng.choice(["fp8", "fp8", dtype])
        if op == "rope":
            rotary = rng.choice([dim, dim, dim // 2])
            case = _rope(dtype, _size(rng, 1, 16384), heads, kv_heads, dim, rotary, rng.random() < 0.4, rng.random() < 0.7)
        elif op == "cache":
            longest = _size(rng, 32, 8192)
            case = _cache(dtype, held, _size(rng, 1, 32), longest, rng.choice([1, 1, _size(rng, 2, longest)]), kv_heads, dim, page)
        elif op == "attention":
            case = _attention(dtype, _size(rng, 1, 32), _size(rng, 16, 8192), heads, kv_heads, dim)
        else:
            longest = _size(rng, 64, 65536)
            case = _paged(dtype, held, _size(rng, 1, 128), longest, rng.choice([1, 1, 1, _size(rng, 2, 512)]), heads, kv_heads, dim, page)
            case["chunk"] = min(case["chunk"], longest)
        if _padded(case) <= _padded(listed()[7]) and _held(case) < 8e9:
            return case


def _padded(case):
    """Products of the plain form, which pads every sequence to the longest."""
    if case["op"] in ("rope", "cache"):
        return 0
    rows = case["longest"] if case["op"] == "attention" else case["chunk"]
    return case["seqs"] * rows * case["longest"] * case["heads"] * case["dim"]


def _held(case):
    """Bytes of keys and values in 32 bits, padded."""
    return 0 if case["op"] == "rope" else 8 * case["seqs"] * case["longest"] * case["kv_heads"] * case["dim"]


def _lengths(case):
    """(new tokens, whole length) of every sequence: the first is the longest, the others spread over the
    logarithm below it, and none has more new tokens than it is long."""
    rng = random.Random("%d %d" % (case["seqs"], case["longest"]))
    whole = [case["longest"]] + [_size(rng, max(1, case["longest"] // 16), case["longest"]) for _ in range(case["seqs"] - 1)]
    if case["op"] == "attention":
        return whole, whole
    new = [case["chunk"]] + [_size(rng, max(1, case["chunk"] // 16), case["chunk"]) for _ in range(case["seqs"] - 1)]
    return [min(a, b) for a, b in zip(new, whole)], whole


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _fill(x, held):
    """What a cache holds for the rows x: (values, scales or None)."""
    if held != "fp8":
        return x, None
    amax = x.float().abs().amax(-1, keepdim=True).clamp(min=LEAST_AMAX)
    return (x.float() * (F8_MOST / amax)).clamp(-F8_MOST, F8_MOST).to(F8), (amax / F8_MOST).squeeze(-1)


def _make_cache(case, gen, whole):
    """Pages in a random order, some of them in nobody's table, filled with earlier tokens' keys and values."""
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    each = [-(-n // page) for n in whole]
    pages = sum(each) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(whole), max(each)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(each):
        table[i, :n] = order[at : at + n]
        at += n
    state = {"table": table}
    for name in ("k", "v"):
        x = _normal(gen, (pages, page, heads, dim), DTYPES[case["dtype"]])
        state[name + "_cache"], state[name + "_scale"] = _fill(x, case["cache"])
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]
    state = {"op": op, "case": case}
    if op == "rope":
        # queries, keys and values as the three parts of one product's rows, as a layer has them
        t, h, hk, d, rot = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rotary"]
        rows = _normal(gen, (t, (h + 2 * hk) * d), dtype)
        state["q"] = rows[:, : h * d].view(t, h, d)
        state["k"] = rows[:, h * d : (h + hk) * d].view(t, hk, d)
        most = max(4096, t)
        turn = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        state["cos"], state["sin"] = turn.cos().float(), turn.sin().float()
        state["positions"] = torch.randint(0, most, (t,), generator=gen, device="cuda")
        for name in ("q", "k"):
            w = 1 + 0.2 * torch.randn(d, generator=gen, device="cuda")
            state[name + "_weight"] = w.to(dtype) if case["norm"] else None
        return state
    new, whole = _lengths(case)
    state.update(cu_q=_starts(new), cu_k=_starts(whole), total_q=sum(new), total_k=sum(whole), most_q=max(new),
                 most_k=max(whole), lens=torch.tensor(whole, dtype=torch.int32, device="cuda"))
    hk, d = case["kv_heads"], case["dim"]
    if op == "attention":
        h = case["heads"]
        state["q"] = _normal(gen, (state["total_q"], h, d), dtype)
        rows = _normal(gen, (state["total_k"], 2, hk, d), dtype)  # keys and values of a token side by side
        state["k"], state["v"] = rows[:, 0], rows[:, 1]
        return state
    state.update(_make_cache(case, gen, whole))
    if op == "paged":
        state["q"] = _normal(gen, (state["total_q"], case["heads"], d), dtype)
        return state
    rows = _normal(gen, (state["total_q"], 2, hk, d), dtype)
    state["k"], state["v"] = rows[:, 0], rows[:, 1]
    seq, at = _places(state["cu_q"], state["total_q"])
    at = at + (state["lens"] - (state["cu_q"][1:] - state["cu_q"][:-1]))[seq]  # new tokens end their sequences
    page = case["page"]
    state["slots"] = state["table"][seq, at // page].long() * page + at % page
    return state


def _places(starts, total):
    """The sequence of each packed row, and its place in it."""
    row = torch.arange(total, device="cuda")
    seq = torch.searchsorted(starts[1:].long(), row, right=True)
    return seq, row - starts.long()[seq]


def _pad(x, starts, total, most):
    """Packed rows [total, ...] as [sequences, most, ...], zero past each length."""
    out = x.new_zeros((starts.numel() - 1, most) + x.shape[1:])
    out[_places(starts, total)] = x
    return out


def _gather(cache, scale, table, most):
    """The rows of each sequence's pages, [sequences, most, heads, dim], in 32 bits."""
    x = cache[table.long()].float()
    if scale is not None:
        x = x * scale[table.long()][..., None]
    return x.flatten(1, 2)[:, :most]


def _plain_rope(x, weight, s):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    rot, half = 2 * cos.shape[-1], cos.shape[-1]
    if s["case"]["interleaved"]:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:rot]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _plain_attention(q, k, v, len_q, len_k):
    """q [n, rows, heads, dim], k and v [n, keys, kv heads, dim] in 32 bits; a row sees the keys up to its
    own place, counted from the end."""
    n, rows, heads, dim = q.shape
    keys, kv_heads = k.shape[1:3]
    q = q.view(n, rows, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, -1, dim)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(dim)
    s = s.view(n, kv_heads, -1, rows, keys)
    last = torch.arange(rows, device=q.device) + (len_k - len_q)[:, None]
    seen = torch.arange(keys, device=q.device) <= torch.minimum(last, len_k[:, None] - 1)[..., None]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    s = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    total = s.sum(-1, keepdim=True)
    s = s.view(n, kv_heads, -1, keys)
    o = torch.matmul(s, v.permute(0, 2, 1, 3)).view(n, kv_heads, -1, rows, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(n, rows, heads, dim)


def _run_plain(s):
    case, op = s["case"], s["op"]
    if op == "rope":
        return _plain_rope(s["q"], s["q_weight"], s), _plain_rope(s["k"], s["k_weight"], s)
    if op == "cache":
        got = []
        for name in ("k", "v"):
            cache, scale = s[name + "_cache"], s[name + "_scale"]
            values, scales = _fill(s[name], case["cache"])
            cache.view(-1, *cache.shape[2:])[s["slots"]] = values
            if scale is not None:
                scale.view(-1, scale.shape[2])[s["slots"]] = scales
            seq, at = _places(s["cu_k"], s["total_k"])
            got.append(_gather(cache, scale, s["table"], s["most_k"])[seq, at].to(s[name].dtype))
        return tuple(got)
    len_q = s["cu_q"][1:] - s["cu_q"][:-1]
    q = _pad(s["q"].float(), s["cu_q"], s["total_q"], s["most_q"])
    if op == "attention":
        k, v = (_pad(s[x].float(), s["cu_k"], s["total_k"], s["most_k"]) for x in ("k", "v"))
    else:
        k, v = (_gather(s[x + "_cache"], s[x + "_scale"], s["table"], s["most_k"]) for x in ("k", "v"))
    return _plain_attention(q, k, v, len_q, s["lens"])[_places(s["cu_q"], s["total_q"])].to(s["q"].dtype)


def _run_own(s):
    import cmpext3

    op = s["op"]
    if op == "rope":
        return cmpext3.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], s["q_weight"], s["k_weight"],
                                    eps=EPS, interleaved=s["case"]["interleaved"])
    if op == "cache":
        cmpext3.kv_cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["k_scale"], s["v_scale"])
        return cmpext3.kv_cache_read(s["k_cache"], s["v_cache"], s["table"], s["cu_k"], s["total_k"],
                                     dtype=s["k"].dtype, k_scale=s["k_scale"], v_scale=s["v_scale"])
    if op == "attention":
        return cmpext3.attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=True)
    one = s["case"]["chunk"] == 1  # one token for each sequence: no starts to give
    return cmpext3.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                   cu_seqlens_q=None if one else s["cu_q"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    if case["op"] == "rope":
        t, h, d = case["tokens"], case["heads"] + case["kv_heads"], case["dim"]
        # rows in and out, each token's row of the two tables and its position, the weights
        return {"bytes": 4 * t * h * d + 4 * t * case["rotary"] + 8 * t + (4 * d if case["norm"] else 0),
                "flops": t * h * d * ((4 if case["norm"] else 0) + 3)}
    new, whole = _lengths(case)
    kv = case["kv_heads"] * case["dim"]
    held = 2 * kv * (1 if case.get("cache") == "fp8" else 2) + (8 * case["kv_heads"] if case.get("cache") == "fp8" else 0)
    if case["op"] == "cache":
        # new rows in and into the cache, the whole lengths out of it and into packed rows
        return {"bytes": sum(new) * (4 * kv + held + 8) + sum(whole) * (held + 4 * kv),
                "flops": 4 * kv * sum(new) + 2 * kv * sum(whole)}
    seen = sum(b * a - a * (a - 1) // 2 for a, b in zip(new, whole))
    rows = 4 * sum(new) * case["heads"] * case["dim"]
    keys = sum(whole) * (held if case["op"] == "paged" else 4 * kv)
    return {"bytes": rows + keys, "flops": 4 * seen * case["heads"] * case["dim"]}


def _exact_rope(x, weight, s):
    """Each pair of a head as a complex number, turned by cos + i sin."""
    y = x.double()
    if weight is not None:
        y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * weight.double()
    angle = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]]
    rot = 2 * angle.shape[-1]
    even, odd = (slice(0, rot, 2), slice(1, rot, 2)) if s["case"]["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    z = torch.complex(y[..., even].contiguous(), y[..., odd].contiguous()) * angle[:, None]
    y[..., even], y[..., odd] = z.real, z.imag
    return y


def _exact_held(x):
    """Rows as e4m3 holds them: the nearest of its values (three bits after the first, none below 2^-9),
    scaled so that the row's largest is 448."""
    x = x.double()
    scale = x.abs().amax(-1, keepdim=True).clamp(min=LEAST_AMAX) / F8_MOST
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)
    return (y / step).round() * step * scale


def _exact_rows(s, name, seq):
    """A sequence's keys or values from its pages, in 64 bits."""
    pages = s["table"][seq, : -(-int(s["lens"][seq]) // s["case"]["page"])].long()
    x = s[name + "_cache"][pages].double()
    if s[name + "_scale"] is not None:
        x = x * s[name + "_scale"][pages].double()[..., None]
    return x.flatten(0, 1)[: int(s["lens"][seq])]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s["q"], s["q_weight"], s), _exact_rope(s["k"], s["k_weight"], s)
    out = []
    if case["op"] == "cache":
        for name in ("k", "v"):
            rows = []
            for i in range(case["seqs"]):
                old = _exact_rows(s, name, i)
                x = s[name][int(s["cu_q"][i]) : int(s["cu_q"][i + 1])]
                rows += [old[: old.shape[0] - x.shape[0]], _exact_held(x) if case["cache"] == "fp8" else x.double()]
            out.append(torch.cat(rows))
        return tuple(out)
    group = case["heads"] // case["kv_heads"]
    for i in range(case["seqs"]):
        q = s["q"][int(s["cu_q"][i]) : int(s["cu_q"][i + 1])].double()
        if case["op"] == "attention":
            k, v = (s[x][int(s["cu_k"][i]) : int(s["cu_k"][i + 1])].double() for x in ("k", "v"))
        else:
            k, v = (_exact_rows(s, x, i) for x in ("k", "v"))
        ahead = torch.ones((q.shape[0], k.shape[0]), dtype=torch.bool, device="cuda").triu(1 + k.shape[0] - q.shape[0])
        o = torch.empty_like(q)
        for h in range(case["heads"]):
            w = (q[:, h] @ k[:, h // group].t() * case["dim"] ** -0.5).masked_fill_(ahead, -math.inf)
            o[:, h] = torch.softmax(w, -1) @ v[:, h // group]
        out.append(o)
    return torch.cat(out)
