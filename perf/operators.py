"""Cases and plain forms of the paged KV cache operators: what is measured of them.

  tables     block tables, sequence lengths and slot maps of a step, from the requests' lengths and a list of free blocks
  store      a step's new K and V rows written into the cache blocks that the slot map names
  attention  a step's new query tokens (whole prompts, chunks of them, single tokens, beams of one request behind a shared
             prefix) against the keys and values in the requests' blocks

`run` computes them with elementary torch operations in 32 bits (`own` false) or through vllm_gr_ehaleva_b200.attention
(`own` true)."""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


# ---------------------------------------------------------------- cases
def _tables(name, requests, cached, new, block, even, mix=1):
    return {"name": name, "op": "tables", "requests": requests, "cached": cached, "new": new, "block": block, "even": even,
            "mix": mix}


def _store(name, tokens, heads, dim, block, dtype="bf16", pitch=1):
    return {"name": name, "op": "store", "tokens": tokens, "heads": heads, "dim": dim, "block": block, "dtype": dtype,
            "pitch": pitch}


def _attention(name, requests, context, new, heads, kv_heads, dim, block, dtype="bf16", causal=True, tail=0, beams=0,
               steps=0, mix=1):
    return {"name": name, "op": "attention", "requests": requests, "context_lo": context[0], "context_hi": context[1],
            "new_lo": new[0], "new_hi": new[1], "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block,
            "dtype": dtype, "causal": causal, "tail": tail, "beams": beams, "steps": steps, "mix": mix}


def listed():
    return [
        # one decoded token for each of a batch's sequences: the smallest bookkeeping step, pure latency
        _tables("tables, 32 single tokens", 32, 4000, 1, 16, True),
        # 64 requests of 128 beams x 8 decoded tokens behind a tail of 24: the layout of the suffix KV benchmark
        _tables("tables, 64 x 1048 tokens", 64, 2048, 1048, 16, True),
        # many ragged chunks at once, blocks of 32
        _tables("tables, 1500 ragged chunks", 1500, 9000, 700, 32, False),
        # the rows of one decode step of a small batch
        _store("store, 32 rows", 32, 8, 128, 16),
        # the rows of the beam step above
        _store("store, 67072 rows", 67072, 8, 128, 16),
        # heads of 256, 2 of them, K and V columns of one projection's output, an odd count
        _store("store, 9999 strided rows", 9999, 2, 256, 32, "f16", 3),
        # two short sequences, one token each: latency
        _attention("attention, 2 single tokens", 2, (300, 1200), (1, 1), 32, 8, 128, 16),
        # a decode batch over long caches: the cache is read once, nothing else matters
        _attention("attention, 64 single tokens", 64, (500, 16383), (1, 1), 32, 8, 128, 16),
        # a whole prompt
        _attention("attention, prompt of 8192", 1, (0, 0), (8192, 8192), 32, 8, 128, 16),
        # a mixed batch of chunks of any length (single tokens among them), 7 query heads to a KV head
        _attention("attention, 16 ragged chunks", 16, (0, 2500), (1, 1000), 28, 4, 128, 32, "f16"),
        # 128 beams x 3 decoded tokens of 32 requests behind a cached prefix and an uncached tail of 24 tokens
        _attention("attention, 32 x 128 beams", 32, (600, 2600), (408, 408), 32, 8, 128, 16, tail=24, beams=128, steps=3),
        # heads of 256 over 2 KV heads, a chunk of each sequence
        _attention("attention, heads of 256", 12, (1, 4000), (1, 300), 16, 2, 256, 32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("tables", "store", "attention", "attention", "attention"))
    mix = rng.randrange(1, 1 << 20)
    if op == "tables":
        requests = _log(rng, 1, 1500)
        c = _tables("", requests, _log(rng, 1, 9000), _log(rng, 1, 700), rng.choice((16, 32, 64)), rng.random() < 0.5,
                    mix)
    elif op == "store":
        heads, dim = rng.choice(((8, 128), (4, 128), (2, 256), (1, 64), (3, 80)))
        c = _store("", _log(rng, 1, 60000), heads, dim, rng.choice((16, 32)), rng.choice(("bf16", "f16")), rng.choice((1, 3)))
    else:
        heads, kv_heads, dim = rng.choice(((32, 8, 128), (16, 2, 256), (28, 4, 128), (16, 16, 64), (8, 1, 128), (12, 4, 96)))
        block, dtype = rng.choice((16, 32, 64)), rng.choice(("bf16", "f16"))
        kind = rng.choice(("single", "chunks", "beams", "whole"))
        if kind == "single":
            c = _attention("", _log(rng, 1, 48), (1, _log(rng, 2, 12000)), (1, 1), heads, kv_heads, dim, block, dtype, mix=mix)
        elif kind == "chunks":
            c = _attention("", _log(rng, 2, 12), (0, _log(rng, 16, 2500)), (1, _log(rng, 16, 1000)), heads, kv_heads, dim,
                           block, dtype, mix=mix)
        elif kind == "beams":
            tail, beams, steps = rng.randrange(0, 40), _log(rng, 4, 128), rng.randrange(1, 5)
            new = tail + beams * steps
            c = _attention("", _log(rng, 1, 16), (1, _log(rng, 16, 2600)), (new, new), heads, kv_heads, dim, block, dtype,
                           tail=tail, beams=beams, steps=steps, mix=mix)
        else:
            n = _log(rng, 64, 4000)
            c = _attention("", 1, (0, 0), (n, n), heads, kv_heads, dim, block, dtype, rng.random() < 0.7, mix=mix)
    del c["name"]
    return c


# ---------------------------------------------------------------- shapes: of the case alone
def _spread(n, lo, hi, mix):
    """n lengths between lo and hi, both among them where there is room, spread over their logarithm."""
    r = np.random.RandomState(mix)
    x = np.exp(r.uniform(math.log(lo + 1), math.log(hi + 1), n)).round().astype(np.int64) - 1
    x[0] = hi
    if n > 1:
        x[r.randint(1, n)] = lo
    return np.clip(x, lo, hi)


def _lengths(c):
    """(cached, new) tokens of each request."""
    if c["op"] == "tables":
        new = np.full(c["requests"], c["new"]) if c["even"] else _spread(c["requests"], 0, c["new"], c["mix"] + 1)
        return _spread(c["requests"], 0, c["cached"], c["mix"]), new
    n = c["requests"]
    return _spread(n, c["context_lo"], c["context_hi"], c["mix"]), _spread(n, c["new_lo"], c["new_hi"], c["mix"] + 1)


def _ceil(a, b):
    return -(-a // b)


def _visible(c):
    """Pairs of a query token and a key that it sees, over all requests."""
    cached, new = _lengths(c)
    if not c["causal"]:
        return int((new * (cached + new)).sum())
    pairs = new * cached + new * (new + 1) // 2
    if c["steps"]:
        tail, steps, beams = c["tail"], c["steps"], c["beams"]
        pairs = new * cached + tail * (tail + 1) // 2 + beams * (steps * tail + steps * (steps + 1) // 2)
    return int(pairs.sum())


def work(c):
    if c["op"] == "tables":
        cached, new = _lengths(c)
        t, r, b = int(new.sum()), c["requests"], c["block"]
        fresh = int((_ceil(cached + new, b) - _ceil(cached, b)).sum())
        partial = int(((cached % b != 0) & (new > 0)).sum())
        return {"bytes": 8 * r + 8 * fresh + 4 * partial + 16 * t + 8 * r + 8, "flops": 0}
    row = c["heads" if c["op"] == "store" else "kv_heads"] * c["dim"] * 2
    if c["op"] == "store":
        return {"bytes": c["tokens"] * (4 * row + 8), "flops": 0}
    cached, new = _lengths(c)
    t, keys = int(new.sum()), int((cached + new).sum())
    return {"bytes": 2 * keys * row + 4 * t * c["heads"] * c["dim"] + 4 * t * c["heads"] + 4 * int(_ceil(cached + new, c["block"]).sum()),
            "flops": 4 * c["heads"] * c["dim"] * _visible(c)}


# ---------------------------------------------------------------- inputs
def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def ints(x, dtype=torch.int32):
        return torch.from_numpy(np.ascontiguousarray(x)).to(DEV, dtype)

    if c["op"] == "tables":
        cached, new = _lengths(c)
        have, need = _ceil(cached, c["block"]), _ceil(cached + new, c["block"])
        held, fresh = int(have.sum()), int((need - have).sum())
        ids = torch.randperm(held + fresh + 64, device=DEV, generator=g).to(torch.int32)
        width = int(need.max()) + 3
        table = torch.full((c["requests"], width), -1, dtype=torch.int32, device=DEV)
        table[torch.arange(width, device=DEV)[None] < ints(have)[:, None]] = ids[:held]
        return {"case": c, "table": table, "cached": ints(cached), "new": ints(new), "free": ids[held:].clone(),
                "tokens": int(new.sum())}
    dtype = DTYPES[c["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device=DEV, generator=g, dtype=torch.float32).mul_(std).to(dtype)

    if c["op"] == "store":
        t, h, d, b = c["tokens"], c["heads"], c["dim"], c["block"]
        blocks = _ceil(t, b) + 2
        kv = normal(t, 1 + c["pitch"], h, d)
        return {"case": c, "k": kv[:, 0], "v": kv[:, 1], "k_cache": normal(blocks, b, h, d), "v_cache": normal(blocks, b, h, d),
                "slots": torch.randperm(blocks * b, device=DEV, generator=g)[:t].contiguous()}
    cached, new = _lengths(c)
    keys = cached + new
    need = _ceil(keys, c["block"])
    blocks = int(need.sum()) + 3
    ids = torch.randperm(blocks, device=DEV, generator=g).to(torch.int32)
    width = max(1, int(need.max()))
    table = torch.zeros(c["requests"], width, dtype=torch.int32, device=DEV)
    table[torch.arange(width, device=DEV)[None] < ints(need)[:, None]] = ids[:int(need.sum())]
    s = {"case": c, "table": table, "cu": ints(np.concatenate([[0], np.cumsum(new)])), "lens": ints(keys),
         "max_new": int(new.max()), "max_keys": int(keys.max()),
         "q": normal(int(new.sum()), c["heads"], c["dim"], std=2.0),
         "k_cache": normal(blocks, c["block"], c["kv_heads"], c["dim"]),
         "v_cache": normal(blocks, c["block"], c["kv_heads"], c["dim"])}
    if c["steps"]:
        s["tail"] = torch.full((c["requests"],), c["tail"], dtype=torch.int32, device=DEV)
        s["steps"] = torch.full((c["requests"],), c["steps"], dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"tables": _own_tables, "store": _own_store, "attention": _own_attention}[op](s)
    return {"tables": _plain_tables, "store": _plain_store, "attention": _plain_attention}[op](s)


def _own_tables(s):
    from vllm_gr_ehaleva_b200.attention import extend_block_tables
    m = extend_block_tables(s["table"], s["cached"], s["new"], s["free"], s["case"]["block"], s["tokens"])
    return {"table": s["table"], "cu": m["cu_seqlens_q"], "lens": m["seq_lens"], "slots": m["slot_mapping"],
            "positions": m["positions"], "used": m["blocks_used"]}


def _own_store(s):
    from vllm_gr_ehaleva_b200.attention import store_kv
    store_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attention(s):
    from vllm_gr_ehaleva_b200.attention import paged_attention
    out, lse = paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["lens"], s["max_new"],
                               causal=s["case"]["causal"], beam_tail=s.get("tail"), beam_steps=s.get("steps"), return_lse=True)
    return {"out": out, "lse": lse}


def _plain_tables(s):
    b, table, cached, new, free = s["case"]["block"], s["table"], s["cached"].long(), s["new"].long(), s["free"]
    have, need = (cached + b - 1) // b, (cached + new + b - 1) // b
    take = need - have
    j = torch.arange(table.shape[1], device=DEV)[None]
    at = (torch.cumsum(take, 0) - take)[:, None] + j - have[:, None]
    table.copy_(torch.where((j >= have[:, None]) & (j < need[:, None]), free[at.clamp(0, free.numel() - 1)], table))
    ends = torch.cumsum(new, 0)
    t = torch.arange(s["tokens"], device=DEV)
    r = torch.searchsorted(ends, t, right=True)
    positions = cached[r] + t - (ends - new)[r]
    slots = table[r, positions // b].long() * b + positions % b
    cu = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    return {"table": table, "cu": cu, "lens": (cached + new).to(torch.int32), "slots": slots, "positions": positions,
            "used": take.sum().reshape(1).to(torch.int32)}


def _plain_store(s):
    for rows, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        cache.view(-1, *cache.shape[2:])[s["slots"]] = rows
    return {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _seen(c, rows, keys, new, lens, tail, steps):
    """Which keys [0, keys) each of the query tokens [0, rows) of every request sees: [requests, rows, keys]."""
    i, k = torch.arange(rows, device=DEV)[None, :, None], torch.arange(keys, device=DEV)[None, None]
    new, lens = new[:, None, None], lens[:, None, None]
    if not c["causal"]:
        return (k < lens) & (i < new)
    at = lens - new + i
    ok = (k <= at) & (i < new)
    if steps is not None:
        first = lens - new + tail[:, None, None]  # the first beam's first token
        of = first + torch.div(at - first, steps[:, None, None], rounding_mode="floor") * steps[:, None, None]
        ok &= (k < first) | (k >= of)
    return ok


def _plain_attention(s):
    c, q = s["case"], s["q"]
    cu, lens = s["cu"].long(), s["lens"].long()
    new, r, n, keys = cu[1:] - cu[:-1], c["requests"], s["max_new"], s["max_keys"]
    h, hk, d, b = c["heads"], c["kv_heads"], c["dim"], c["block"]
    g = h // hk
    i, k = torch.arange(n, device=DEV), torch.arange(keys, device=DEV)
    there = (k[None] < lens[:, None])[:, :, None, None]
    kk = torch.where(there, s["k_cache"][s["table"][:, k // b].long(), k % b].float(), 0)
    vv = torch.where(there, s["v_cache"][s["table"][:, k // b].long(), k % b].float(), 0)
    rows = (cu[:-1, None] + i[None]).clamp(max=q.shape[0] - 1)
    qq = q[rows].float().view(r, n, hk, g, d).permute(0, 2, 3, 1, 4).reshape(r, hk, g * n, d)
    scores = torch.matmul(qq, kk.permute(0, 2, 3, 1)).view(r, hk, g, n, keys)
    seen = _seen(c, n, keys, new, lens, s["tail"].long() if "tail" in s else None, s["steps"].long() if "steps" in s else None)
    scores.mul_(1 / math.sqrt(d)).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(r, hk, g * n, keys), vv.permute(0, 2, 1, 3)).view(r, hk, g, n, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(r * n, h, d)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2).reshape(r * n, h)
    # back to the tokens in their order: token t of request i is padded row i * n + t
    t = torch.arange(q.shape[0], device=DEV)
    of = torch.searchsorted(cu[1:], t, right=True)
    back = of * n + t - cu[of]
    return {"out": o[back].to(q.dtype), "lse": lse[back]}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "tables":
        return None  # whole numbers: compared as they are
    if c["op"] == "store":
        res = {}
        for rows, cache in (("k", "k_cache"), ("v", "v_cache")):
            x = s[cache].double()
            b = c["block"]
            x[s["slots"] // b, s["slots"] % b] = s[rows].double()
            res[cache] = x
        return res
    cu, lens, b, g = s["cu"].tolist(), s["lens"].tolist(), c["block"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for r in range(c["requests"]):
        n, total = cu[r + 1] - cu[r], lens[r]
        if n == 0 or total == 0:
            continue
        ids = s["table"][r, : _ceil(total, b)].long()
        kr = s["k_cache"][ids].reshape(-1, c["kv_heads"], c["dim"])[:total].double()
        vr = s["v_cache"][ids].reshape(-1, c["kv_heads"], c["dim"])[:total].double()
        i, k = torch.arange(n, device=DEV)[:, None], torch.arange(total, device=DEV)[None]
        hidden = torch.zeros(n, total, dtype=torch.bool, device=DEV)
        if c["causal"]:
            hidden |= k - (total - n) > i
        if c["steps"]:
            # a beam's token sees the tokens of other beams never: j counts new tokens, beams start behind the tail
            j = k - (total - n)
            beam_q, beam_k = (i - c["tail"]) // c["steps"], (j - c["tail"]) // c["steps"]
            hidden |= (j >= c["tail"]) & ((i < c["tail"]) | (beam_q != beam_k))
        for head in range(c["heads"]):
            z = s["q"][cu[r]:cu[r + 1], head].double() @ kr[:, head // g].T / math.sqrt(c["dim"])
            z[hidden] = -math.inf
            e = torch.logsumexp(z, 1)
            w = torch.exp(z - torch.where(e == -math.inf, torch.zeros_like(e), e)[:, None])
            out[cu[r]:cu[r + 1], head] = w @ vr[:, head // g]
            lse[cu[r]:cu[r + 1], head] = e
    return {"out": out, "lse": lse}
