"""Attention over blocks with the plan of its own kernel: more query blocks than
a CTA plans for itself, pairs cut between CTAs.  Each case computes the plan
from the lengths (with the constants of the source) and states that it takes
that path and what is cut there; results against oracle/paged.py with the
tolerances of test_paged_gpu.py."""
import os
import re

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_paged_gpu import BF16, DEV, F16, Batch, _i32  # noqa: E402
from vllm_gr_ehaleva_b200.attention import paged_attention  # noqa: E402
from vllm_gr_ehaleva_b200.build import CSRC  # noqa: E402

TILE = 128


def _constants():
    text = open(os.path.join(CSRC, "gr_paged_attn.cu")).read()
    return {n: int(re.search(rf"constexpr int {n} = (\d+);", text).group(1))
            for n in ("kSmallItems", "kCost", "kSnap", "kMinRun", "kJoin", "kMaxCtas")}


class Plan:
    """The query blocks of a batch and the borders of the CTAs' runs."""

    def __init__(self, b, max_new, causal=True, tail=None, steps=None):
        k = _constants()
        HK, D = b.k.shape[2:]
        tp = 128 // (b.q.shape[1] // HK)
        per = tp * (1 if D > 128 or max_new <= tp else 2)
        self.gaps, span = [], []
        for r in range(len(b.lens)):
            n, length = int(b.cu[r + 1] - b.cu[r]), int(b.lens[r])
            ctx, t = length - n, 0 if tail is None else int(tail[r])
            for t0 in range(0, n, per):
                t1 = min(n, t0 + per)
                hi = min(max(ctx + t1, 0), length) if causal else length
                tiles, gap = -(-hi // TILE), 0
                if steps is not None and steps[r] > 0 and t1 > t:
                    own = ctx + t + (max(t0, t) - t) // steps[r] * steps[r]
                    gap = max(own // TILE - -(-(ctx + t) // TILE), 0)
                self.gaps.append(gap)
                span.append(max(tiles - gap, 1) + k["kCost"])
        self.items, pre = len(span), np.concatenate([[0], np.cumsum(span)])
        ctas = min(torch.cuda.get_device_properties(0).multi_processor_count, k["kMaxCtas"])
        units = int(pre[-1])
        total = units * HK
        runs = min(ctas, max(total // k["kMinRun"], 1))
        even, whole = [], []
        for c in range(ctas + 1):
            if c >= runs:
                even.append(total), whole.append(total)
                continue
            u = total * c // runs
            i = int(np.searchsorted(pre, u % units, side="right")) - 1
            off = u % units - int(pre[i])
            whole.append(u - off + (0 if 2 * off < span[i] else span[i]))
            even.append(whole[-1] if span[i] <= k["kSnap"] else u)
        longest = max(b - a for a, b in zip(whole, whole[1:]))
        self.borders = even if longest > total // runs + k["kJoin"] else whole
        # (KV head, query block) of every border behind a pair's first key tile
        self.cuts = set()
        for u in self.borders:
            if u < total:
                i = int(np.searchsorted(pre, u % units, side="right")) - 1
                if u % units - pre[i] > k["kCost"]:
                    self.cuts.add((u // units, i))
        self.head_starts = [u for u in self.borders if u % units == 0 and 0 < u < total]
        assert self.items > k["kSmallItems"], "few query blocks: planned by the CTAs for themselves"
        assert self.cuts, "no pair is cut"


def _singles(D, dtype, H=8, HK=2):
    rng = np.random.default_rng(D)
    ctx = rng.integers(0, 500, 130)
    ctx[[3, 77]] = 20000, 4000
    return Batch(ctx, np.ones(130, np.int64), H, HK, D, 16, dtype, seed=D)


@pytest.mark.parametrize("H,HK,D,dtype", [(8, 2, 128, BF16), (12, 3, 64, F16), (4, 2, 256, F16), (48, 2, 128, BF16)])
def test_single_tokens_one_of_them_over_a_long_cache(H, HK, D, dtype):
    b = _singles(D, dtype, H, HK)
    p = Plan(b, 1)
    assert {h for h, _ in p.cuts} == set(range(HK)), "a cut pair of every KV head"
    b.check(*b.run())
    p = Plan(b, 1, causal=False)
    b.check(*b.run(causal=False), causal=False)


def test_heads_of_256_in_chunks():
    rng = np.random.default_rng(1)
    new = rng.integers(0, 150, 40)
    b = Batch(rng.integers(0, 3000, 40), new, 8, 2, 256, 32, BF16, seed=31)
    p = Plan(b, int(new.max()))
    assert len(p.cuts) > 20
    b.check(*b.run())


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
def test_a_long_chunk(D, dtype):
    # two query tiles to a block; one request whose pairs grow with its own tokens
    b = Batch([500, 9], [3300, 40], 16, 2, D, 16, dtype, seed=32)
    p = Plan(b, 3300)
    assert len(p.cuts) > 20 and len({h for h, _ in p.cuts}) == 2
    b.check(*b.run())


BEAMS = dict(tail=[24] * 16, steps=[3] * 16)


def _beams():
    rng = np.random.default_rng(33)
    return Batch(rng.integers(300, 2600, 16), [24 + 128 * 3] * 16, 8, 2, 128, 16, BF16, seed=33)


def test_beams_behind_long_prefixes():
    b = _beams()
    p = Plan(b, 408, **BEAMS)
    assert any(p.gaps[i] for _, i in p.cuts), "a cut pair that leaves other beams' tiles out"
    b.check(*b.run(beam_tail=_i32(BEAMS["tail"]), beam_steps=_i32(BEAMS["steps"])), **BEAMS)


def test_a_border_at_a_kv_heads_first_pair():
    # runs that end with the last query block of the KV head before
    for b, new, kw in ((_singles(128, BF16), 1, {}), (_beams(), 408, BEAMS)):
        p = Plan(b, new, **kw)
        if torch.cuda.get_device_properties(0).multi_processor_count % 2 == 0:
            assert p.head_starts


@pytest.mark.parametrize("kind", ["single tokens", "beams"])
def test_captured_and_replayed_with_other_lengths(kind):
    b, kw, mx = (_singles(128, BF16), {}, 1) if kind == "single tokens" else (_beams(), BEAMS, 408)
    dev = {f"beam_{n}": _i32(x) for n, x in kw.items()}
    t, cu, lens = _i32(b.table), _i32(b.cu), _i32(b.lens)

    def call():
        return paged_attention(b.q, b.k, b.v, t, cu, lens, mx, return_lse=True, **dev)

    want = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    first = b.lens.copy()
    rng = np.random.default_rng(5)
    for turn in range(4):
        # shorter caches (every key there is still a written one), each time cut elsewhere
        b.lens = first if turn % 2 == 0 else first - (rng.random(len(first)) * b.ctx).astype(first.dtype)
        Plan(b, mx, **kw)
        lens.copy_(_i32(b.lens))
        for _ in range(3):
            out.fill_(float("nan")), lse.fill_(float("nan"))
            graph.replay()
        torch.cuda.synchronize()
        if turn % 2 == 0:
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        else:
            b.check(out, lse, **kw)
