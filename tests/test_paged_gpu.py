"""GPU parity of the paged KV cache operators (block tables and slot maps,
cache write, attention over blocks) against their definitions in 64 bits
(oracle/paged.py), at the sizes and masks where they can go wrong.

Tolerance of an attention output, from the arithmetic (h: half a step of the
16-bit type, relative): the output is rounded once (h |out|); each probability
is rounded once before the second product (h sum w|v|); a score's fp32 error
makes a relative error of its weight, e_w = 2 (D 2^-23 Smax + 2^-22 (1 + Smax)),
Smax the largest scale * sum |q||k|: D additions of one step each, the scaling,
the exponential; the fp32 sums over L keys, L 2^-22 for numerator and
denominator.  In f16, probabilities below its normal range add up to 2^-25 each
against a sum of at least 1."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from oracle import paged as ref  # noqa: E402
from vllm_gr_ehaleva_b200 import _lib  # noqa: E402
from vllm_gr_ehaleva_b200.attention import (build_suffix_metadata, extend_block_tables, extract_suffix_kv,  # noqa: E402
                                            paged_attention, store_kv)

DEV = "cuda"
BF16, F16 = torch.bfloat16, torch.float16


def _i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=DEV)


class Batch:
    """Requests with `ctx` cached and `new` query tokens each; every slot that no request
    owns, the rest of the last blocks among them, holds NaN."""

    def __init__(self, ctx, new, H, HK, D, bs, dtype, seed=0, std=1.0, lens=None, width=None, spare=3):
        rng = np.random.default_rng(seed)
        self.ctx, self.new = np.asarray(ctx), np.asarray(new)
        self.lens = self.ctx + self.new if lens is None else np.asarray(lens)
        need = -(-self.lens // bs)
        nb = int(need.sum()) + spare
        ids = rng.permutation(nb)
        self.table = np.full((len(self.lens), width or max(1, int(need.max()))), -7, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = ids[at:at + n]
            at += n
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        g = torch.Generator(device=DEV).manual_seed(seed)

        def normal(*shape, s=1.0):
            return (torch.randn(*shape, device=DEV, generator=g) * s).to(dtype)

        self.q = normal(int(self.new.sum()), H, D, s=std)
        self.k, self.v = normal(nb, bs, HK, D), normal(nb, bs, HK, D)
        owned = torch.zeros(nb * bs, dtype=torch.bool, device=DEV)
        for r in range(len(self.lens)):
            p = np.arange(int(self.lens[r]))
            owned[torch.as_tensor(self.table[r, p // bs].astype(np.int64) * bs + p % bs, device=DEV)] = True
        for c in (self.k, self.v):
            c.view(nb * bs, HK, D)[~owned] = float("nan")

    def run(self, **kw):
        return paged_attention(self.q, self.k, self.v, _i32(self.table), _i32(self.cu), _i32(self.lens),
                               kw.pop("max_new", int(self.new.max(initial=0))), return_lse=True, **kw)

    def check(self, out, lse, causal=True, scale=None, tail=None, steps=None):
        torch.cuda.synchronize()
        q, k, v = (x.double().cpu().numpy() for x in (self.q, self.k, self.v))
        o, e, absv = ref.attention(q, k, v, self.table, self.cu, self.lens, causal=causal, scale=scale, tail=tail,
                                   steps=steps)
        D = q.shape[2]
        h = torch.finfo(self.q.dtype).eps / 2
        L = max(1, int(self.lens.max(initial=1)))
        smax = (scale or D ** -0.5) * np.abs(q).sum(2).max(initial=0) * np.nanmax(np.abs(k), initial=0)
        smax = min(smax, (scale or D ** -0.5) * np.sqrt((q ** 2).sum(2).max(initial=0) *
                                                        np.nanmax((k ** 2).sum(3), initial=0)))
        # (the second bound, by Cauchy-Schwarz, holds for sum |q||k| too)
        ew = 2 * (D * 2.0 ** -23 * smax + 2.0 ** -22 * (1 + smax))
        tiny = L * 2.0 ** -25 * np.nanmax(np.abs(v), initial=0) if self.q.dtype == F16 else 0.0
        tol = h * np.abs(o) + (h + ew + L * 2.0 ** -22) * absv * 1.01 + tiny + 1e-30
        got = out.double().cpu().numpy()
        assert np.isfinite(got).all()
        worst = (np.abs(got - o) / tol).max(initial=0)
        assert worst <= 1, f"output {worst:.2f} times its tolerance"
        ge = lse.double().cpu().numpy()
        assert (np.isneginf(ge) == np.isneginf(e)).all()
        fin = ~np.isneginf(e)
        tol_e = ew + L * 2.0 ** -22 + np.abs(e[fin]) * 2.0 ** -22
        assert (np.abs(ge[fin] - e[fin]) <= tol_e).all(), np.abs(ge[fin] - e[fin]).max()


# single tokens, short and long; block tables that end inside a tile; heads of every padded size
@pytest.mark.parametrize("H,HK,D,bs,dtype", [(32, 8, 128, 16, BF16), (8, 8, 64, 16, F16), (16, 2, 256, 32, BF16),
                                             (7, 1, 128, 24, F16), (12, 4, 96, 8, BF16), (4, 2, 40, 48, F16),
                                             (6, 2, 8, 64, BF16), (128, 1, 128, 256, BF16), (5, 5, 200, 16, F16)])
def test_single_tokens(H, HK, D, bs, dtype):
    b = Batch([0, 1, 15, 16, 127, 128, 129, 700, 1999, 3], [1] * 10, H, HK, D, bs, dtype, seed=D + bs)
    b.check(*b.run())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,HK,D,bs,dtype", [(8, 2, 128, 16, BF16), (4, 4, 64, 16, F16), (8, 1, 256, 32, BF16),
                                             (14, 2, 128, 40, F16), (3, 1, 72, 8, BF16)])
def test_chunks_of_any_length(H, HK, D, bs, dtype, causal):
    ctx = [0, 0, 5, 130, 64, 1, 300, 0, 250]
    new = [1, 200, 0, 1, 257, 33, 129, 64, 128]
    b = Batch(ctx, new, H, HK, D, bs, dtype, seed=7)
    b.check(*b.run(causal=causal), causal=causal)


@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, F16), (256, BF16)])
def test_whole_prompts(D, dtype):
    b = Batch([0, 0], [1000, 641], 4, 2, D, 16, dtype, seed=3, std=2.0)
    b.check(*b.run())


@pytest.mark.parametrize("H,HK,D,bs,dtype", [(8, 2, 128, 16, BF16), (8, 1, 64, 32, F16), (4, 2, 256, 16, BF16),
                                             (7, 1, 128, 16, F16)])
def test_beams_see_prefix_tail_and_themselves(H, HK, D, bs, dtype):
    # beams that start at, before and behind tile and block borders; one-token beams; a plain
    # request, an all-tail request and a request without a cached prefix among them
    ctx = [300, 0, 127, 700, 64, 5, 40]
    tail = [24, 0, 1, 100, 3, 50, 0]
    steps = [3, 1, 4, 5, 0, 2, 130]
    new = [24 + 3 * 64, 200, 1 + 4 * 37, 100 + 5 * 31, 70, 50, 260]
    b = Batch(ctx, new, H, HK, D, bs, dtype, seed=11)
    b.check(*b.run(beam_tail=_i32(tail), beam_steps=_i32(steps)), tail=tail, steps=steps)


def test_beams_whose_last_one_is_cut_short():
    # the reference builder cuts the last beam when the query budget ends
    b = Batch([90, 31], [10 + 3 * 20 + 2, 1 + 4 * 9 + 1], 8, 2, 128, 16, BF16, seed=12)
    kw = dict(tail=[10, 1], steps=[3, 4])
    b.check(*b.run(beam_tail=_i32(kw["tail"]), beam_steps=_i32(kw["steps"])), **kw)


def test_rows_that_see_nothing():
    # fewer keys than query tokens: the first rows' mask is empty; no keys at all; both kinds
    b = Batch([0] * 5, [4, 200, 1, 300, 1], 8, 2, 128, 16, BF16, seed=5, lens=[2, 150, 0, 0, 1])
    out, lse = b.run()
    b.check(out, lse)
    assert (out[:2] == 0).all() and torch.isneginf(lse[:2]).all()
    assert (out[205:505] == 0).all() and torch.isneginf(lse[205:505]).all()
    out, lse = b.run(causal=False)
    b.check(out, lse, causal=False)
    empty = Batch([0, 0], [3, 1], 8, 2, 128, 16, BF16, seed=6, lens=[0, 0])
    out, lse = empty.run()
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, F16), (256, F16)])
@pytest.mark.parametrize("new", [1, 300])
def test_scores_that_rise_over_the_keys(D, dtype, new):
    # every key tile raises the running maximum by far more than the rescaling threshold
    b = Batch([1000, 390], [new, new], 4, 2, D, 16, dtype, seed=13)
    b.q.fill_(1.0)
    for r in range(2):
        n = int(b.lens[r])
        p = np.arange(n)
        at = torch.as_tensor(b.table[r, p // 16].astype(np.int64) * 16 + p % 16, device=DEV)
        ramp = torch.arange(n, device=DEV, dtype=torch.float32)[:, None, None] / 8
        b.k.view(-1, 2, D)[at] = (ramp * D ** -0.5).expand(n, 2, D).to(dtype)
    b.check(*b.run())
    # and falling: the first tile holds the maximum
    b.q.fill_(-1.0)
    b.check(*b.run())


def test_long_caches_split_over_the_grid():
    b = Batch([20000, 3], [1, 1], 8, 2, 128, 16, BF16, seed=14)
    b.check(*b.run())
    b = Batch([9000], [2], 2, 1, 256, 32, F16, seed=15)
    b.check(*b.run())
    b = Batch([12000], [100], 4, 2, 64, 16, BF16, seed=16)
    b.check(*b.run(max_new=100))


@pytest.mark.parametrize("D,dtype", [(128, BF16), (256, F16)])
@pytest.mark.parametrize("group", [24, 32])
def test_pairs_in_more_parts_than_a_warp_has_lanes(group, D, dtype):
    # a single token's pair over 79 CTAs or more, rows that stay with their lanes (more than 16 a
    # warp): each lane waits for parts that all lanes read
    b = Batch([25000], [1], group, 1, D, 16, dtype, seed=30 + group)
    o, e = b.run()
    b.check(o, e)
    for _ in range(20):
        again = b.run()
        assert torch.equal(again[0], o) and torch.equal(again[1], e)


@pytest.mark.parametrize("R", [95, 96, 97, 1024, 1025, 2300])
def test_many_requests(R):
    rng = np.random.default_rng(R)
    ctx, new = rng.integers(0, 90, R), rng.integers(0, 3, R)
    b = Batch(ctx, new, 4, 2, 64, 16, BF16, seed=R)
    b.check(*b.run())
    b.check(*b.run(max_new=1000))           # a bound far above the longest query: the two-tile kernel


def test_many_query_blocks():
    # more than one pass of the plan, and sums beyond its shared memory
    b = Batch([0, 17], [4500, 4000], 4, 1, 64, 16, F16, seed=17)
    b.check(*b.run())
    b = Batch([0] * 30, [90] * 30, 128, 1, 8, 8, BF16, seed=18)
    b.check(*b.run())


def test_results_do_not_depend_on_the_run():
    b = Batch([3000, 40, 700], [1, 90, 300], 8, 2, 128, 16, BF16, seed=18)
    o1, e1 = b.run()
    for _ in range(3):
        o2, e2 = b.run()
        assert torch.equal(o1, o2) and torch.equal(e1, e2)
    # without the log-sum-exp, and into a tensor of the caller's
    out = torch.empty_like(b.q)
    got = paged_attention(b.q, b.k, b.v, _i32(b.table), _i32(b.cu), _i32(b.lens), 300, out=out)
    assert got is out and torch.equal(out, o1)


def test_the_query_bound_only_picks_the_kernel():
    # a bound below the longest query and one far above: the other kernel, the same rows
    for D in (64, 128):
        b = Batch([500, 30, 0], [1, 150, 70], 8, 2, D, 16, BF16, seed=26)
        for bound in (0, 1, 10 ** 9):
            b.check(*b.run(max_new=bound))


def test_scale():
    b = Batch([200], [130], 4, 2, 128, 16, BF16, seed=19)
    b.check(*b.run(scale=0.3), scale=0.3)


def test_strided_queries_caches_and_outputs():
    H, HK, D, bs = 8, 2, 128, 16
    b = Batch([40, 300, 0], [1, 70, 200], H, HK, D, bs, BF16, seed=20)
    o, e = b.run()
    b.check(o, e)
    t, cu, lens = _i32(b.table), _i32(b.cu), _i32(b.lens)
    nb = b.k.shape[0]
    # K and V interleaved per block, heads before tokens, a table that is a view of a wider one
    kv = torch.full((nb, 2, HK, bs, D), float("nan"), dtype=BF16, device=DEV)
    kv[:, 0], kv[:, 1] = b.k.transpose(1, 2), b.v.transpose(1, 2)
    k, v = kv[:, 0].transpose(1, 2), kv[:, 1].transpose(1, 2)
    wide = torch.full((3, t.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + t.shape[1]] = t
    # q as a slice of a projection's output, out as every second head of a wider tensor
    qkv = torch.randn(b.q.shape[0], H + 2 * HK, D, device=DEV).to(BF16)
    qkv[:, :H] = b.q
    out = torch.full((b.q.shape[0], 2 * H, D), 7.0, dtype=BF16, device=DEV)
    got, lse = paged_attention(qkv[:, :H], k, v, wide[:, 2:2 + t.shape[1]], cu, lens, 200, out=out[:, ::2],
                               return_lse=True)
    assert torch.equal(got, o) and torch.equal(lse, e)
    assert (out[:, 1::2] == 7).all()


def test_smallest_sizes():
    # one token, one head, one block; strides of dimensions of one entry mean nothing
    for ctx, D in ((0, 8), (5, 8), (3, 256)):
        b = Batch([ctx], [1], 1, 1, D, 8, BF16, seed=ctx, spare=0)
        b.check(*b.run())
        q = b.q.as_strided((1, 1, D), (3, 5, 1))
        k, v = (x.as_strided((1, 8, 1, D), (7, D, 3, 1)) for x in (b.k, b.v))
        assert torch.equal(paged_attention(q, k, v, _i32(b.table), _i32(b.cu), _i32(b.lens), 1), b.run()[0])


def test_one_request_among_many_without_tokens():
    # plan passes of 1024 requests, most of them empty
    new = np.zeros(3000, np.int64)
    new[[0, 1023, 1024, 2999]] = [3, 200, 1, 70]
    b = Batch(np.full(3000, 2), new, 4, 2, 64, 8, BF16, seed=28)
    b.check(*b.run())


def test_rows_of_no_request_stay():
    b = Batch([10, 20], [5, 6], 4, 2, 64, 16, BF16, seed=21)
    o, _ = b.run()
    q = torch.cat([b.q, torch.full((9, 4, 64), float("nan"), dtype=BF16, device=DEV)])
    out = torch.full_like(q, 3.0)
    paged_attention(q, b.k, b.v, _i32(b.table), _i32(b.cu), _i32(b.lens), 6, out=out)
    assert torch.equal(out[:11], o) and (out[11:] == 3).all()


def test_cache_beyond_32_bit_offsets():
    # 2.2e9 elements per cache: rows behind 2^31 elements and 2^32 bytes
    HK, D, bs = 8, 128, 16
    nb = 2_200_000_000 // (HK * D * bs)
    k = torch.zeros(nb, bs, HK, D, dtype=BF16, device=DEV)
    v = torch.zeros(nb, bs, HK, D, dtype=BF16, device=DEV)
    n = 100
    table = torch.arange(nb - 7, nb, dtype=torch.int32, device=DEV)[None]
    g = torch.Generator(device=DEV).manual_seed(3)
    kr, vr = (torch.randn(n, HK, D, device=DEV, generator=g).to(BF16) for _ in range(2))
    slots = (nb - 7) * bs + torch.arange(n, dtype=torch.int64, device=DEV)
    store_kv(kr, vr, k, v, slots)
    assert torch.equal(k.view(-1, HK, D)[slots], kr) and torch.equal(v.view(-1, HK, D)[slots], vr)
    assert int((k[:nb - 7] != 0).sum()) == 0
    b = Batch([n - 1], [1], 8, HK, D, bs, BF16, seed=1)
    b.k, b.v = torch.zeros(7, bs, HK, D, dtype=BF16, device=DEV), torch.zeros(7, bs, HK, D, dtype=BF16, device=DEV)
    b.k.view(-1, HK, D)[:n], b.v.view(-1, HK, D)[:n] = kr, vr
    b.table = np.arange(7, dtype=np.int32)[None]
    out, lse = paged_attention(b.q, k, v, table, _i32(b.cu), _i32(b.lens), 1, return_lse=True)
    b.check(out, lse)


def test_bad_blocks_and_records_are_reported():
    b = Batch([100, 40, 60], [3, 2, 1], 4, 2, 64, 16, BF16, seed=22)
    o, e = b.run()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    b.run(err=err)
    assert int(err) == 0
    nb = b.k.shape[0]
    good = b.table.copy()
    for bad in (nb, -1, 2 ** 31 - 1, -2 ** 31):
        b.table = good.copy()
        b.table[1, 0] = bad
        err.zero_()
        out, lse = b.run(err=err)
        assert int(err) == 0x20
        assert torch.equal(out[:3], o[:3]) and torch.equal(out[5:], o[5:])
        # zero rows: the scores of that block's 16 keys are 0, their values add nothing
        k, v = b.k.clone(), b.v.clone()
        k[good[1, 0]] = 0
        v[good[1, 0]] = 0
        want = paged_attention(b.q, k, v, _i32(good), _i32(b.cu), _i32(b.lens), 3)
        assert torch.equal(out, want)
    b.table = good
    # lengths outside the table's row (clamped), query offsets that fall or leave the tokens
    for lens, cu in (([103, 42, 10 ** 6], b.cu), ([103, 42, -5], b.cu), (b.lens, [0, 3, 2, 6]),
                     (b.lens, [0, 3, 5, 100]), (b.lens, [-4, 3, 5, 6])):
        err.zero_()
        paged_attention(b.q, b.k, b.v, _i32(b.table), _i32(cu), _i32(lens), 3, err=err)
        assert int(err) & 0x40, (lens, cu)
    torch.cuda.synchronize()
    o2, e2 = b.run()
    assert torch.equal(o, o2) and torch.equal(e, e2)


def test_sizes_of_zero():
    k = torch.zeros(4, 16, 2, 64, dtype=BF16, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    out, lse = paged_attention(torch.zeros(0, 4, 64, dtype=BF16, device=DEV), k, k, _i32(np.zeros((2, 1))),
                               _i32([0, 0, 0]), _i32([5, 0]), 0, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    q = torch.ones(3, 4, 64, dtype=BF16, device=DEV)
    kept = torch.full_like(q, 2.0)
    paged_attention(q, k, k, torch.zeros(0, 1, dtype=torch.int32, device=DEV), _i32([0]), none, 3, out=kept)
    assert (kept == 2).all()
    # a cache without blocks, a table without columns: every row is empty
    for kc, tab in ((k[:0], np.zeros((1, 1))), (k, np.zeros((1, 0)))):
        out, lse = paged_attention(q, kc, kc, _i32(tab), _i32([0, 3]), _i32([0]), 3, return_lse=True)
        assert (out == 0).all() and torch.isneginf(lse).all()


def test_refusals():
    b = Batch([20, 3], [2, 1], 4, 2, 64, 16, BF16, seed=27)
    t, cu, lens = _i32(b.table), _i32(b.cu), _i32(b.lens)

    def call(q=b.q, k=b.k, v=b.v, t=t, cu=cu, lens=lens, n=2, **kw):
        return paged_attention(q, k, v, t, cu, lens, n, **kw)

    want = call()
    wide = torch.zeros(3, 4, 72, dtype=BF16, device=DEV)
    for match, kw in (
            ("bf16 or f16", dict(q=b.q.float())), ("bf16 or f16", dict(q=b.q.half())),
            ("same dtype", dict(v=b.v.half())), ("num_blocks, block_size", dict(k=b.k[0], v=b.v[0])),
            ("head_dim", dict(q=wide)), ("multiple of", dict(q=b.q[:, :3])), ("unit stride", dict(q=b.q.transpose(0, 2).contiguous().transpose(0, 2))),
            ("int32", dict(lens=lens.long())), ("int32", dict(cu=cu.long())), ("int32", dict(t=t.long())),
            ("shape", dict(cu=cu[:2])), ("rows for", dict(t=t[:1])), ("1-D", dict(lens=lens[None])),
            ("unit stride", dict(t=torch.zeros(2, 6, dtype=torch.int32, device=DEV)[:, ::2])),
            ("contiguous", dict(lens=torch.zeros(4, dtype=torch.int32, device=DEV)[::2])),
            ("int32", dict(lens=lens.cpu())), ("CUDA", dict(q=b.q.cpu())),
            ("go together", dict(beam_tail=lens)), ("go together", dict(beam_steps=lens)),
            ("causal", dict(beam_tail=lens, beam_steps=lens, causal=False)),
            ("scale", dict(scale=0.0)), ("scale", dict(scale=-1)), ("scale", dict(scale=float("nan"))),
            ("scale", dict(scale=float("inf"))), ("out must", dict(out=torch.empty_like(b.q).half())),
            ("out must", dict(out=torch.empty_like(b.q)[:2])), ("err must", dict(err=lens.long()))):
        with pytest.raises(ValueError, match=match):
            call(**kw)
    with pytest.raises(RuntimeError, match="GR_ERR_MISALIGNED"):
        call(q=torch.zeros(3 * 4 * 64 + 1, dtype=BF16, device=DEV)[1:].view(3, 4, 64))
    with pytest.raises(RuntimeError, match="GR_ERR_MISALIGNED"):
        call(out=torch.zeros(3, 4, 68, dtype=BF16, device=DEV)[..., :64])
    with pytest.raises(RuntimeError, match="GR_ERR_UNSUPPORTED"):
        call(k=b.k.view(-1, 4, 2, 64), v=b.v.view(-1, 4, 2, 64))
    with pytest.raises(RuntimeError, match="GR_ERR_BAD_DESC"):
        call(n=-1)
    assert torch.equal(call(), want)

    s = torch.arange(3, device=DEV)
    k = torch.zeros(3, 2, 64, dtype=BF16, device=DEV)
    for match, args in (("cache's heads", (k[:, :1], k[:, :1], b.k, b.v, s)), ("dtype", (k.half(), k.half(), b.k, b.v, s)),
                        ("shape", (k, k, b.k, b.v, s[:2])), ("int64", (k, k, b.k, b.v, s.float())),
                        ("no blocks", (k, k, b.k[:0], b.v[:0], s)), ("element size", (k.double(), k.double(), b.k.double(), b.v.double(), s)),
                        ("CUDA", (k, k, b.k.cpu(), b.v.cpu(), s))):
        with pytest.raises(ValueError, match=match):
            store_kv(*args)
    for match, args in (("rows for", (t, lens[:1], lens[:1], lens, 16, 3)), ("shape", (t, lens, lens[:1], lens, 16, 3)),
                        ("int32", (t, lens, lens, lens.long(), 16, 3)), ("positive", (t, lens, lens, lens, 0, 3)), ("2\\^31", (t, lens, lens, lens, 2 ** 32 + 16, 3)),
                        ("num_tokens", (t, lens, lens, lens, 16, -1)), ("1-D", (t, lens[None], lens, lens, 16, 3)),
                        ("overlap", (torch.zeros(4, dtype=torch.int32, device=DEV).as_strided((2, 3), (1, 1)), lens, lens, lens, 16, 3))):
        with pytest.raises(ValueError, match=match):
            extend_block_tables(*args)


def test_captured_beside_eager_calls_and_on_another_stream():
    b = Batch([700, 40, 1500], [1, 90, 1], 8, 2, 128, 16, BF16, seed=23)
    c = Batch([900, 10, 30], [1, 90, 1], 8, 2, 128, 16, BF16, seed=24)
    t, cu, lens = _i32(b.table), _i32(b.cu), _i32(b.lens)
    tc, cuc, lensc = _i32(c.table), _i32(c.cu), _i32(c.lens)

    def one():
        return paged_attention(b.q, b.k, b.v, t, cu, lens, 90, return_lse=True)

    def two():
        return paged_attention(c.q, c.k, c.v, tc, cuc, lensc, 90, return_lse=True)

    want1, want2 = one(), two()
    torch.cuda.synchronize()
    graphs = []
    for fn in (one, two):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = fn()
        graphs.append((gr, res))
    # both graphs at once on two streams, eager calls on a third: each has its own workspace
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for (gr, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        with torch.cuda.stream(streams[2]):
            got = one()
        torch.cuda.synchronize()
        for (_, res), want in zip(graphs, (want1, want2)):
            assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])
        assert torch.equal(got[0], want1[0]) and torch.equal(got[1], want1[1])
    # a replay reads new lengths
    lens.copy_(_i32([701, 95, 1501]))
    graphs[0][0].replay()
    torch.cuda.synchronize()
    b.lens = np.array([701, 95, 1501])
    b.check(*graphs[0][1])


def test_expired_waits_report_and_return(monkeypatch):
    # no copies are issued: every wait runs out, the call returns with the bit set
    for new, D in (([1, 1], 128), ([200, 60], 128), ([3, 2], 256)):
        b = Batch([300, 50], new, 4, 2, D, 16, BF16, seed=25)
        want = b.run()
        torch.cuda.synchronize()
        monkeypatch.setenv("GR_TEST_STALL_COPIES", "1")
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        b.run(err=err)
        torch.cuda.synchronize()
        assert int(err) & 0x4
        monkeypatch.delenv("GR_TEST_STALL_COPIES")
        got = b.run()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_expired_waits_of_cut_pairs(monkeypatch):
    # every CTA has a part of a pair: roles that wait for copies, for one another and for other
    # CTAs' parts all leave; with few query blocks, and with a plan of its own kernel
    for ctx, new in (([20000], [1]), ([20000] + [5] * 119, [1] * 120)):
        b = Batch(ctx, new, 8, 2, 128, 16, BF16, seed=29)
        want = b.run()
        torch.cuda.synchronize()
        monkeypatch.setenv("GR_TEST_STALL_COPIES", "1")
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        b.run(err=err)
        torch.cuda.synchronize()
        assert int(err) & 0x4
        monkeypatch.delenv("GR_TEST_STALL_COPIES")
        got = b.run()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---------------------------------------------------------------- block tables and slot maps
@pytest.mark.parametrize("R,bs", [(1, 16), (5, 1), (37, 16), (256, 16), (257, 16), (1024, 32), (2047, 16), (2048, 32), (2049, 48), (5000, 16)])
def test_block_tables(R, bs):
    rng = np.random.default_rng(R)
    cached = rng.integers(0, 200, R) * (rng.random(R) < 0.8)
    fresh = rng.integers(0, 70, R) * (rng.random(R) < 0.7)
    need = -(-(cached + fresh) // bs)
    have = -(-cached // bs)
    width = int(need.max()) + 2
    total = int(need.sum())
    ids = rng.permutation(total + 40).astype(np.int32)
    table = np.full((R, width), -1, np.int32)
    for r in range(R):
        table[r, :have[r]] = ids[:have[r]]
    free = rng.permutation(300000).astype(np.int32)[:int((need - have).sum()) + 5]
    for pad in (0, 13):
        n = int(fresh.sum()) + pad
        want = ref.extend_block_tables(table, cached, fresh, free, bs, n)
        dev = torch.full((R, width + 3), -9, dtype=torch.int32, device=DEV)
        view = dev[:, 1:1 + width]
        view.copy_(torch.from_numpy(table))
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        m = extend_block_tables(view, _i32(cached), _i32(fresh), _i32(free), bs, n, err=err)
        assert int(err) == 0
        assert np.array_equal(view.cpu().numpy(), want[0])
        assert (dev[:, 0] == -9).all() and (dev[:, width + 1:] == -9).all()
        assert np.array_equal(m["cu_seqlens_q"].cpu().numpy(), want[1])
        assert np.array_equal(m["seq_lens"].cpu().numpy(), want[2])
        assert np.array_equal(m["slot_mapping"].cpu().numpy(), want[3])
        assert np.array_equal(m["positions"].cpu().numpy(), want[4])
        assert int(m["blocks_used"]) == want[5]


def test_block_tables_one_long_request_among_empty_ones():
    cached, fresh = [0, 7, 0, 0, 16, 0], [0, 0, 50000, 0, 0, 0]
    table = np.full((6, 3200), -1, np.int32)
    table[1, 0], table[4, 0] = 90001, 90002
    free = np.random.default_rng(0).permutation(80000).astype(np.int32)[:3200]
    want = ref.extend_block_tables(table, np.array(cached), np.array(fresh), free, 16, 50000)
    dev = torch.from_numpy(table).to(DEV)
    m = extend_block_tables(dev, _i32(cached), _i32(fresh), _i32(free), 16, 50000)
    assert np.array_equal(dev.cpu().numpy(), want[0])
    assert np.array_equal(m["slot_mapping"].cpu().numpy(), want[3])


def test_block_tables_report_what_does_not_fit():
    err = torch.zeros(1, dtype=torch.int32, device=DEV)

    def call(cached, fresh, free, n, width=4, held=3):
        err.zero_()
        table = torch.full((len(cached), width), -1, dtype=torch.int32, device=DEV)
        table[:, :held] = torch.arange(100, 100 + held, dtype=torch.int32, device=DEV)
        m = extend_block_tables(table, _i32(cached), _i32(fresh), _i32(free), 16, n, err=err)
        return table.cpu().numpy(), {k: v.cpu().numpy() for k, v in m.items()}, int(err)

    # the free list is one block short: the last request's last token has no slot
    table, m, e = call([16, 16], [17, 17], [1, 2, 3], 34)
    assert e == 0x80 and m["blocks_used"][0] == 4
    want = ref.extend_block_tables(np.tile(np.array([100, 101, 102, -1], np.int32), (2, 1)), [16, 16], [17, 17],
                                   [1, 2, 3], 16, 34)
    assert np.array_equal(m["slot_mapping"], want[3]) and np.array_equal(table, want[0])
    # the row has no room
    table, m, e = call([60], [10], [7, 8], 10)
    assert e == 0x80 and (m["slot_mapping"][4:] == -1).all() and (table[0] == [100, 101, 102, -1]).all()
    # the partly filled block's entry is negative
    table, m, e = call([60], [2], [], 2)
    assert e == 0x80 and (m["slot_mapping"] == -1).all()
    # negative and overflowing lengths count as no new token
    table, m, e = call([5, -3, 2 ** 31 - 1, 20], [2, 4, 1, 1], [50], 3, width=4)
    assert e & 0x40 and list(m["cu_seqlens_q"]) == [0, 2, 2, 2, 3]
    assert list(m["slot_mapping"]) == [1605, 1606, 101 * 16 + 4]
    # more new tokens than entries
    table, m, e = call([0], [40], [50, 51, 52], 33)
    assert e == 0x40 and len(m["slot_mapping"]) == 33 and list(m["cu_seqlens_q"]) == [0, 40]
    # no request: padding only
    m = extend_block_tables(torch.zeros(0, 4, dtype=torch.int32, device=DEV), _i32([]), _i32([]), _i32([]), 16, 5)
    assert (m["slot_mapping"] == -1).all() and int(m["cu_seqlens_q"]) == 0 and int(m["blocks_used"]) == 0


@pytest.mark.parametrize("R", [3, 300])
@pytest.mark.parametrize("bs", [1, 16])
def test_block_tables_end_with_the_free_list_whatever_the_lengths_ask_for(R, bs):
    # lengths near 2^31 ask for up to 10^11 blocks; the work is that of the 40 there are
    free = np.random.default_rng(R).permutation(500).astype(np.int32)[:40]
    table = torch.full((R, 50), -1, dtype=torch.int32, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    n = 41 * bs
    m = extend_block_tables(table, _i32([0] * R), _i32([2 ** 31 - 1] * R), _i32(free), bs, n, err=err)
    assert int(err) == 0x80 | 0x40
    want = np.full((R, 50), -1, np.int32)
    want[0, :40] = free
    assert np.array_equal(table.cpu().numpy(), want)
    assert (m["seq_lens"] == 2 ** 31 - 1).all() and int(m["blocks_used"]) == min(2 ** 31 - 1, R * -(-(2 ** 31 - 1) // bs))
    assert m["cu_seqlens_q"].tolist() == [0] + [2 ** 31 - 1] * R
    slots = np.concatenate([free.astype(np.int64).repeat(bs) * bs + np.tile(np.arange(bs), 40), np.full(bs, -1)])
    assert np.array_equal(m["slot_mapping"].cpu().numpy(), slots)
    assert m["positions"].tolist() == list(range(n))


# ---------------------------------------------------------------- cache write
@pytest.mark.parametrize("dtype", [BF16, F16, torch.float32, torch.uint8])
@pytest.mark.parametrize("H,D,bs", [(8, 128, 16), (2, 256, 32), (1, 8, 1), (3, 5, 7), (1, 1, 16), (16, 256, 16)])
def test_store(H, D, bs, dtype):
    for T in (1, 3, 200):
        nb = T // bs + 3
        g = torch.Generator(device=DEV).manual_seed(T)
        make = lambda *s: torch.randint(0, 250, s, device=DEV, generator=g).to(dtype)  # noqa: E731
        k, v, kc, vc = make(T, H, D), make(T, H, D), make(nb, bs, H, D), make(nb, bs, H, D)
        slots = torch.randperm(nb * bs, device=DEV, generator=g)[:T].clone()
        if T > 2:
            slots[1] = -1                       # padding
        keep = slots >= 0
        wk, wv = kc.clone(), vc.clone()
        wk.view(-1, H, D)[slots[keep]], wv.view(-1, H, D)[slots[keep]] = k[keep], v[keep]
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        store_kv(k, v, kc, vc, slots, err=err)
        assert torch.equal(kc, wk) and torch.equal(vc, wv) and int(err) == 0
        store_kv(k, v, kc, vc, slots.to(torch.int32))
        assert torch.equal(kc, wk) and torch.equal(vc, wv)


def test_store_strided_rows_and_caches():
    T, H, D, bs, nb = 50, 4, 64, 16, 9
    g = torch.Generator(device=DEV).manual_seed(1)
    qkv = torch.randn(T, 12, D, device=DEV, generator=g).to(BF16)
    k, v = qkv[:, 4:8], qkv[:, 8:]
    slots = torch.randperm(nb * bs, device=DEV, generator=g)[:T]
    b, o = slots // bs, slots % bs
    kv = torch.zeros(nb, 2, bs, H, D, dtype=BF16, device=DEV)          # K and V beside each other in a block
    want = kv.clone()
    want[b, 0, o], want[b, 1, o] = k, v
    store_kv(k, v, kv[:, 0], kv[:, 1], slots)
    assert torch.equal(kv, want)
    hnd = torch.zeros(2, nb, H, bs, D, dtype=BF16, device=DEV)         # heads before tokens: element kernel
    kc, vc = hnd[0].transpose(1, 2), hnd[1].transpose(1, 2)
    store_kv(k, v, kc, vc, slots)
    assert torch.equal(kc[b, o], k) and torch.equal(vc[b, o], v)
    rows = torch.randn(T, D, H, device=DEV, generator=g).to(BF16).transpose(1, 2)   # head dim strided, odd address
    kc = torch.zeros(nb * bs * H * D + 1, dtype=BF16, device=DEV)[1:].view(nb, bs, H, D)
    vc = kc.clone()
    store_kv(rows, rows, kc, vc, slots)
    assert torch.equal(kc[b, o], rows) and torch.equal(vc[b, o], rows)


def test_store_reports_slots_behind_the_cache():
    kc, vc = torch.zeros(3, 16, 2, 64, dtype=BF16, device=DEV), torch.zeros(3, 16, 2, 64, dtype=BF16, device=DEV)
    rows = torch.ones(4, 2, 64, dtype=BF16, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    store_kv(rows, rows, kc, vc, torch.tensor([47, 48, -1, 2 ** 62], device=DEV), err=err)
    assert int(err) == 0x20
    assert (kc[2, 15] == 1).all() and int((kc != 0).sum()) == 128
    store_kv(rows[:0], rows[:0], kc, vc, torch.zeros(0, dtype=torch.int64, device=DEV))


# ---------------------------------------------------------------- together
def test_a_mega_request_decode_through_all_of_them():
    """Two steps of a batch as the worker would run them: prompts first, then the beams'
    tokens; the beam attention equals the reference's way (prefix pass, suffix gather, a
    causal pass per beam, joined by their log-sum-exps) computed in 64 bits on the gathered
    rows."""
    H, HK, D, bs, dtype = 8, 2, 128, 16, BF16
    g = torch.Generator(device=DEV).manual_seed(5)
    rows = lambda t: (torch.randn(t, HK, D, device=DEV, generator=g).to(dtype) for _ in range(2))  # noqa: E731
    prompts, W, steps = [75, 200, 48], 12, 3
    free = torch.randperm(200, device=DEV, generator=g).to(torch.int32)
    k_cache = torch.full((200, bs, HK, D), float("nan"), dtype=dtype, device=DEV)
    v_cache = k_cache.clone()
    table = torch.full((3, 40), -1, dtype=torch.int32, device=DEV)
    cached_len = [64, 160, 48]                     # cached up to there; the rest of the prompt is the tail

    def step(cached, fresh, q, **kw):
        n = int(sum(fresh))
        m = extend_block_tables(table, _i32(cached), _i32(fresh), free, bs, n)
        k, v = rows(n)
        store_kv(k, v, k_cache, v_cache, m["slot_mapping"])
        out, lse = paged_attention(q, k_cache, v_cache, table, m["cu_seqlens_q"], m["seq_lens"], int(max(fresh)),
                                   return_lse=True, **kw)
        return m, out, lse

    q = torch.randn(sum(cached_len), H, D, device=DEV, generator=g).to(dtype)
    m, out, lse = step([0, 0, 0], cached_len, q)
    free = free[int(m["blocks_used"]):]
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    tail = [p - c for p, c in zip(prompts, cached_len)]
    fresh = [t + W * steps for t in tail]
    q = torch.randn(sum(fresh), H, D, device=DEV, generator=g).to(dtype)
    m, out, lse = step(cached_len, fresh, q, beam_tail=_i32(tail), beam_steps=_i32([steps] * 3))

    # the reference's split, on the same cache
    mega = [dict(prefix_len=p, cache_len=c, beam_width=W, steps=steps) for p, c in zip(prompts, cached_len)]
    q_starts = [0] + list(np.cumsum(fresh))
    md = build_suffix_metadata(mega, q_starts, 1024, DEV)      # blocks of 1024: no prefix goes apart
    slots = m["slot_mapping"][md["mega_prefix_indices"]]
    sk, sv = extract_suffix_kv(k_cache, v_cache, slots, md["suffix_slot_mapping_out"], md["suffix_total_tokens"])
    cu_q, cu_k = md["suffix_cu_seqlens_q"].tolist(), md["suffix_cu_seqlens_k"].tolist()
    want = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    wlse = torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    tab = table.long()
    for b in range(len(cu_q) - 1):
        a, z = cu_q[b], cu_q[b + 1]
        r = next(i for i in range(3) if q_starts[i] <= a < q_starts[i + 1])
        pos = torch.arange(cached_len[r], device=DEV)
        pk, pv = (c[tab[r, pos // bs], pos % bs].double() for c in (k_cache, v_cache))
        n, kn = z - a, cu_k[b + 1] - cu_k[b]
        ok = torch.arange(kn, device=DEV)[None] <= torch.arange(n, device=DEV)[:, None] + kn - n
        for h in range(H):
            qq = q[a:z, h].double() * D ** -0.5
            s1 = qq @ pk[:, h // 4].T
            s2 = (qq @ sk[cu_k[b]:cu_k[b + 1], h // 4].double().T).masked_fill(~ok, -torch.inf)
            e1, e2 = s1.logsumexp(1), s2.logsumexp(1)
            e = torch.logaddexp(e1, e2)
            want[a:z, h] = torch.exp(s1 - e[:, None]) @ pv[:, h // 4] + \
                torch.exp(s2 - e[:, None]) @ sv[cu_k[b]:cu_k[b + 1], h // 4].double()
            wlse[a:z, h] = e
    h = torch.finfo(dtype).eps / 2
    # |v| < 6 here: two roundings of at most h each, as at the top of this file, plus the fp32 terms
    assert ((out.double() - want).abs() <= h * want.abs() + (h + 2.0 ** -14) * 6).all()
    rel = (out.double() - want).norm() / want.norm()
    assert rel <= 2 * h
    assert (lse.double() - wlse).abs().max() <= 2.0 ** -14
