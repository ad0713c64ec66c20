"""Paged KV cache operators on the CPU: struct layouts against the header, what
the entry points refuse (before any device work), the wrappers' checks, and the
oracle against the reference builder's own suffix metadata."""
import ctypes
import json
import os
import subprocess
import tempfile

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import paged as ref
from vllm_gr_ehaleva_b200 import _lib
from vllm_gr_ehaleva_b200.attention import extend_block_tables, paged_attention, store_kv

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NULL, BAD, DTYPE, MISALIGNED, WORKSPACE, UNSUPPORTED = -1, -2, -3, -4, -5, -6


def test_struct_layouts_match_header():
    structs = {"gr_block_table_desc": _lib.BlockTableDesc, "gr_kv_store_desc": _lib.KvStoreDesc,
               "gr_paged_attn_desc": _lib.PagedAttnDesc, "gr_paged_attn_io": _lib.PagedAttnIO}
    lines, want = [], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "gr_beam.h"\nint main(void) {' + "\n".join(lines) + "return 0; }"
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = list(map(int, subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()))
    assert got == want
    assert _lib.describe_deverr(0x80) == "GR_DEVERR_NO_BLOCK"


def _attn(**kw):
    d = dict(num_seqs=2, num_tokens=3, num_heads=8, num_kv_heads=2, head_dim=128, block_size=16, max_blocks=4, dtype=1,
             causal=1, max_query_len=2, scale=0.1, reserved=0, num_blocks=9, table_stride=4, q_stride_tok=1024,
             q_stride_head=128, k_stride_block=4096, k_stride_tok=256, k_stride_head=128, v_stride_block=4096,
             v_stride_tok=256, v_stride_head=128, out_stride_tok=1024, out_stride_head=128)
    d.update(kw)
    return _lib.PagedAttnDesc(*[d[n] for n, _ in _lib.PagedAttnDesc._fields_])


@pytest.mark.parametrize("kw,status", [
    (dict(), 0), (dict(head_dim=256), 0), (dict(head_dim=8), 0), (dict(num_seqs=0, num_tokens=0), 0),
    (dict(num_heads=256), 0), (dict(max_blocks=0, num_blocks=0), 0),
    (dict(num_seqs=-1), BAD), (dict(num_tokens=-1), BAD), (dict(num_heads=7), BAD), (dict(num_kv_heads=0), BAD),
    (dict(head_dim=0), BAD), (dict(block_size=0), BAD), (dict(causal=2), BAD), (dict(max_query_len=-1), BAD),
    (dict(scale=0.0), BAD), (dict(scale=-1.0), BAD), (dict(scale=float("nan")), BAD), (dict(scale=float("inf")), BAD),
    (dict(table_stride=3), BAD), (dict(num_blocks=2 ** 31), BAD), (dict(max_blocks=2 ** 27, table_stride=2 ** 27), BAD),
    (dict(num_tokens=2 ** 31 - 1000), BAD), (dict(scale=3e38), BAD),
    (dict(dtype=0), DTYPE), (dict(dtype=9), DTYPE),
    (dict(head_dim=264), UNSUPPORTED), (dict(head_dim=100), UNSUPPORTED), (dict(block_size=12), UNSUPPORTED),
    (dict(num_heads=258), UNSUPPORTED),
])
def test_attention_descriptors(kw, status):
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    assert lib.gr_paged_attention_workspace_size(_attn(**kw), n) == status
    assert (n.value > 0) == (status == 0)
    if status:
        io = _lib.PagedAttnIO()
        assert lib.gr_paged_attention(_attn(**kw), io, None, 0, None) == status


def test_attention_pointers():
    lib = _lib.load()
    n = ctypes.c_size_t(0)
    assert lib.gr_paged_attention_workspace_size(None, n) == NULL
    assert lib.gr_paged_attention_workspace_size(_attn(), None) == NULL
    assert lib.gr_paged_attention(_attn(), None, None, 0, None) == NULL
    d = _attn()
    lib.gr_paged_attention_workspace_size(d, n)

    def io(**kw):
        x = _lib.PagedAttnIO()
        for f in ("q", "k_cache", "v_cache", "block_table", "cu_seqlens", "seq_lens", "out"):
            setattr(x, f, kw.get(f, 4096))
        for f in ("beam_tail", "beam_steps"):
            setattr(x, f, kw.get(f))
        return x

    def call(desc=d, ws=4096, size=n.value, **kw):
        return lib.gr_paged_attention(desc, io(**kw), ws, size, None)

    for f in ("q", "k_cache", "v_cache", "block_table", "cu_seqlens", "seq_lens", "out"):
        assert call(**{f: None}) == NULL, f
    assert call(ws=None) == NULL
    assert call(beam_tail=4096) == NULL and call(beam_steps=4096) == NULL
    assert call(_attn(causal=0), beam_tail=4096, beam_steps=4096) == BAD
    for f in ("q", "k_cache", "v_cache", "out"):
        assert call(**{f: 4104}) == MISALIGNED, f
    for f in ("q_stride_tok", "q_stride_head", "k_stride_block", "k_stride_tok", "k_stride_head", "v_stride_block",
              "v_stride_tok", "v_stride_head", "out_stride_tok", "out_stride_head"):
        for bad in (132, 0, -128):
            assert call(_attn(**{f: bad})) == MISALIGNED, (f, bad)
    assert call(ws=4096 + 16) == MISALIGNED
    assert call(size=n.value - 1) == WORKSPACE
    # nothing to do: no pointer is looked at
    assert lib.gr_paged_attention(_attn(num_seqs=0), _lib.PagedAttnIO(), None, 0, None) == 0
    assert lib.gr_paged_attention(_attn(num_tokens=0), _lib.PagedAttnIO(), None, 0, None) == 0


def test_block_table_and_store_arguments():
    lib = _lib.load()
    p = [4096] * 10

    def tables(ptrs=p, **kw):
        d = dict(num_seqs=2, num_tokens=3, num_free=4, block_size=16, max_blocks=5, reserved=0, table_stride=5)
        d.update(kw)
        return lib.gr_extend_block_tables(_lib.BlockTableDesc(*d.values()), *ptrs, None)

    assert lib.gr_extend_block_tables(None, *p, None) == NULL
    for kw in (dict(num_seqs=-1), dict(num_tokens=-1), dict(num_free=-1), dict(block_size=0), dict(max_blocks=-1),
               dict(table_stride=4)):
        assert tables(**kw) == BAD, kw
    for i in range(9):
        if i != 7:                                  # positions may be missing
            assert tables(p[:i] + [None] + p[i + 1:]) == NULL, i

    def store(ptrs=(4096,) * 5, **kw):
        d = dict(num_tokens=1, num_blocks=2, block_size=16, num_heads=2, head_dim=64, elem_bytes=2)
        d.update(kw)
        return lib.gr_store_kv(_lib.KvStoreDesc(*d.values(), *[64] * 14), *ptrs, None, None)

    assert lib.gr_store_kv(None, *p[:5], None, None) == NULL
    for kw in (dict(num_tokens=-1), dict(num_blocks=-1), dict(block_size=0), dict(num_heads=0), dict(head_dim=0)):
        assert store(**kw) == BAD, kw
    assert store(elem_bytes=8) == DTYPE
    assert store(num_tokens=0, ptrs=(None,) * 5) == 0
    for i in range(5):
        assert store(ptrs=[None if j == i else 4096 for j in range(5)]) == NULL


def test_store_refuses_rows_whose_indexes_pass_32_bits():
    # a warp's element index runs up to 31 behind the row
    def status(heads, dim):
        d = _lib.KvStoreDesc(1, 2, 16, heads, dim, 1, *[1] * 14)
        return _lib.load().gr_store_kv(d, None, *(4096,) * 4, None, None)

    for heads, dim in ((1, 2 ** 31 - 1), (2 ** 31 - 1, 1), (2, 2 ** 30), (1, 2 ** 31 - 1023)):
        assert status(heads, dim) == BAD, (heads, dim)
    assert status(1, 2 ** 31 - 1024) == NULL   # the limit itself gets as far as the missing pointer


def test_block_tables_refuse_batches_whose_indexes_pass_32_bits():
    # the request index runs up to 2047 behind the batch
    def status(num_seqs):
        d = _lib.BlockTableDesc(num_seqs, 3, 4, 16, 5, 0, 5)
        return _lib.load().gr_extend_block_tables(d, *[4096] * 4, None, *[4096] * 5, None)

    for n in (2 ** 31 - 1, 2 ** 31 - 2048, 2 ** 31 - 4095):
        assert status(n) == BAD, n
    assert status(2 ** 31 - 4096) == NULL      # the limit itself gets as far as the missing pointer


def test_attention_refuses_batches_whose_indexes_pass_32_bits():
    # the request index runs up to 1023 behind the batch
    n = ctypes.c_size_t(0)
    for r in (2 ** 31 - 1, 2 ** 31 - 1023):
        assert _lib.load().gr_paged_attention_workspace_size(_attn(num_seqs=r), n) == BAD, r
    assert _lib.load().gr_paged_attention_workspace_size(_attn(num_seqs=2 ** 31 - 1024), n) == 0


def test_wrappers_refuse_host_tensors():
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    c = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged_attention(x, c, c, i[None], i[:2], i[:1], 3)
    with pytest.raises(ValueError, match="CUDA"):
        store_kv(x, x, c, c, i.long())
    with pytest.raises(ValueError, match="CUDA"):
        extend_block_tables(i[None], i[:1], i[:1], i, 16, 3)


def test_oracle_masks_by_hand():
    assert ref.seen(2, 3, True).tolist() == [[True, True, False], [True, True, True]]
    assert ref.seen(3, 2, True).tolist() == [[False, False], [True, False], [True, True]]
    assert ref.seen(2, 2, False).all()
    # prefix of 1, tail of 1, two beams of 2
    want = ["110000", "111000", "111100", "110010", "110011"]
    got = ["".join("01"[int(x)] for x in row) for row in ref.seen(5, 6, True, 1, 2)]
    assert got == want


def test_oracle_beam_mask_equals_the_reference_builders_suffixes():
    # a beam's keys behind the cached prefix are exactly the suffix the reference's metadata gathers for it
    from oracle.suffix_kv import suffix_metadata
    for prefix, cached, W, steps, bs in ((24, 16, 5, 3, 16), (40, 40, 3, 1, 16), (9, 0, 4, 2, 16), (33, 20, 6, 4, 16)):
        tail = prefix - cached
        n = tail + W * steps
        mega = [dict(prefix_len=prefix, cache_len=cached, beam_width=W, steps=steps)]
        idx, smo, q_lens, k_lens = suffix_metadata(mega, [0, n], bs)
        mask = ref.seen(n, cached + n, True, tail, steps)
        assert mask[:, :cached].all()
        qa = ka = 0
        for ql, kl in zip(q_lens, k_lens):
            toks, keys = idx[qa:qa + ql], np.asarray(idx)[np.asarray(smo[ka:ka + kl])]
            for i, t in enumerate(toks):
                want = np.zeros(n, bool)
                want[keys[:kl - ql + i + 1]] = True
                assert (mask[t, cached:] == want).all(), (prefix, cached, W, steps, t)
            qa, ka = qa + ql, ka + kl


def test_oracle_attention_against_one_dense_softmax():
    rng = np.random.default_rng(0)
    q = rng.standard_normal((5, 4, 8))
    k, v = rng.standard_normal((6, 8, 2, 8)), rng.standard_normal((6, 8, 2, 8))
    table = np.array([[4, 1], [2, 0]])
    out, lse, absv = ref.attention(q, k, v, table, [0, 2, 5], [13, 3])
    kk = np.concatenate([k[4], k[1]])[:13]
    s = np.einsum("d,kd->k", q[1, 3], kk[:, 1]) / np.sqrt(8)
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(out[1, 3], w @ np.concatenate([v[4], v[1]])[:13, 1])
    assert np.allclose(lse[1, 3], np.log(np.exp(s).sum()))
    assert (absv >= np.abs(out) - 1e-12).all()
    s0 = q[2, 0] @ k[2][0, 0] / np.sqrt(8)
    assert np.allclose(out[2, 0], v[2][0, 0]) and np.isclose(lse[2, 0], s0)


def test_oracle_block_tables_by_hand():
    table = np.array([[7, -1, -1], [-1, -1, -1], [9, 8, -1]])
    t, cu, lens, slots, pos, used, no_block = ref.extend_block_tables(table, [3, 0, 8], [3, 0, 1], [1, 2, 3], 4, 5)
    assert t.tolist() == [[7, 1, -1], [-1, -1, -1], [9, 8, 2]] and used == 2 and not no_block
    assert cu.tolist() == [0, 3, 3, 4] and lens.tolist() == [6, 0, 9]
    assert slots.tolist() == [31, 4, 5, 8, -1] and pos.tolist() == [3, 4, 5, 8, 0]


def _changed_signature(size, stride):
    return None


def _other_answer(size, stride, dtype):
    return torch.empty(1)


@pytest.mark.parametrize("private", [_changed_signature, _other_answer, None])
def test_allocation_without_torchs_private_entry(monkeypatch, private):
    # a torch whose entry is gone, takes other arguments or answers otherwise: the public one is taken
    import importlib.util
    from vllm_gr_ehaleva_b200.attention import paged
    if private is None:
        monkeypatch.delattr(torch._C._dynamo.guards, "_empty_strided_cuda", raising=False)
    else:
        monkeypatch.setattr(torch._C._dynamo.guards, "_empty_strided_cuda", private, raising=False)
    made = []
    monkeypatch.setattr(torch, "empty_strided", lambda *a, **k: made.append((a, k)) or len(made))
    spec = importlib.util.spec_from_file_location(paged.__name__, paged.__file__)
    fresh = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(fresh)
    for i in (1, 2):
        assert fresh._empty((2, 3), (3, 1), torch.int32) == i
    assert made == 2 * [(((2, 3), (3, 1)), dict(dtype=torch.int32, device="cuda"))]
