"""bench.py's measurement of the paged KV cache on the GPU."""
import argparse
import json

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

import bench  # noqa: E402
from vllm_gr_ehaleva_b200 import attention  # noqa: E402


def test_the_cache_write_is_timed_on_rows_of_its_own_for_k_and_v(monkeypatch, capsys):
    # with one tensor for both, a row's second read comes from the chip and not from memory
    seen = []
    store = attention.store_kv

    def record(k, v, k_cache, v_cache, slots):
        seen.append(len({x.untyped_storage().data_ptr() for x in (k, v, k_cache, v_cache)}))
        return store(k, v, k_cache, v_cache, slots)

    monkeypatch.setattr(attention, "store_kv", record)
    bench.run_paged(argparse.Namespace(steps=1, warmup=3))
    lines = [json.loads(x) for x in capsys.readouterr().out.splitlines()]
    assert [x["batch"] for x in lines] == ["single_tokens", "prompt", "beams"]
    assert all(x["store_ms"] > 0 and x["value"] > 0 for x in lines)
    assert seen and set(seen) == {4}
