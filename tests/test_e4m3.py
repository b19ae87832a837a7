"""The e4m3 cache without a GPU: codec model, layout, pool refusals."""
import numpy as np
import pytest

import _e4m3 as M
import tge_kv as tk
from test_host_plan import build_and_run

PLAN_CHECK = ["aegean-tge_amd/host/plan.cpp", "aegean-tge_amd/host/plan_e4m3.cpp", "tests/native/plan_e4m3_check.cpp"]


def test_model_codec():
    assert M.POSITIVE[126] == 448.0 and M.POSITIVE[1] == 2.0 ** -9 and len(set(M.POSITIVE)) == 127
    for c in range(127):
        assert M.encode(M.POSITIVE[c]) == c and M.encode(-M.POSITIVE[c]) == c + 128
    mid = (M.POSITIVE[:-1] + M.POSITIVE[1:]) / 2
    assert (M.encode(mid) % 2 == 0).all()
    assert M.encode(1e30) == 126 and M.encode(-np.inf) == 254 and M.encode(np.nan) == 0


@pytest.mark.parametrize("width", [64, 128, 256])
def test_layout_is_a_bijection(tk, width):
    index = tk.lib().tge_kv_e4m3_index
    for part in range(2):
        at = sorted(index(part, t, d, width) for t in range(16) for d in range(width))
        assert at == list(range(16 * width))
    for args in [(2, 0, 0, width), (0, 16, 0, width), (0, -1, 0, width), (0, 0, width, width), (1, 0, 0, 96)]:
        assert index(*args) == -1


@pytest.mark.parametrize("width", [64, 128, 256])
def test_layout_follows_the_formulas(tk, width):
    for t in range(16):
        for d in range(width):
            lane, j = (d // 16) % 4 * 16 + t, d // 64 * 16 + d % 16
            assert tk.lib().tge_kv_e4m3_index(0, t, d, width) == j // 16 * 1024 + lane * 16 + j % 16
            lane, j = t // 4 * 16 + d % 16, d // 16 % 2 * (width // 8) + d // 32 * 4 + t % 4
            assert tk.lib().tge_kv_e4m3_index(1, t, d, width) == j // 16 * 1024 + lane * 16 + j % 16


@pytest.mark.parametrize("head_dim", [0, -8, 4, 12, 100, 264])
def test_pool_refuses_head_sizes(tk, head_dim):
    with pytest.raises(tk.TgeError) as e:
        tk.KvPool(1, 4, 2, head_dim, tk.KV_E4M3)
    assert e.value.status == tk.ERR_INVALID


def test_pool_refuses_more_blocks_than_int(tk):
    with pytest.raises(tk.TgeError) as e:
        tk.KvPool(1, 1 << 30, 8, 64, tk.KV_E4M3)
    assert e.value.status == tk.ERR_INVALID


def test_calls_refuse_null(tk):
    L = tk.lib()
    assert L.tge_kv_append_rows(None, None, 0, None, None) == tk.ERR_INVALID
    assert L.tge_attention_rows(None, None, 0, None, None) == tk.ERR_INVALID
    assert L.tge_qwen2_kv_layer_rows(None, 0, None, None, None) == tk.ERR_INVALID


def test_plans_under_sanitizers(tmp_path):
    assert "plan_e4m3_check ok" in build_and_run(tmp_path, "plan_e4m3_check", PLAN_CHECK)


def test_plans_of_the_long_items(tmp_path):
    """The GPU tests' long items are what they are named for."""
    out = build_and_run(tmp_path, "plan_e4m3_check", PLAN_CHECK, M.LONG_ITEMS)
    for (case, rw), line in zip(M.LONG_ITEMS.items(), out.splitlines(), strict=True):
        p = dict(zip(line.split()[::2], map(int, line.split()[1::2])))
        assert p["longest"] > 1024 and p["rw"] == rw, (case, line)
