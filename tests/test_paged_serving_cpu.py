"""Refusals of the paged serving tick's entry points: checked on the host before
any CUDA call, so they run without a GPU; and the reference of its GPU tests
on cases worked out by hand."""
import ctypes

import numpy as np
import pytest
import torch

import paged_reference as ref
from infercache_b200 import _lib

INVALID, UNSUPPORTED = _lib.IC_ERR_INVALID_ARG, _lib.IC_ERR_UNSUPPORTED


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


@pytest.fixture(scope="module")
def p():
    buf = (ctypes.c_int64 * 1024)()
    p.buf = buf
    return (ctypes.addressof(buf) + 63) // 64 * 64


def expect(lib, name, cls, base, bad, want=INVALID):
    args = cls(**{**base, **bad})
    assert getattr(lib, name)(ctypes.byref(args), None) == want, (name, bad)


def test_plan_and_release_refusals(lib, p):
    base = dict(lens=p, counts=p, block_table=p, free_pages=p, free_count=p, q_start=p, slots=p, positions=p, lens_out=p,
                free_count_out=p, workspace=p, num_sessions=2, width=4, total=8, free_capacity=9)
    for bad in ([{k: 0} for k in ("lens", "counts", "block_table", "free_pages", "free_count", "q_start", "slots",
                                  "positions", "lens_out", "free_count_out", "workspace", "num_sessions", "width")]
                + [dict(total=-1), dict(free_capacity=-1), dict(num_sessions=-3)]):
        expect(lib, "ic_page_plan", _lib.ic_page_plan_args, base, bad)
    expect(lib, "ic_page_plan", _lib.ic_page_plan_args, base, dict(num_sessions=8193), UNSUPPORTED)
    expect(lib, "ic_page_plan", _lib.ic_page_plan_args, base, dict(width=(1 << 26) + 1), UNSUPPORTED)
    base = dict(lens=p, keep=p, block_table=p, free_pages=p, free_count=p, num_sessions=2, width=4, free_capacity=9)
    for bad in ([{k: 0} for k in ("lens", "keep", "block_table", "free_pages", "free_count", "num_sessions", "width")]
                + [dict(free_capacity=-1)]):
        expect(lib, "ic_page_release", _lib.ic_page_release_args, base, bad)


@pytest.mark.parametrize("name", ["ic_page_write_q8", "ic_page_read_q8"])
def test_page_rows_refusals(lib, p, name):
    def pool(**kw):
        return _lib.ic_pool(**{**dict(k=p, v=p, pool_tokens=64, num_layers=2, num_kv_heads=1, head_dim=128, dtype=_lib.IC_I8), **kw})

    def rows(**kw):
        d = dict(page_ids=p, n_page_ids=2, k_buf=p, v_buf=p, start_token=0, n_tokens=8, stride_l=2048, stride_h=2048,
                 stride_t=128)
        return (_lib.ic_page_q8_rows * 1)(_lib.ic_page_q8_rows(**{**d, **kw}))

    base = dict(pool=pool(), k_scale=p, v_scale=p, rows=rows(), count=1, layer_begin=0, layer_end=2, buf_dtype=_lib.IC_F16)
    for bad in (dict(k_scale=0), dict(v_scale=0), dict(rows=None), dict(count=0), dict(count=33), dict(layer_begin=-1),
                dict(layer_end=3), dict(layer_begin=2, layer_end=1), dict(buf_dtype=7), dict(buf_dtype=_lib.IC_I8),
                dict(pool=pool(k=0)), dict(pool=pool(dtype=_lib.IC_F16)), dict(pool=pool(pool_tokens=40)),
                dict(pool=pool(pool_tokens=0)), dict(pool=pool(pool_tokens=2 ** 31)), dict(pool=pool(num_kv_heads=40000)),
                dict(pool=pool(k=p + 8)), dict(rows=rows(n_tokens=-1)), dict(rows=rows(k_buf=0)),
                dict(rows=rows(page_ids=0)), dict(rows=rows(start_token=-1)), dict(rows=rows(start_token=25)),
                dict(rows=rows(stride_t=129)), dict(rows=rows(v_buf=p + 2))):
        expect(lib, name, _lib.ic_page_q8_args, base, bad)
    expect(lib, name, _lib.ic_page_q8_args, base, dict(pool=pool(head_dim=96)), UNSUPPORTED)
    for nothing in (dict(rows=rows(n_tokens=0)), dict(layer_end=0)):
        expect(lib, name, _lib.ic_page_q8_args, base, nothing, _lib.IC_OK)


def test_attention_refusals(lib, p):
    base = dict(q=p, out=p, k=p, v=p, k_scale=p, v_scale=p, block_table=p, lens=p, q_start=p, workspace=p,
                workspace_bytes=1 << 40, pool_tokens=64, q_stride_t=1024, q_stride_h=128, num_sessions=2, table_width=4000,
                num_q_tokens=3, max_count=3, num_q_heads=8, num_kv_heads=2, head_dim=128, q_dtype=_lib.IC_F16,
                code_dtype=_lib.IC_E4M3, scale=0.1)  # a wide table: the shares of a line, which need workspace
    cls = _lib.ic_paged_attn_args
    need = lib.ic_paged_attention_workspace(ctypes.byref(cls(**base)))
    assert need > 0 and lib.ic_paged_attention_workspace(None) == 0
    for bad in ([{k: 0} for k in ("q", "out", "k", "v", "k_scale", "v_scale", "block_table", "lens", "q_start", "workspace",
                                  "num_sessions", "num_q_tokens", "num_q_heads", "num_kv_heads", "pool_tokens")]
                + [dict(table_width=-1), dict(max_count=-1), dict(num_q_heads=7), dict(pool_tokens=40),
                   dict(pool_tokens=2 ** 31), dict(q_stride_t=-8), dict(q_stride_h=4), dict(q_dtype=_lib.IC_F32),
                   dict(code_dtype=_lib.IC_F16), dict(q=p + 8), dict(out=p + 2), dict(k=p + 4), dict(workspace=p + 4),
                   dict(workspace_bytes=need - 1), dict(table_width=(1 << 26) + 1)]):
        expect(lib, "ic_paged_attention", cls, base, bad)
    assert lib.ic_paged_attention_workspace(ctypes.byref(cls(**{**base, "table_width": 4, "max_count": 1}))) == 0
    for bad in (dict(head_dim=96), dict(num_sessions=4097), dict(table_width=1 << 26, num_q_tokens=1000)):
        expect(lib, "ic_paged_attention", cls, base, bad, UNSUPPORTED)
        assert lib.ic_paged_attention_workspace(ctypes.byref(cls(**{**base, **bad}))) == 0


def test_logits_refusals(lib, p):
    base = dict(logits=p, out=p, logits_stride=40, out_stride=40, tokens=p, bias_ids=p, bias_values=p, mask=p,
                tokens_stride=5, bias_stride=4, mask_stride=2, rows=2, vocab=40, dtype=_lib.IC_F32, max_tokens=5,
                bias_width=4)
    for bad in (dict(logits=0), dict(out=0), dict(rows=-1), dict(vocab=0), dict(max_tokens=-1), dict(bias_width=-1),
                dict(bias_values=0), dict(logits_stride=39), dict(out_stride=39), dict(tokens_stride=4),
                dict(bias_stride=3), dict(mask_stride=1), dict(dtype=_lib.IC_I8)):
        expect(lib, "ic_process_logits", _lib.ic_logits_args, base, bad)
    expect(lib, "ic_process_logits", _lib.ic_logits_args, base, dict(rows=65536), UNSUPPORTED)
    expect(lib, "ic_process_logits", _lib.ic_logits_args, base, dict(rows=0), _lib.IC_OK)


def test_16_bit_verbs_refuse_8_bit_pools(lib, p):
    pool = _lib.ic_pool(k=p, v=p, pool_tokens=64, num_layers=1, num_kv_heads=1, head_dim=128, dtype=_lib.IC_I8)
    a = _lib.ic_page_rows_args(pool=pool, page_ids=p, n_page_ids=2, layer_begin=0, layer_end=1, start_token=0, n_tokens=4,
                               k_buf=p, v_buf=p, stride_l=512, stride_h=512, stride_t=128)
    for name in ("ic_page_gather", "ic_page_write"):
        assert getattr(lib, name)(ctypes.byref(a), None) == UNSUPPORTED
    from infercache_b200 import CacheConfig
    from infercache_b200.hierarchical_cache import _check_cfg
    with pytest.raises(ValueError):
        _check_cfg(CacheConfig(num_layers=1, num_kv_heads=1, head_dim=128, dtype=torch.int8))


def test_ops_run_on_cuda_tensors_only():
    from infercache_b200 import page_plan, process_logits
    z = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        page_plan(z, z, z[None], z, z[:1], 0)
    with pytest.raises(ValueError):
        process_logits(torch.zeros(1, 8))


def test_reference_rounds_and_plans_as_worked_out_by_hand():
    e4m3, i8 = torch.float8_e4m3fn, torch.int8
    x = np.array([17.0, 18.0, 19.0, 0.0029296875, 0.001, 460.0, -2.5])
    assert ref.round_code(x, e4m3).tolist() == [16.0, 18.0, 20.0, 0.00390625, 0.001953125, 448.0, -2.5]
    assert ref.round_code(np.array([0.5, 1.5, -2.5, 127.4, 500.0]), i8).tolist() == [0.0, 2.0, -2.0, 127.0, 127.0]
    t = torch.linspace(-448, 448, 40001)  # 32-bit values, so that the cast rounds once
    assert np.array_equal(ref.round_code(t.double().numpy(), e4m3), t.to(e4m3).double().numpy())
    assert [ref.exponent(a, i8) for a in (0.0, 127.0, 127.0001, 1.0, 1e300)] == [-60, 0, 1, -6, 60]
    assert [ref.exponent(a, e4m3) for a in (448.0, 449.0, 1.0)] == [0, 1, -8]
    got = ref.plan([15, 0], [2, 3], [[4, -1], [-1, -1]], [7, 8, 9], 3, 5)
    assert got == ([0, 2, 5], [79, 144, 128, 129, 130], [15, 16, 0, 1, 2], [17, 3], 1, [[4, 9], [8, -1]], [])
    assert ref.release([17, 3], [1, 0], [[4, 9], [8, -1]], [7, 0, 0], 1) == ([1, 0], [[4, -1], [-1, -1]], [7, 8, 9])
