"""Edges of the paged serving tick that show without a GPU."""
import pytest
import torch


def test_batch_counts_beyond_32_bits_stay_beyond_every_session():
    from infercache_b200 import PagedBatch
    b = PagedBatch.__new__(PagedBatch)
    b.max_sessions, b.device = 6, torch.device("cpu")
    big = 2 ** 32
    got = b._ints("keep", torch.tensor([big, big + 7, -big + 7, 5, 2 ** 63 - 1, -2 ** 63]))
    assert got.dtype == torch.int32
    assert got.tolist() == [2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, 5, 2 ** 31 - 1, -2 ** 31]


def test_smoke_as_a_script_finds_every_part():
    """What the script's last lines call has been defined by then."""
    import ast
    from pathlib import Path
    body = ast.parse((Path(__file__).resolve().parents[1] / "__graft_entry__.py").read_text()).body
    guard = [i for i, x in enumerate(body) if isinstance(x, ast.If)]
    defs = [i for i, x in enumerate(body) if isinstance(x, ast.FunctionDef)]
    assert len(guard) == 1 and guard[0] > max(defs)


def attention_args(**kw):
    import ctypes
    from infercache_b200 import _lib
    buf = ctypes.create_string_buffer(64)
    p = (ctypes.addressof(buf) + 15) // 16 * 16  # never read: the workspace's size alone is asked for
    base = dict(q=p, out=p, k=p, v=p, k_scale=p, v_scale=p, block_table=p, lens=p, q_start=p, pool_tokens=2 ** 20,
                q_stride_t=4096, q_stride_h=128, num_sessions=1, table_width=8192, num_q_heads=32, num_kv_heads=8, head_dim=128,
                q_dtype=_lib.IC_F16, code_dtype=_lib.IC_E4M3, scale=0.1)
    base.update(kw)
    base.setdefault("max_count", base["num_q_tokens"])
    return _lib.ic_paged_attn_args(**base)


def attention_takes(**kw):
    import ctypes
    from infercache_b200 import _lib
    return _lib.load().ic_paged_attention_workspace(ctypes.byref(attention_args(**kw))) > 0


def test_attention_takes_long_prompts_under_wide_tables():
    """The table's width bounds the streaming kernel's work, not the tile kernel's."""
    assert attention_takes(num_q_tokens=65_300)
    assert attention_takes(num_q_tokens=131_072, head_dim=256)
    assert attention_takes(num_q_tokens=200_000, num_sessions=64, max_count=130_000)
    assert not attention_takes(num_q_tokens=65_300, max_count=1)               # all of it the streaming kernel's
    assert not attention_takes(num_q_tokens=2 ** 29)                           # 2^31 rows per KV head
    assert not attention_takes(num_q_tokens=2 ** 26, num_q_heads=8192, num_kv_heads=8192, table_width=64)


def test_page_ids_reach_the_kernels_as_int32_on_the_pools_device():
    """A host or int64 tensor's address would be read as if it were neither."""
    from infercache_b200 import PagePool
    pool = PagePool.__new__(PagePool)
    pool.K = torch.empty(0, device="meta")
    ready = torch.empty(4, dtype=torch.int32, device="meta")
    assert pool._page_ids(ready) is ready
    for ids in (torch.arange(4), torch.arange(4, dtype=torch.int32), ready.long(), ready[::2], [1, 2, 3]):
        got = pool._page_ids(ids)
        assert got.dtype == torch.int32 and got.device == pool.device and got.is_contiguous()
    pool.K = torch.empty(0)
    assert pool._page_ids(torch.tensor([3, 2 ** 32 + 1, -2 ** 40])).tolist() == [3, 2 ** 31 - 1, -2 ** 31]


@pytest.mark.parametrize("missing", ["cuda", "headers"])
def test_library_builds_without_what_the_binding_needs(missing, monkeypatch, capsys):
    from pathlib import Path
    from infercache_b200 import build
    before = build.BINDING.stat().st_mtime_ns
    if missing == "cuda":
        monkeypatch.setattr(torch.version, "cuda", None)
    else:
        monkeypatch.setattr(build, "_python_include", lambda: Path("/nonexistent"))
    assert build.build() == build.LIB
    assert "binding is not built" in capsys.readouterr().err
    assert build.BINDING.stat().st_mtime_ns == before


def test_binding_is_rebuilt_for_another_torch(monkeypatch):
    from infercache_b200 import _lib, build
    build.build()
    ran = []

    class Done:
        returncode = 1
        stdout = stderr = ""

    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: ran.append(cmd) or Done)
    assert build.build_binding() == build.BINDING and not ran
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    with pytest.raises(RuntimeError):  # it set out to compile
        build.build_binding()
    assert len(ran) == 1
    monkeypatch.setattr(_lib, "_BINDING", None)
    with pytest.raises(ImportError, match="9.9.9"):
        _lib.binding()
