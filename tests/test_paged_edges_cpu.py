"""Edges of the paged serving tick that show without a GPU."""
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
