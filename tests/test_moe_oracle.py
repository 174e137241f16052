"""The oracle's sort by expert against the definition taken entry by entry."""
import pytest
import torch

from oracle import formulas


@pytest.mark.parametrize("T,k,E,block,rows", [(1, 1, 1, 1, 1), (40, 3, 7, 1, 120), (40, 3, 7, 8, 168), (40, 3, 7, 8, 64), (64, 4, 3, 16, 400)])
@pytest.mark.parametrize("seed", [0, 1])
def test_route_oracle_is_the_definition(T, k, E, block, rows, seed):
    """c_e entries ask for expert e; e's rows start behind ceil(c_f / block) * block rows for each f < e; an entry's row is
    that start plus the number of earlier entries of its expert, unless it reaches the end of the buffer."""
    g = torch.Generator().manual_seed(seed + T * E)
    ids = torch.randint(-1, E + 1, (T, k), generator=g, dtype=torch.int32)
    row_of, entry_of, offsets = formulas.moe_route_ref(ids, E, block, rows)
    flat = ids.flatten()
    start = [sum(-(-int((flat == f).sum()) // block) * block for f in range(e)) for e in range(E + 1)]
    assert offsets.tolist() == [min(s, rows) for s in start]
    owner = {}
    for i, e in enumerate(flat.tolist()):
        row = start[e] + int((flat[:i] == e).sum()) if 0 <= e < E else rows
        row = row if row < rows else -1
        assert int(row_of.flatten()[i]) == row
        if row >= 0:
            owner[row] = i
    assert entry_of.tolist() == [owner.get(r, -1) for r in range(rows)]
