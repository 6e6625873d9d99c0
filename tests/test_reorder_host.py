"""Reorders of more sequences than one launch's arguments name copies for (sllm_gfx950_attn.h),
on the CPU against the HIP stand-in of tests/fakehip: a reorder that fails has copied nothing,
so that what it gives back is as it was."""
import pytest

from test_attn_host import F32, HIP, I, Cache, L  # noqa: F401  (the fixture)


@pytest.mark.parametrize("dtype", [F32, 4])
@pytest.mark.parametrize("n", [2, 321, 322, 700])
def test_all_copies_or_none(amd, L, dtype, n):
    """Every page in use, so that all copies go to pages that the call itself freed."""
    c = Cache(amd, L, n_pages=n, dtype=dtype, kv=1, layers=1)
    ids = [c.new() for _ in range(n)]
    c.grow(ids, [5] * n)
    was, parent = c.state(ids), I(*[n // 2] * n)
    for skip in range(50):
        L.fakehip_clear()
        L.fakehip_fail(b"*", 999, skip)
        st = L.sllm_gfx950_seq_reorder(c.p, I(*ids), parent, n)
        copies = [x for x in L.fakehip_launches().decode().split() if "copy" in x]
        if not L.fakehip_fired():
            break
        assert st == HIP and copies == [] and c.state(ids) == was, skip
    L.fakehip_clear()
    assert st == 0 and len(copies) == 1
    used, tables = c.state(ids)
    assert used == n and len({t[0] for _, t in tables}) == n and tables[n // 2] == was[1][n // 2]
    c.close()
    assert L.fakehip_live() >= 0


def test_a_list_of_copies_beside_batches(amd, L):
    """The list's memory is a batch's that ended, and a later batch's."""
    n = 400
    c = Cache(amd, L, n_pages=2 * n, kv=1, layers=1)
    ids = [c.new() for _ in range(n)]
    for step in range(4):
        c.grow(ids, [3] * n)
        live = L.fakehip_live()
        assert L.sllm_gfx950_seq_reorder(c.p, I(*ids), I(*[(7 * i + step) % n // 2 for i in range(n)]), n) == 0
        assert L.fakehip_live() <= live + 3
    c.close()
