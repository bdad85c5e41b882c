"""Page tables of pools that are marked a window at a time: a used page must count as used whatever the order in which warps
come through a window.  Every input against the definition, and many runs of each against the first: one lost mark is a page of two rows."""
import numpy as np
import pytest
import torch

from gpu_util import load_executor
from reef_b200 import capi, decode
from test_gpu_decode import I, check_tables, dev, random_rows, tables_by_hand

pytestmark = pytest.mark.gpu


def pool(seed, R, M, S, pages):
    """Rows that use most of the pages, the new tokens going to what is left."""
    rng = np.random.default_rng([seed, R, pages])
    table, lens = random_rows(rng, R, M, S, pages, min(M * S, 9 * pages * S // (10 * R)))
    return table, lens, rng.integers(0, 40, R), np.arange(R) // 2 * 2 if seed % 2 else None


# one window holds 173056 pages (1024 rows) to 202240 (one row): two windows, and as many as there can be
@pytest.mark.parametrize("R,M,S,pages", [(3, 80000, 2, 210000), (40, 8200, 2, 230000), (256, 900, 4, 200000), (1024, 600, 2, 1 << 19)])
def test_pools_of_several_windows(R, M, S, pages):
    for seed in range(4):
        table, lens, new, parent = pool(seed, R, M, S, pages)
        first = check_tables(table, lens, new, parent, pages, S, 20 * R)
        args = [dev(x, I) for x in (table, lens, new)]
        out = decode.PageState(*(None if x is None else torch.empty_like(x) for x in first))
        wrong = torch.zeros((), dtype=I, device="cuda")
        for _ in range(100):
            for x in out:
                if x is not None:
                    x.fill_(-9)
            decode.page_tables(*args, pages=pages, page_size=S, tokens=20 * R, parent=None if parent is None else dev(parent, I), out=out)
            for a, b in zip(out, first):
                if a is not None:
                    wrong += (a != b).any()
        assert wrong.item() == 0
    assert capi.device_error() == 0


@pytest.mark.parametrize("R,M,S,pages", [(40, 8200, 2, 230000), (300, 1500, 2, 1 << 19)])
def test_pools_of_several_windows_in_every_flavour(tmp_path, R, M, S, pages):
    from reef_b200.resources import decoding
    from reef_b200.resources.graph import Graph
    g = Graph("large_tables")
    names = ("table", "lens", "new", "parent", "table_out", "lens_out", "start", "tok", "status", "fork")
    name = decoding.page_tables(R, M, S, pages, 20 * R, fork=True)
    sizes = [b // 4 for b in capi.Kernel(name).arg_bytes]
    bufs = [g.input(n, sizes[i], "int32") if i < 4 else g.add_storage("output" if n == "table_out" else n, sizes[i], "int32") for i, n in enumerate(names)]
    g.kernel(name, bufs)
    e = load_executor(g.write(str(tmp_path), capi.plan_fn), params=False)
    for seed in (1, 3):
        table, lens, new, parent = pool(seed, R, M, S, pages)
        want = tables_by_hand(table, lens, new, parent, pages, S, 20 * R)
        for n, v in zip(names, (table, lens, new, parent)):
            e.set_input(n, v.astype(np.int32))
        for run in (e.execute, e.execute_graph, e.execute_preemptable, e.execute_dispatch) * 3:
            run()
            for b, n, y in zip(bufs[4:], sizes[4:], want):
                assert np.array_equal(e.get_data(b, 4 * n, np.int32), y.ravel())
    assert capi.device_error() == 0
    e.close()
