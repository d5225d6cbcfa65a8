"""GPU tests of fork_tables' rule for ids that stand in both lists, case by case
as it is documented (test_gpu_page_tables.py holds random ones to a model)."""

import pytest

from tests.test_gpu_page_tables import Model, extend, ints

pytestmark = pytest.mark.gpu

# sequences 0 (20 tokens) and 1 (9 tokens) have some, 2 to 5 none


@pytest.mark.parametrize("seqs,into,made", [
    ([0, 1], [1, 2], []),              # 0 into 1: not empty and in seqs; 1 into 2: 1 stands in into
    ([0, 2], [2, 3], []),              # 0 into 2: in seqs; 2 into 3: 2 stands in into
    ([0, 1], [3, 2], [(0, 3), (1, 2)]),
    ([-1, 0], [0, 2], [(0, 2)]),       # the other pair has an id outside: 0 is nobody's into
    ([1, 0], [9, 2], [(0, 2)]),
    ([6, 0, 0], [2, 2, 3], [(0, 2), (0, 3)]),
    ([0, -1], [2, 3], [(0, 2)]),
    ([2, 1], [-1, 2], []),             # 2 stands in seqs, though that pair has an id outside
    ([0, 1, 0], [2, 2, 3], [(0, 2), (0, 3)]),
    ([0], [0], []), ([2], [2], [])])
def test_ids_in_both_lists(jasper, seqs, into, made):
    m = Model(6, 3, 40, 8)
    extend(jasper, m, [0, 1], [20, 9], 29)
    jasper.fork_tables(*m.gpu, ints(seqs), ints(into), 8)
    lens, tables, refs = list(m.lens), m.tables.copy(), m.refs.copy()
    for s, t in made:
        lens[t], tables[t] = lens[s], tables[s]
        refs[tables[s][tables[s] >= 0]] += 1
    for got, want in zip(m.gpu, (tables, lens, refs)):
        assert got.tolist() == [list(x) for x in want] if got.dim() == 2 else got.tolist() == list(want)
