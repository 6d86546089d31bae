"""Steps behind one whose pages ran out: what an earlier request left in a table row is nobody's page."""
import pytest
import torch

from adallm_b200.step_metadata import step_metadata
from oracle import kv4
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def run(cached, new, tables, free, start, page, tokens):
    i32 = dict(dtype=torch.int32, device=dev())
    err = torch.zeros(1, **i32)
    m = step_metadata(torch.tensor(cached, **i32), torch.tensor(new, **i32), tables, torch.tensor(free, **i32),
                      torch.tensor([start], **i32), page, tokens, err=err)
    return m, int(err)


def test_pages_that_ran_out_are_none_in_later_steps():
    """Two rows that were used before (9s): the first page needed is there, the others are not."""
    page = 16
    rows = [[5, 9, 9, 9], [9, 9, 9, 9]]
    tables = torch.tensor(rows, dtype=torch.int32, device=dev())
    cached, new, free = [16, 0], [20, 17], [7]
    m, err = run(cached, new, tables, free, 0, page, 37)
    assert err == 0x100
    assert tables.tolist() == [[5, 7, -1, 9], [-1, -1, 9, 9]]
    assert m.slot_mapping.tolist() == [*range(112, 128)] + [-1] * 21
    want = kv4.step_metadata(cached, new, rows, free, 0, page, 37)
    assert tables.tolist() == want[6] and m.slot_mapping.tolist() == want[1]
    lens, at, rows = want[4], want[5], want[6]
    for _ in range(20):  # (both reach into columns that they do not have, and past them)
        m, err = run(lens, [1, 1], tables, free, at, page, 2)
        _, slots, _, _, lens, at, rows, bits = kv4.step_metadata(lens, [1, 1], rows, free, at, page, 2)
        assert m.slot_mapping.tolist() == slots == [-1, -1] and tables.tolist() == rows and err == bits
    assert max(max(r) for r in rows) == 9 and rows[0][:3] == [5, 7, -1] and rows[1][:3] == [-1, -1, -1]


def test_a_start_outside_the_list():
    """Before it or behind it there is no page; the table says so."""
    for start in (-3, 2, 2 ** 31 - 1):
        tables = torch.full((1, 3), 9, dtype=torch.int32, device=dev())
        m, err = run([0], [33], tables, [4, 6], start, 16, 33)
        want = kv4.step_metadata([0], [33], [[9, 9, 9]], [4, 6], start, 16, 33)
        assert tables.tolist() == want[6] and m.slot_mapping.tolist() == want[1] and err == want[7] == 0x100
        assert int(m.free_next) == want[5]
        if start > 0:
            assert tables.tolist() == [[-1, -1, -1]]
