"""A step's metadata built on the GPU against host lists (oracle/kv4.py): all values are whole numbers and
must be equal."""
import random

import pytest
import torch

from adallm_b200.step_metadata import StepMetadata, empty_step_metadata, step_metadata
from oracle import kv4
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def _case(seed, requests, new_hi, cached_hi, page, width=None, spare=3, start=2, zeros=True):
    r = random.Random(seed)
    cached = [r.randint(0, cached_hi) for _ in range(requests)]
    new = [r.randint(0 if zeros else 1, new_hi) for _ in range(requests)]
    most = max([1] + [-(-(c + n) // page) for c, n in zip(cached, new)])
    width = most + 1 if width is None else width
    pages = list(range(1, 4000 + sum(-(-c // page) for c in cached) + requests * (new_hi // page + 2)))
    r.shuffle(pages)
    tables = [[pages.pop() if i < -(-c // page) else -1 for i in range(width)] for c in cached]
    take = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new))
    return cached, new, tables, pages[:start + take + spare], start, page


def _run(case, tokens, out=None, tables=None):
    cached, new, table_list, free, start, page = case
    d = dev()
    i32 = dict(dtype=torch.int32, device=d)
    if tables is None:
        tables = torch.tensor(table_list, **i32).reshape(len(cached), -1)
    err = torch.zeros(1, **i32)
    m = step_metadata(torch.tensor(cached, **i32), torch.tensor(new, **i32), tables, torch.tensor(free, **i32),
                      torch.tensor([start], **i32), page, tokens, out=out, err=err)
    torch.cuda.synchronize()
    return m, tables, int(err)


def _check(case, tokens, m, tables, err):
    pos, slots, cu_q, cu_k, context, nxt, want, want_err = kv4.step_metadata(*case, tokens)
    assert m.positions.tolist() == pos
    assert m.slot_mapping.tolist() == slots
    assert m.cu_seqlens_q.tolist() == cu_q
    assert m.cu_seqlens_k.tolist() == cu_k
    assert m.context_lens.tolist() == context
    assert m.free_next.tolist() == [nxt]
    assert tables.tolist() == want
    assert err == want_err


@pytest.mark.parametrize("seed,requests,new_hi,cached_hi,page,pad", [
    (1, 1, 1, 0, 16, 0), (2, 1, 1, 700, 16, 63), (3, 16, 1, 300, 16, 5), (4, 33, 40, 100, 32, 1),
    (5, 513, 9, 50, 16, 100), (6, 1025, 3, 20, 48, 0), (7, 7, 5000, 5000, 256, 11), (8, 64, 2, 1000, 1, 3)])
def test_matches_host_lists(seed, requests, new_hi, cached_hi, page, pad):
    case = _case(seed, requests, new_hi, cached_hi, page)
    tokens = sum(case[1]) + pad
    _check(case, tokens, *_run(case, tokens))


def test_largest_batch():
    case = _case(9, 8192, 2, 40, 16)
    tokens = sum(case[1])
    _check(case, tokens, *_run(case, tokens))


def test_the_same_inputs_give_the_same_outputs_again():
    case = _case(10, 40, 30, 100, 16)
    tokens = sum(case[1]) + 7
    out = empty_step_metadata(40, tokens, dev())
    m, tables, err = _run(case, tokens, out)
    again, tables, err2 = _run(case, tokens, out, tables)
    assert again.positions.data_ptr() == out.positions.data_ptr() and err == err2 == 0
    _check(case, tokens, again, tables, err2)


def test_free_list_at_its_end():
    cached, new, tables, free, start, page = _case(11, 20, 60, 100, 16, spare=0)
    case = (cached, new, tables, free[:-5], start, page)
    tokens = sum(new)
    m, t, err = _run(case, tokens)
    assert err == 0x100 and int(m.free_next) == len(free) - 5
    _check(case, tokens, m, t, err)
    case = (cached, new, tables, [], 0, page)
    m, t, err = _run(case, tokens)
    _check(case, tokens, m, t, err)


def test_table_too_narrow():
    case = _case(12, 9, 100, 60, 16, width=4, zeros=False)
    cached = [min(c, 64) for c in case[0]]
    case = (cached, *case[1:])
    tokens = sum(case[1])
    m, t, err = _run(case, tokens)
    assert err & 0x200
    _check(case, tokens, m, t, err)


def test_more_tokens_than_laid_out_for():
    case = _case(13, 9, 100, 60, 16)
    tokens = sum(case[1]) - 31
    m, t, err = _run(case, tokens)
    assert err == 0x400
    _check(case, tokens, m, t, err)
    m, t, err = _run(case, 0)
    assert err == 0x400 and m.positions.numel() == 0


def test_negative_and_zero_lengths_and_no_request():
    case = _case(14, 6, 5, 40, 16)
    case = ([-3, *case[0][1:]], [*case[1][:5], -7], [[-1] * len(case[2][0]), *case[2][1:]], *case[3:])
    case[2][5] = list(case[2][5])
    tokens = 40
    _check(case, tokens, *_run(case, tokens))
    case = ([], [], [], [5, 6, 7], 1, 16)
    d = dev()
    m, t, err = _run(case, 4, tables=torch.empty((0, 3), dtype=torch.int32, device=d))
    assert m.positions.tolist() == [0] * 4 and m.slot_mapping.tolist() == [-1] * 4
    assert m.cu_seqlens_q.tolist() == [0] == m.cu_seqlens_k.tolist() and int(m.free_next) == 1 and err == 0


def test_hole_in_a_table_and_far_slots():
    d = dev()
    i32 = dict(dtype=torch.int32, device=d)
    big = (2 ** 31 - 1) // 256
    tables = torch.tensor([[3, -1], [big - 1, -1], [big + 1, -1]], **i32)
    err = torch.zeros(1, **i32)
    m = step_metadata(torch.tensor([20, 250, 250], **i32), torch.tensor([1, 1, 1], **i32), tables,
                      torch.tensor([9], **i32), torch.tensor([0], **i32), 256, 3, err=err)
    assert m.slot_mapping.tolist() == [3 * 256 + 20, (big - 1) * 256 + 250, -1] and int(err) == 0x400
    tables = torch.tensor([[-1, 7]], **i32)
    m = step_metadata(torch.tensor([10], **i32), torch.tensor([1], **i32), tables, torch.tensor([9], **i32),
                      torch.tensor([0], **i32), 16, 1)
    assert m.slot_mapping.tolist() == [-1]


def test_strided_table_and_captured_decode_steps():
    """Steps replayed from a graph with the copies that feed the next one."""
    d = dev()
    i32 = dict(dtype=torch.int32, device=d)
    cached0, page, steps = [15, 0, 31, 40], 16, 40
    wide = torch.full((4, 12), -1, **i32)
    tables = wide[:, 2:10]
    for b, c in enumerate(cached0):
        for j in range(-(-c // page)):
            tables[b, j] = 10 * b + j
    cached, new, start = torch.tensor(cached0, **i32), torch.ones(4, **i32), torch.zeros(1, **i32)
    free = torch.arange(100, 140, **i32)
    out = empty_step_metadata(4, 8, d)
    first = tables.clone()

    def step():
        step_metadata(cached, new, tables, free, start, page, 8, out=out)
        cached.copy_(out.context_lens)
        start.copy_(out.free_next)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step()
    lens, at, want = list(cached0), 0, first.tolist()
    for _ in range(steps):
        g.replay()
        torch.cuda.synchronize()
        pos, slots, _, _, lens, at, want, _ = kv4.step_metadata(lens, [1] * 4, want, free.tolist(), at, page, 8)
        assert out.positions.tolist() == pos and out.slot_mapping.tolist() == slots
        assert tables.tolist() == want and cached.tolist() == lens and int(start) == at
    assert (wide[:, :2] == -1).all() and (wide[:, 10:] == -1).all()


def test_refusals():
    d = dev()
    i32 = dict(dtype=torch.int32, device=d)
    a = [torch.tensor([3, 4], **i32), torch.tensor([1, 1], **i32), torch.zeros((2, 4), **i32),
         torch.arange(9, **i32), torch.zeros(1, **i32), 16, 8]

    def bad(i, value, **kw):
        args = list(a)
        args[i] = value
        with pytest.raises(ValueError):
            step_metadata(*args, **kw)

    bad(0, a[0].long())
    bad(1, torch.ones(3, **i32))
    bad(2, torch.zeros((3, 4), **i32))
    bad(2, torch.zeros((2, 4), **i32).t().contiguous().t())
    bad(2, torch.zeros((1, 4), **i32).expand(2, 4))  # rows that share their pages' memory
    bad(3, torch.arange(18, **i32)[::2])
    bad(4, torch.zeros(2, **i32))
    bad(5, 0)
    bad(6, -1)
    out = empty_step_metadata(2, 8, d)
    bad(6, 7, out=out)
    with pytest.raises(ValueError):  # an output that is an input
        step_metadata(*a, out=out._replace(free_next=a[4]))
    with pytest.raises(ValueError):
        step_metadata(*a, out=out._replace(context_lens=a[0]))
    many = torch.zeros(8193, **i32)
    with pytest.raises(ValueError):
        step_metadata(many, many, torch.zeros((8193, 1), **i32), a[3], a[4], 16, 8)
    with pytest.raises(RuntimeError):
        step_metadata(a[0].cpu(), *a[1:])
    assert isinstance(step_metadata(*a, out=tuple(out)), StepMetadata)
