"""RotaryEmbedding.forward over no tokens: the heads are counted from the shape, with nothing to infer them from."""
import pytest
import torch

from adallm_b200.rotary_embedding import RotaryEmbedding, get_rope

FORMS = [(128, 128, False), (128, 64, False), (128, 128, True), (256, 64, True)]
SHAPES = [((0,), (0, 4, 0), (0, 1, 0)), ((0,), (0, 0), (0, 0)), ((2, 0), (2, 0, 0), (2, 0, 0)), ((3, 0), (3, 0, 4, 0), (3, 0, 2, 0))]


def inputs(d, shapes, device):
    """Shapes whose last 0 stands for the head size (times four heads where the heads are not apart)."""
    pos, q, k = shapes
    wide = [s[:-1] + (d if len(s) == len(pos) + 2 else 4 * d,) for s in (q, k)]
    return (torch.zeros(pos, dtype=torch.int64, device=device),
            *(torch.zeros(s, dtype=torch.bfloat16, device=device) for s in wide))


@pytest.mark.parametrize("d,r,interleaved", FORMS)
@pytest.mark.parametrize("shapes", SHAPES)
def test_no_tokens_reach_the_call(d, r, interleaved, shapes):
    with pytest.raises(RuntimeError, match="requires CUDA"):
        RotaryEmbedding(d, r, 16, 1e4, interleaved=interleaved)(*inputs(d, shapes, "cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("d,r,interleaved", FORMS)
@pytest.mark.parametrize("shapes", SHAPES)
def test_no_tokens(d, r, interleaved, shapes):
    pos, q, k = inputs(d, shapes, "cuda")
    qo, ko = RotaryEmbedding(d, r, 16, 1e4, interleaved=interleaved).cuda()(pos, q, k)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == ko.dtype == torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("d,r,interleaved", FORMS)
def test_shapes_of_few_tokens(d, r, interleaved):
    """Heads apart or side by side, tokens in one or two dimensions: the same rows."""
    g = torch.Generator().manual_seed(0)
    pos = torch.randint(0, 16, (6,), generator=g).cuda()
    q, k = (torch.randn((6, h, d), generator=g).to(torch.bfloat16).cuda() for h in (4, 1))
    m = RotaryEmbedding(d, r, 16, 1e4, interleaved=interleaved).cuda()
    want = m(pos, q, k)
    assert not torch.equal(want[0], q)
    for a, b, c in ((pos, q.flatten(1), k.flatten(1)), (pos.view(2, 3), q.view(2, 3, 4, d), k.view(2, 3, 1, d)),
                    (pos.view(2, 3), q.view(2, 3, 4 * d), k.view(2, 3, d))):
        qo, ko = m(a, b, c)
        assert qo.shape == b.shape and ko.shape == c.shape
        assert torch.equal(qo.view(6, 4, d), want[0]) and torch.equal(ko.view(6, 1, d), want[1])
    no = q[:, :0].reshape(6, 0, d)
    if r < d or interleaved:  # (without key heads)
        assert torch.equal(m(pos, q, no)[0], want[0])


@pytest.mark.parametrize("d,r,interleaved", FORMS)
def test_get_rope_gives_every_form(d, r, interleaved):
    m = get_rope(d, r, 16, 1e4, None, interleaved)
    assert (m.head_size, m.rotary_dim, m.interleaved) == (d, r, interleaved) and m.cos_sin_cache.shape == (16, 1, r)
    assert get_rope(d, r, 16, 1e4, None, interleaved) is m and get_rope(d, r, 16, 1e4, None, not interleaved) is not m
    assert get_rope(d, r, 16, 1e4).interleaved is False
