"""token_log_probs at logits and scales near the ends of f32, and its outputs
as tensors that a program keeps."""
import io

import pytest
import torch

from tests._paged import U32, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [50, 8194, 40000])
@pytest.mark.parametrize("size,scale", [(3e38, 1e-38), (2.0 ** 127, 2.0 ** -125), (1e38, 2.5e-38), (1e-30, 1e30), (1e-38, 2.0 ** 125)])
def test_far_logits_of_a_small_scale(cbx, vocab, size, scale):
    """Logits of both signs whose difference passes the largest f32, and
    differences of 1e-38 under a scale that makes them count.  z carries 3
    roundings of at most 2 |scale x|, an exponential 4 more, their sum V, the
    logarithm 2 of log V."""
    g = gen(50 + vocab)
    x = (torch.rand(5, vocab, device="cuda", generator=g) * 2 - 1) * size
    x[:, 7], x[:, 11] = size, -size
    ids = torch.tensor([7, 11, 0, 3, 11], dtype=torch.int32, device="cuda")
    logp, ent, ti, tl = cbx.token_log_probs(x, ids, top_n=4, scale=scale)
    ref = torch.log_softmax(x.double() * scale, -1)
    err = U32 * (12 * size * scale + 16 + vocab)
    assert bool(((logp.double() - ref.gather(1, ids.long()[:, None])[:, 0]).abs() <= err).all())
    # each p's relative error on log T and on p z
    h = torch.special.entr(ref.exp()).sum(-1)
    assert bool(((ent.double() - h).abs() <= 4 * err * (1 + h)).all())
    order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :4]
    assert torch.equal(ti.long(), order)
    assert bool(((tl.double() - ref.gather(1, order)).abs() <= err).all())


def test_scales_past_the_range_are_refused(cbx):
    x = torch.zeros(2, 50, device="cuda")
    for scale in (2.0 ** 126, 3e38):
        with pytest.raises(cbx.CbxError, match="scale"):
            cbx.token_log_probs(x, top_n=2, scale=scale)


def test_outputs_are_saved_together(cbx):
    """Numbers and tokens kept in one file, read back."""
    x = torch.randn(6, 300, device="cuda", generator=gen(51))
    ids = torch.arange(6, dtype=torch.int32, device="cuda")
    for kw in (dict(ids=ids, top_n=3), dict(top_n=3, entropy=False), dict(ids=ids)):
        got = [t for t in cbx.token_log_probs(x, **kw) if t is not None]
        f = io.BytesIO()
        torch.save(got, f)
        f.seek(0)
        back = torch.load(f, weights_only=True)
        assert all(torch.equal(a, b) for a, b in zip(got, back))
