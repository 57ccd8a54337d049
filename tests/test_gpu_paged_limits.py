"""What the paged operators refuse on the host once the device is known, and
the rows that their other tests' bounds say little about."""
import pytest
import torch

from tests._paged import gen

pytestmark = pytest.mark.gpu


def test_attention_scratch_overlaps_a_tensor(cbx):
    d, page, width = 64, 64, 40
    kc = torch.zeros(width, 1, page, d, dtype=torch.float16, device="cuda")
    vc, tables = torch.zeros_like(kc), torch.arange(width, dtype=torch.int32, device="cuda")[None]
    lens, q = torch.tensor([width * page], dtype=torch.int32, device="cuda"), torch.zeros(1, 1, d, device="cuda")
    need = cbx.paged_attention_workspace(q, kc, tables)
    assert need > 0
    arena = torch.zeros(need // 4 + 64 + d, device="cuda")
    y = arena[need // 4 - 16:need // 4 - 16 + d].view(1, 1, d)
    with pytest.raises(cbx.CbxError, match="ws must not overlap"):
        cbx.paged_attention(q, kc, vc, tables, lens, 0.125, out=y, ws=arena)
    with pytest.raises(cbx.CbxError, match="ws must not overlap"):
        cbx.paged_attention(q, kc, vc, tables, lens, 0.125, ws=kc.view(-1))
    y = arena[-d:].view(1, 1, d)                   # an arena that holds more than the scratch
    assert torch.equal(cbx.paged_attention(q, kc, vc, tables, lens, 0.125, out=y, ws=arena), torch.zeros_like(y))


def test_log_prob_scratch_overlaps_a_tensor(cbx):
    x = torch.zeros(1, 40000, device="cuda")
    assert 0 < cbx.token_log_probs_workspace(x, 4) < x.numel() * 4
    with pytest.raises(cbx.CbxError, match="ws must not overlap"):
        cbx.token_log_probs(x, top_n=4, ws=x.view(-1))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("v", [70, 8194, 40000])
def test_lowest_logits_mask_as_infinite_ones(cbx, dt, v):
    """Logits of the type's lowest value beside usual ones have p = 0 in f32 as
    those of -inf do: the other tokens' results are the same bits."""
    g = gen(31)
    x = (torch.randn(9, v, device="cuda", generator=g) * 3).to(dt)
    mask = torch.rand(9, v, device="cuda", generator=g) < 0.5
    mask[:, 5] = False
    ids = torch.full((9,), 5, dtype=torch.int32, device="cuda")
    low = cbx.token_log_probs(x.masked_fill(mask, torch.finfo(dt).min), ids, top_n=8, scale=0.7)
    inf = cbx.token_log_probs(x.masked_fill(mask, float("-inf")), ids, top_n=8, scale=0.7)
    for a, b in zip(low, inf):
        assert torch.equal(a, b) and bool(torch.isfinite(a.float()).all())
