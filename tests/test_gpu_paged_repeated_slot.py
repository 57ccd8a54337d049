"""A slot given to several tokens of a call: its rows hold elements of them,
each from one token, and no other row of the cache changes."""
import pytest
import torch

from tests._paged import gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,cdt", [(torch.float32, torch.float16), (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("d", [64, 129])
def test_elements_of_the_tokens(cbx, dt, cdt, d):
    tok, hkv, page, pages = 200, 2, 16, 6
    r = gen(60 + d)
    k, v = (torch.randn(tok, hkv, d, device="cuda", generator=r).to(dt) for _ in range(2))
    kc, vc = (torch.randn(pages, hkv, page, d, device="cuda", generator=r).to(cdt) for _ in range(2))
    slots = torch.arange(tok, device="cuda", dtype=torch.int32) % 3 * 17      # slots 0, 17 and 34
    before = kc.clone(), vc.clone()
    cbx.paged_store(k, v, slots, kc, vc)
    forms = [(kc, vc, k, v)]
    if d % 8 == 0:
        rope = cbx.RopeCache(d, n_pos=8)
        pos = torch.zeros(tok, dtype=torch.int32, device="cuda")
        _, yk = cbx.qk_norm_rope(k.float(), k.float(), None, None, 1e-6, pos, rope)
        k2, v2 = before[0].clone(), before[1].clone()
        cbx.qk_norm_rope_store(k, k, v, None, None, 1e-6, pos, rope, slots, k2, v2)
        forms.append((k2, v2, yk, v))
        rope.close()
    for cache_k, cache_v, rows_k, rows_v in forms:
        for cache, rows, old in ((cache_k, rows_k, before[0]), (cache_v, rows_v, before[1])):
            cut = cache.transpose(1, 2).reshape(-1, hkv, d)
            for i in range(3):
                assert bool((rows[i::3].to(cdt) == cut[17 * i]).any(0).all()), f"slot {17 * i}"
            rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
            rest[[0, 17, 34]] = False
            assert torch.equal(cut[rest], old.transpose(1, 2).reshape(-1, hkv, d)[rest])
    assert cbx.device_errors(clear=True) == 0
