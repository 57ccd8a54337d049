"""qk_norm_rope and its storing form: the bits of rms_norm_mul then rope_ext
in f32, rounded once to the stored type."""
import numpy as np
import pytest
import torch

from chatterbox_amdvulkan_amd import workloads as W
from tests._util import assert_bitexact

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ref(oracle, x, g, eps, pos, nd, mode, **kw):
    """x [tok, heads, D] any float type -> f32, by the oracle's two ops."""
    x = x.detach().float().cpu().numpy()
    y = oracle.rms_norm(x, eps) if g is None else oracle.rms_norm_mul(x, g.cpu().numpy(), eps)
    return oracle.rope_ext(y.reshape(x.shape), pos.cpu().numpy(), nd, mode=mode, **kw)


def same(got, exp, what):
    assert_bitexact(got.cpu().numpy(), torch.from_numpy(exp).to(got.dtype).numpy(), what)


CASES = [(64, 64, 2, 16, 16), (64, 64, 0, 6, 2), (64, 32, 2, 3, 1), (128, 128, 2, 8, 2), (96, 48, 0, 5, 5), (80, 80, 2, 4, 1),
         (8, 8, 2, 2, 1), (256, 64, 2, 3, 3), (512, 512, 0, 2, 1), (40, 24, 2, 7, 7)]


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("d,nd,mode,hq,hkv", CASES)
def test_heads(cbx, oracle, dt, d, nd, mode, hq, hkv):
    tok = 13
    rows = dev(W.normal(900 + d + nd, (tok, (hq + 2 * hkv) * d + 8), 0.2, 1.7)).to(dt)
    q, k = rows[:, :hq * d].unflatten(1, (hq, d)), rows[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    gq, gk = dev(W.normal(901, (d,), 1.0, 0.2)), dev(W.normal(902, (d,), 1.0, 0.2))
    pos = dev(W.randint(903, (tok,), 0, 300))
    c = cbx.RopeCache(nd, mode=mode, n_pos=300)
    yq, yk = cbx.qk_norm_rope(q, k, gq, gk, 1e-6, pos, c)
    same(yq, ref(oracle, q, gq, 1e-6, pos, nd, mode), "q")
    same(yk, ref(oracle, k, gk, 1e-6, pos, nd, mode), "k")
    yq, yk = cbx.qk_norm_rope(q, k, None, None, 1e-5, pos, c)
    same(yq, ref(oracle, q, None, 1e-5, pos, nd, mode), "q without weights")
    # in place, over the strided rows themselves
    exp = ref(oracle, q, gq, 1e-6, pos, nd, mode), ref(oracle, k, gk, 1e-6, pos, nd, mode)
    v = rows[:, (hq + hkv) * d:].clone()
    cbx.qk_norm_rope(q, k, gq, gk, 1e-6, pos, c, out_q=q, out_k=k)
    same(q, exp[0], "q in place")
    same(k, exp[1], "k in place")
    assert torch.equal(rows[:, (hq + hkv) * d:], v)
    c.close()


@pytest.mark.parametrize("tok", [1, 2, 63, 64, 65, 1000])
def test_token_counts_and_odd_strides(cbx, oracle, tok):
    """Rows at an odd step (no vector loads), outputs of their own stride."""
    d, hq, hkv = 64, 3, 1
    rows = dev(W.normal(910 + tok, (tok, hq * d + hkv * d + 3)))
    q, k = rows[:, 1:1 + hq * d].unflatten(1, (hq, d)), rows[:, 2 + hq * d:2 + (hq + hkv) * d].unflatten(1, (hkv, d))
    pos = dev(W.randint(911, (tok,), 0, 64))
    c = cbx.RopeCache(d, n_pos=64)
    out = torch.zeros(tok, hq, d + 5, device="cuda")[:, :, 1:1 + d]
    g = dev(W.normal(912, (d,), 1.0, 0.1))
    yq, yk = cbx.qk_norm_rope(q, k, g, g, 1e-6, pos, c, out_q=out)
    same(yq, ref(oracle, q, g, 1e-6, pos, d, 2), "q")
    same(yk, ref(oracle, k, g, 1e-6, pos, d, 2), "k")
    c.close()


def test_scaled_rotation_and_far_positions(cbx, oracle):
    """YaRN with frequency factors from the table; positions past it (and
    below 0) from the device's cosf and sinf, 2 f32 ulps of the pair each."""
    d, tok = 128, 24
    kw = dict(n_ctx_orig=4096, freq_base=10000.0, freq_scale=0.25, ext_factor=1.0, attn_factor=1.0, beta_fast=32.0, beta_slow=1.0)
    ff = W.uniform_range(920, (64,), 1.0, 4.0)
    c = cbx.RopeCache(d, n_pos=2000, freq_factors=ff, **kw)
    x = dev(W.normal(921, (tok, 2, d)))
    g = dev(W.normal(922, (d,), 1.0, 0.1))
    pos = torch.arange(tok, dtype=torch.int32, device="cuda") * 83
    yq, _ = cbx.qk_norm_rope(x, x.clone(), g, None, 1e-6, pos, c)
    same(yq, ref(oracle, x, g, 1e-6, pos, d, 2, freq_factors=ff, **kw), "scaled")
    far = pos + 5000
    far[0] = -4
    yq, _ = cbx.qk_norm_rope(x, x.clone(), g, None, 1e-6, far, c)
    exp = ref(oracle, x, g, 1e-6, far, d, 2, freq_factors=ff, **kw)
    pair = np.hypot(exp[..., :64], exp[..., 64:])
    err = np.abs(yq.cpu().numpy() - exp) / np.concatenate([pair, pair], -1)
    # two of cos and sin an ulp or two off each (2 * 2^-23), three roundings
    assert err.max() < 2 * 2.0 ** -22 + 3 * 2.0 ** -24, err.max()
    c.close()


@pytest.mark.parametrize("dt,cdt", [(torch.float16, torch.float16), (torch.float32, torch.float16), (torch.float32, torch.float32),
                                    (torch.float16, torch.float32)])
@pytest.mark.parametrize("d,page,tokens_inner", [(64, 16, False), (96, 5, True), (128, 64, False)])
def test_store(cbx, oracle, dt, cdt, d, page, tokens_inner):
    tok, hq, hkv, pages = 41, 4, 2, 20
    rows = dev(W.normal(930 + d, (tok, (hq + 2 * hkv) * d))).to(dt)
    cut = lambda a, h: rows[:, a * d:(a + h) * d].unflatten(1, (h, d))  # noqa: E731
    q, k, v = cut(0, hq), cut(hq, hkv), cut(hq + hkv, hkv)
    g, pos = dev(W.normal(931, (d,), 1.0, 0.1)), dev(W.randint(932, (tok,), 0, 500))
    both = torch.randn(pages, 2, hkv, page, d, device="cuda").to(cdt)       # K and V of one allocation
    if tokens_inner:
        both = torch.randn(pages, page, 2, hkv, d, device="cuda").to(cdt).permute(0, 2, 3, 1, 4)
    kc, vc = both[:, 0], both[:, 1]
    slots = torch.randperm(pages * page, device="cuda")[:tok].to(torch.int32)
    slots[3] = slots[40] = -1
    ek, ev = kc.clone(), vc.clone()
    c = cbx.RopeCache(d, n_pos=500)
    rk = torch.from_numpy(ref(oracle, k, g, 1e-6, pos, d, 2)).cuda()
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            ek[s // page, :, s % page], ev[s // page, :, s % page] = rk[t].to(cdt), v[t].to(cdt)
    exp = ref(oracle, q, g, 1e-6, pos, d, 2)
    yq = cbx.qk_norm_rope_store(q, k, v, g, g, 1e-6, pos, c, slots, kc, vc)
    same(yq, exp, "q")
    assert torch.equal(kc, ek) and torch.equal(vc, ev)
    assert cbx.device_errors(clear=True) == 0
    slots[7] = pages * page
    cbx.qk_norm_rope_store(q, k, v, g, g, 1e-6, pos, c, slots, kc, vc, out_q=q)   # q in place
    same(q, exp, "q in place")
    assert cbx.device_errors(clear=True) == 4
    c.close()


def test_nothing_to_do_and_refusals(cbx):
    c = cbx.RopeCache(64, n_pos=10)
    e = torch.zeros(0, 2, 64, device="cuda")
    yq, yk = cbx.qk_norm_rope(e, e[:, :1], None, None, 1e-6, torch.zeros(0, dtype=torch.int32, device="cuda"), c)
    assert yq.shape == e.shape
    x, p = torch.zeros(3, 2, 48, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(cbx.CbxError, match="n_dims > head_dim"):
        cbx.qk_norm_rope(x, x.clone(), None, None, 1e-6, p, c)
    odd = cbx.RopeCache(12, n_pos=10)
    with pytest.raises(cbx.CbxError, match="multiple of 8"):
        cbx.qk_norm_rope(x, x.clone(), None, None, 1e-6, p, odd)
    x = torch.zeros(3, 4, 64, device="cuda")
    with pytest.raises(cbx.CbxError, match="overlap"):
        cbx.qk_norm_rope(x[:, :2], x[:, 2:], None, None, 1e-6, p, c, out_q=x[:, 1:3])
    with pytest.raises(cbx.CbxError, match="overlap"):
        cbx.qk_norm_rope(x[:, :2], x[:, 2:], None, None, 1e-6, p, c, out_k=x[:, :2])
    # a row of zeros: 0 * 1/sqrt(eps), 0 whatever the weights
    z = torch.zeros(1, 1, 64, device="cuda")
    yq, _ = cbx.qk_norm_rope(z, z.clone(), None, None, 1e-6, torch.ones(1, dtype=torch.int32, device="cuda"), c)
    assert bool((yq == 0).all())
    c.close()
    odd.close()
