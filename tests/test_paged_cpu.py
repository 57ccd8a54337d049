"""The paged-cache entry points' argument checks, without a GPU: every refusal
is an error code and a message from the host, before anything is launched."""
import ctypes

import pytest
import torch

from chatterbox_amdvulkan_amd import cbxops as C

N, HQ, HKV, D, PAGE, PAGES, WIDTH = 3, 4, 2, 64, 16, 8, 5


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def ref(t):
    return ctypes.byref(C.desc(t)) if t is not None else None


def refused(rc, text, code=None):
    assert rc in ((C.ERR_INVALID_ARG, C.ERR_UNSUPPORTED) if code is None else (code,)), (rc, C.last_error())
    assert text in C.last_error(), C.last_error()


def append(**kw):
    a = dict(n_past=i32(N), n_new=i32(N), free=i32(PAGES), n_free=i32(1), tables=i32(N, WIDTH), page=PAGE, lens=i32(N),
             left=i32(1), start=i32(N + 1), slots=i32(7), pos=i32(7))
    a.update(kw)
    return C.load().cbx_paged_append(ref(a["n_past"]), ref(a["n_new"]), ref(a["free"]), ref(a["n_free"]), ref(a["tables"]),
                                     a["page"], ref(a["lens"]), ref(a["left"]), ref(a["start"]), ref(a["slots"]),
                                     ref(a["pos"]), None)


def test_append_refusals():
    refused(append(page=0), "page_size")
    refused(append(n_new=i32(N + 1)), "n_new")
    refused(append(n_past=torch.zeros(N)), "n_past")
    refused(append(tables=i32(N + 1, WIDTH)), "block_tables")
    refused(append(start=i32(N)), "tok_start")
    refused(append(pos=i32(8)), "positions")
    refused(append(n_free=i32(2)), "n_free")
    refused(append(page=2 ** 31 - 1), "2^31", C.ERR_UNSUPPORTED)
    refused(append(n_past=None), "NULL")
    many = 4097
    refused(append(n_past=i32(many), n_new=i32(many), tables=i32(many, WIDTH), lens=i32(many), start=i32(many + 1)), "4096",
            C.ERR_UNSUPPORTED)
    x = i32(N)
    refused(append(n_past=x, lens=x), "seq_lens must not overlap an input")
    both = i32(9)
    refused(append(slots=both[:7], pos=both[2:]), "slots must not overlap positions")
    refused(append(tables=i32(1, WIDTH).expand(N, WIDTH)), "stride of 0")


def test_release_refusals():
    def release(**kw):
        a = dict(lens=i32(N), release=i32(N), tables=i32(N, WIDTH), page=PAGE, free=i32(PAGES), n_free=i32(1), lens_out=i32(N),
                 left=i32(1))
        a.update(kw)
        return C.load().cbx_paged_release(ref(a["lens"]), ref(a["release"]), ref(a["tables"]), a["page"], ref(a["free"]),
                                          ref(a["n_free"]), ref(a["lens_out"]), ref(a["left"]), None)

    refused(release(page=-1), "page_size")
    refused(release(release=i32(N - 1)), "release")
    refused(release(left=i32(0)), "n_free_out")
    x = i32(1)
    refused(release(n_free=x, left=x), "n_free_out must not overlap an input")


def cache(dtype=torch.float16, pages=PAGES, d=D, hkv=HKV):
    return torch.zeros(pages, hkv, PAGE, d, dtype=dtype)


def test_store_refusals():
    def store(k=torch.zeros(N, HKV, D), v=torch.zeros(N, HKV, D), slots=i32(N), kc=cache(), vc=cache()):
        return C.load().cbx_paged_store(ref(k), ref(v), ref(slots), ref(kc), ref(vc), None)

    refused(store(k=torch.zeros(N, HKV, D, dtype=torch.float16)), "types differ")
    refused(store(v=torch.zeros(N, HKV, D // 2)), "k and v")
    refused(store(kc=cache(torch.float32)), "types differ")
    refused(store(kc=cache(d=32), vc=cache(d=32)), "head_dim")
    refused(store(slots=i32(N + 1)), "slots")
    c = cache()
    refused(store(kc=c, vc=c), "k_cache must not overlap v_cache")
    refused(store(kc=cache(pages=1).expand(PAGES, HKV, PAGE, D)), "stride of 0")


def test_interleaved_caches_are_apart():
    """K and V of one allocation share a byte range but no element: taken up
    to the missing device, and refused once they do share one."""
    if torch.cuda.is_available():
        pytest.skip("would launch over host memory")
    both = torch.zeros(PAGES, 2, HKV, PAGE, D, dtype=torch.float16)
    inner = torch.zeros(PAGES, PAGE, 2, HKV, D, dtype=torch.float16).permute(2, 0, 3, 1, 4)
    L, k, v, slots = C.load(), torch.zeros(N, HKV, D), torch.zeros(N, HKV, D), i32(N)
    for kc, vc in ((both[:, 0], both[:, 1]), (inner[0], inner[1])):
        assert L.cbx_paged_store(ref(k), ref(v), ref(slots), ref(kc), ref(vc), None) in (C.ERR_HIP, C.ERR_NOT_INITIALIZED)
        assert "overlap" not in C.last_error()
    flat = torch.zeros(2 * PAGES * HKV * PAGE * D, dtype=torch.float16)
    n = PAGES * HKV * PAGE * D
    kc, vc = flat[:n].view(PAGES, HKV, PAGE, D), flat[n - 1:2 * n - 1].view(PAGES, HKV, PAGE, D)
    refused(L.cbx_paged_store(ref(k), ref(v), ref(slots), ref(kc), ref(vc), None), "overlap")


def qk(q=torch.zeros(N, HQ, D), gq=torch.zeros(D), k=torch.zeros(N, HKV, D), gk=None, eps=1e-6, pos=i32(N), yq=None, yk=None):
    yq = torch.zeros_like(q) if yq is None else yq
    yk = torch.zeros_like(k) if yk is None else yk
    return C.load().cbx_qk_norm_rope(ref(q), ref(gq), ref(k), ref(gk), eps, ref(pos), None, ref(yq), ref(yk), None)


def test_qk_refusals():
    refused(qk(), "rope is NULL")
    refused(qk(k=torch.zeros(N, HKV, D, dtype=torch.float16)), "types differ")
    refused(qk(k=torch.zeros(N + 1, HKV, D)), "n_tok")
    refused(qk(q=torch.zeros(N, HQ, 60), k=torch.zeros(N, HKV, 60), gq=None), "multiple of 8")
    refused(qk(eps=-1.0), "eps")
    refused(qk(eps=float("nan")), "eps")
    refused(qk(gq=torch.zeros(D + 1)), "gq")
    refused(qk(pos=i32(N + 1)), "pos")
    refused(qk(yq=torch.zeros(N, HQ, D, dtype=torch.float16)), "types differ")


def attention(**kw):
    a = dict(q=torch.zeros(N, HQ, D), kc=cache(), vc=cache(), tables=i32(N, WIDTH), lens=i32(N), scale=0.125, cap=0.0, window=0,
             y=torch.zeros(N, HQ, D), ws=None, size=0)
    a.update(kw)
    return C.load().cbx_paged_attention(ref(a["q"]), ref(a["kc"]), ref(a["vc"]), ref(a["tables"]), ref(a["lens"]), a["scale"],
                                        a["cap"], a["window"], ref(a["y"]), a["ws"], a["size"], None)


def test_attention_refusals():
    refused(attention(q=torch.zeros(N, 3, D), y=torch.zeros(N, 3, D)), "n_head_kv")
    refused(attention(q=torch.zeros(N, HQ, 32), y=torch.zeros(N, HQ, 32)), "head_dim")
    refused(attention(y=torch.zeros(N, HQ, D, dtype=torch.float16)), "types differ")
    refused(attention(kc=cache(torch.float32)), "types differ")
    refused(attention(lens=i32(N + 1)), "seq_lens")
    refused(attention(tables=i32(N - 1, WIDTH)), "block_tables")
    refused(attention(tables=torch.zeros(N, WIDTH)), "block_tables")
    for bad in (float("nan"), float("inf")):
        refused(attention(scale=bad), "scale")
        refused(attention(cap=bad), "softcap")
    refused(attention(cap=-1.0), "softcap")
    refused(attention(window=-1), "window")
    q = torch.zeros(N, HQ, D)
    refused(attention(q=q, y=q), "y must not overlap")
    refused(attention(q=torch.zeros(N, HQ, 520), y=torch.zeros(N, HQ, 520), kc=cache(d=520), vc=cache(d=520)), "512")
    n = ctypes.c_size_t(7)
    refused(C.load().cbx_paged_attention_workspace(ref(torch.zeros(N, 3, D)), ref(cache()), ref(i32(N, WIDTH)), ctypes.byref(n)),
            "n_head_kv")
    assert n.value == 0


def logp(x=torch.zeros(N, 50), ids=i32(N), scale=1.0, lp=torch.zeros(N), ent=torch.zeros(N), ti=i32(N, 4), tl=torch.zeros(N, 4)):
    return C.load().cbx_token_log_probs(ref(x), ref(ids), scale, ref(lp), ref(ent), ref(ti), ref(tl), None, 0, None)


def test_log_prob_refusals():
    refused(logp(ids=None), "go together")
    refused(logp(tl=None), "go together")
    refused(logp(ids=None, lp=None, ent=None, ti=None, tl=None), "no output")
    refused(logp(scale=0.0), "scale")
    refused(logp(scale=float("nan")), "scale")
    refused(logp(ti=i32(N, 65), tl=torch.zeros(N, 65), x=torch.zeros(N, 100)), "64", C.ERR_UNSUPPORTED)
    refused(logp(x=torch.zeros(N, 3)), "n_vocab")
    refused(logp(tl=torch.zeros(N, 5)), "top_logp")
    refused(logp(ent=torch.zeros(N + 1)), "entropy")
    refused(logp(ids=i32(N + 1)), "ids")
    refused(logp(x=torch.zeros(N, 50, dtype=torch.int32)), "F32 or F16")
    x = torch.zeros(N, 50)
    refused(logp(x=x, ent=x[0, :N]), "entropy must not overlap")


def test_python_front_end_refuses_host_tensors():
    with pytest.raises(C.CbxError, match="ROCm device"):
        C.paged_attention(torch.zeros(N, HQ, D), cache(), cache(), i32(N, WIDTH), i32(N), 0.125)
    with pytest.raises(C.CbxError, match="ROCm device"):
        C.token_log_probs(torch.zeros(N, 50), i32(N))
    with pytest.raises(C.CbxError, match="ROCm device"):
        C.paged_append(i32(N), i32(N), i32(PAGES), i32(1), i32(N, WIDTH), PAGE, 4)
