"""Refusals of the prompt, shared and 8-bit entry points, without a GPU."""
import ctypes

import pytest
import torch

from chatterbox_amdvulkan_amd import cbxops as C

N, HQ, HKV, D, PAGE, PAGES, WIDTH = 3, 4, 2, 64, 16, 8, 5


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def ref(t):
    return ctypes.byref(C.desc(t, C.I8 if t.dtype == torch.int8 else None)) if t is not None else None


def refused(rc, text, code=None):
    assert rc in ((C.ERR_INVALID_ARG, C.ERR_UNSUPPORTED) if code is None else (code,)), (rc, C.last_error())
    assert text in C.last_error(), C.last_error()


def cache(dtype=torch.float16, d=D, hkv=HKV):
    return torch.zeros(PAGES, hkv, PAGE, d, dtype=dtype)


def scales(hkv=HKV, page=PAGE):
    return torch.zeros(PAGES, hkv, page)


def store(**kw):
    a = dict(k=torch.zeros(N, HKV, D), v=torch.zeros(N, HKV, D), slots=i32(N), kc=cache(torch.int8), ks=scales(),
             vc=cache(torch.int8), vs=scales())
    a.update(kw)
    return C.load().cbx_paged_store_q8(ref(a["k"]), ref(a["v"]), ref(a["slots"]), ref(a["kc"]), ref(a["ks"]), ref(a["vc"]),
                                       ref(a["vs"]), None)


def test_store_q8_refusals():
    refused(store(ks=None), "NULL")
    refused(store(kc=cache()), "must be I8", C.ERR_UNSUPPORTED)
    refused(store(vc=cache(torch.float32)), "must be I8", C.ERR_UNSUPPORTED)
    refused(store(ks=scales(hkv=HKV + 1)), "k_scale must be F32")
    refused(store(vs=scales(page=PAGE - 1)), "v_scale must be F32")
    refused(store(vs=scales().half()), "v_scale must be F32")
    refused(store(slots=i32(N + 1)), "slots")
    refused(store(k=torch.zeros(N, HKV, D, dtype=torch.float16)), "types differ")
    one = scales()
    refused(store(ks=one, vs=one), "k_scale must not overlap v_scale")
    both = torch.zeros(PAGES, HKV, PAGE, D + 4, dtype=torch.int8)
    refused(store(kc=both[..., :D], ks=both.view(torch.float32)[..., D // 4]), "overlap")   # taken as one: types of two sizes
    refused(store(ks=torch.zeros(1).expand(PAGES, HKV, PAGE)), "stride of 0")
    buf = torch.zeros(PAGES * HKV * PAGE * D, dtype=torch.int8)
    refused(store(kc=buf.view(PAGES, HKV, PAGE, D), vs=buf.view(torch.float32)[:PAGES * HKV * PAGE].view(PAGES, HKV, PAGE)),
            "must not overlap")


def test_i8_is_a_cache_type_only():
    x = torch.zeros(4, 64, dtype=torch.int8)
    refused(C.load().cbx_paged_store(ref(torch.zeros(N, HKV, D)), ref(torch.zeros(N, HKV, D)), ref(i32(N)), ref(cache(torch.int8)),
                                     ref(cache(torch.int8)), None), "unknown type")
    with pytest.raises(C.CbxError):
        C.desc(x)


def load(**kw):
    a = dict(slots=i32(N), kc=cache(torch.int8), ks=scales(), vc=cache(torch.int8), vs=scales(), k=torch.zeros(N, HKV, D),
             v=torch.zeros(N, HKV, D))
    a.update(kw)
    return C.load().cbx_paged_load(ref(a["slots"]), ref(a["kc"]), ref(a["ks"]), ref(a["vc"]), ref(a["vs"]), ref(a["k"]),
                                   ref(a["v"]), None)


def test_load_refusals():
    refused(load(ks=None), "go together")
    refused(load(ks=None, vs=None), "unknown type")
    refused(load(kc=cache(), vc=cache()), "must be I8", C.ERR_UNSUPPORTED)
    refused(load(v=torch.zeros(N, HKV, D // 2)), "k and v")
    refused(load(k=torch.zeros(N, HKV, D, dtype=torch.float16)), "types differ")
    refused(load(slots=i32(N - 1)), "slots")
    x = torch.zeros(N, HKV, D)
    refused(load(k=x, v=x), "k must not overlap v")
    refused(load(kc=cache(d=32), vc=cache(d=32), ks=None, vs=None), "cache must be")
    refused(load(k=torch.zeros(1, HKV, D).expand(N, HKV, D)), "stride of 0")


def qk(**kw):
    a = dict(q=torch.zeros(N, HQ, D), k=torch.zeros(N, HKV, D), v=torch.zeros(N, HKV, D), pos=i32(N), slots=i32(N),
             yq=torch.zeros(N, HQ, D), kc=cache(torch.int8), ks=scales(), vc=cache(torch.int8), vs=scales())
    a.update(kw)
    return C.load().cbx_qk_norm_rope_store_q8(ref(a["q"]), None, ref(a["k"]), None, ref(a["v"]), 1e-6, ref(a["pos"]),
                                              a.get("rope"), ref(a["slots"]), ref(a["yq"]), ref(a["kc"]), ref(a["ks"]),
                                              ref(a["vc"]), ref(a["vs"]), None)


def test_qk_store_q8_refusals():
    refused(qk(), "rope is NULL")
    refused(qk(vs=None), "NULL")
    some = ctypes.c_void_p(1)                               # nothing looks at it before the refusal
    refused(qk(rope=some, kc=cache()), "must be I8", C.ERR_UNSUPPORTED)
    refused(qk(rope=some, ks=scales(page=4)), "k_scale must be F32")
    y = torch.zeros(N * HQ * D)
    refused(qk(rope=some, yq=y.view(N, HQ, D), ks=y[:PAGES * HKV * PAGE].view(PAGES, HKV, PAGE)), "yq must not overlap k_scale")


T = 7


def prompt(**kw):
    a = dict(q=torch.zeros(T, HQ, D), kc=cache(), ks=None, vc=cache(), vs=None, tables=i32(N, WIDTH), lens=i32(N),
             start=i32(N + 1), scale=0.125, cap=0.0, window=0, y=torch.zeros(T, HQ, D))
    a.update(kw)
    return C.load().cbx_paged_prompt_attention(ref(a["q"]), ref(a["kc"]), ref(a["ks"]), ref(a["vc"]), ref(a["vs"]),
                                               ref(a["tables"]), ref(a["lens"]), ref(a["start"]), a["scale"], a["cap"],
                                               a["window"], ref(a["y"]), None, 0, None)


def shared(**kw):
    a = dict(q=torch.zeros(N, HQ, D), kc=cache(), ks=None, vc=cache(), vs=None, tables=i32(N, WIDTH), lens=i32(N),
             start=i32(3), pre=i32(2), scale=0.125, cap=0.0, window=0, y=torch.zeros(N, HQ, D))
    a.update(kw)
    return C.load().cbx_paged_shared_attention(ref(a["q"]), ref(a["kc"]), ref(a["ks"]), ref(a["vc"]), ref(a["vs"]),
                                               ref(a["tables"]), ref(a["lens"]), ref(a["start"]), ref(a["pre"]), a["scale"],
                                               a["cap"], a["window"], ref(a["y"]), None, 0, None)


@pytest.mark.parametrize("call", [prompt, shared])
def test_attention_refusals(call):
    q = call.__name__ == "prompt" and T or N
    refused(call(kc=cache(torch.float32)), "types differ", C.ERR_UNSUPPORTED)
    refused(call(kc=cache(d=32), vc=cache(d=32)), "head_dim")
    refused(call(q=torch.zeros(q, 3, D), y=torch.zeros(q, 3, D)), "multiple of n_head_kv")
    refused(call(y=torch.zeros(q, HQ, D, dtype=torch.float16)), "types differ", C.ERR_UNSUPPORTED)
    refused(call(y=torch.zeros(q, HQ, D + 8)), "shapes differ")
    refused(call(scale=float("inf")), "scale")
    refused(call(cap=-1.0), "softcap")
    refused(call(window=-1), "window")
    refused(call(lens=i32(N + 1)), "seq_lens")
    refused(call(start=torch.zeros(N + 1)), "start")
    refused(call(tables=None), "NULL")
    refused(call(kc=None), "NULL")
    refused(call(ks=scales()), "go together")
    refused(call(ks=scales(), vs=scales()), "must be I8", C.ERR_UNSUPPORTED)
    refused(call(kc=cache(torch.int8), vc=cache(torch.int8)), "unknown type")
    refused(call(kc=cache(torch.int8), vc=cache(torch.int8), ks=scales(), vs=scales(hkv=1)), "v_scale must be F32")
    x = torch.zeros(q, HQ, D)
    refused(call(q=x, y=x), "y must not overlap an input")
    refused(call(y=torch.zeros(1, HQ, D).expand(q, HQ, D)), "stride of 0")


def test_prompt_refusals():
    refused(prompt(start=i32(N)), "tok_start")
    refused(prompt(tables=i32(N + 1, WIDTH)), "seq_lens")
    big = torch.zeros(1, 1, D).expand(1 << 22, HQ, D)
    refused(prompt(q=big, y=big), "2^24", C.ERR_UNSUPPORTED)
    n = ctypes.c_size_t(7)
    refused(C.load().cbx_paged_prompt_attention_workspace(ref(torch.zeros(T, HQ, 32)), ref(cache()), ref(i32(N, WIDTH)),
                                                          ctypes.byref(n)), "head_dim")
    assert n.value == 0
    refused(C.load().cbx_paged_prompt_attention_workspace(ref(torch.zeros(T, HQ, D)), ref(cache()), ref(i32(N, WIDTH)), None), "NULL")


def test_shared_refusals():
    refused(shared(start=i32(0)), "group_start")
    refused(shared(pre=i32(3)), "shared_lens")
    refused(shared(start=None), "NULL")
    refused(shared(tables=i32(N + 1, WIDTH)), "block_tables")
    refused(C.load().cbx_paged_shared_attention_workspace(ref(torch.zeros(N, HQ, D)), ref(cache()), ref(i32(N, WIDTH)), ref(i32(2)),
                                                          None), "NULL")


def test_attention_q8_refusals():
    def attend(ks, vs, kc=cache(torch.int8), vc=cache(torch.int8)):
        q = torch.zeros(N, HQ, D)
        return C.load().cbx_paged_attention_q8(ref(q), ref(kc), ref(ks), ref(vc), ref(vs), ref(i32(N, WIDTH)), ref(i32(N)), 0.125,
                                               0.0, 0, ref(torch.zeros(N, HQ, D)), None, 0, None)

    refused(attend(None, None), "NULL")
    refused(attend(scales(), None), "NULL")
    refused(attend(scales(), scales(), kc=cache(), vc=cache()), "must be I8", C.ERR_UNSUPPORTED)
    refused(attend(scales(page=3), scales()), "k_scale must be F32")
