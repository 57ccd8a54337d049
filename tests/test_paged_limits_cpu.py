"""Sizes past a launch's threads are refused by the host: descriptors of
tensors that are not there, no device."""
import ctypes

import pytest
import torch

from chatterbox_amdvulkan_amd import cbxops as C

BIG, ERR = 1 << 24, C.ERR_UNSUPPORTED


def desc(type_, *ne):
    """Contiguous, at an address that nothing reads."""
    t = C.Tensor()
    t.data, t.type = ctypes.c_void_p(1 << 40 | desc.at << 44), type_
    desc.at += 1
    nb = 2 if type_ == C.F16 else 4
    for i in range(4):
        t.ne[i] = ne[i] if i < len(ne) else 1
        t.nb[i] = nb
        nb *= t.ne[i]
    return ctypes.byref(t)


desc.at = 0


def check(rc):
    assert rc == ERR and ("2^24" in C.last_error() or "too large" in C.last_error()), (rc, C.last_error())


def test_too_many_workgroups():
    L, f, i = C.load(), C.F16, C.I32
    cache = (f, 64, 16, 2, 8)
    check(L.cbx_paged_store(desc(f, 64, 2, BIG), desc(f, 64, 2, BIG), desc(i, BIG), desc(*cache), desc(*cache), None))
    check(L.cbx_paged_attention(desc(f, 64, 4, BIG // 4), desc(*cache), desc(*cache), desc(i, 2, BIG // 4), desc(i, BIG // 4), 0.125,
                                0.0, 0, desc(f, 64, 4, BIG // 4), None, 0, None))
    check(L.cbx_token_log_probs(desc(f, 8, BIG), None, 1.0, None, desc(C.F32, BIG), None, None, None, 0, None))


def test_append_outputs_are_all_given_or_none():
    z = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    with pytest.raises(C.CbxError, match="all five"):
        C.paged_append(z(3), z(3), z(8), z(1), torch.zeros(3, 5, dtype=torch.int32), 16, 4, out=(None, z(1), z(4), z(4), z(4)))
