"""Numbers that the paged operators' entry points refuse, without a GPU."""
import ctypes

import pytest
import torch

from chatterbox_amdvulkan_amd import cbxops as C


def ref(t):
    return ctypes.byref(C.desc(t))


@pytest.mark.parametrize("scale", [2.0 ** 126, 3e38])
def test_log_prob_scales(scale):
    x, ent = torch.zeros(3, 50), torch.zeros(3)
    rc = C.load().cbx_token_log_probs(ref(x), None, scale, None, ref(ent), None, None, None, 0, None)
    assert rc == C.ERR_UNSUPPORTED and "scale" in C.last_error(), (rc, C.last_error())
