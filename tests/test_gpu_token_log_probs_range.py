"""token_log_probs' outputs as tensors that a program keeps."""
import io

import pytest
import torch

from tests._paged import gen

pytestmark = pytest.mark.gpu


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
