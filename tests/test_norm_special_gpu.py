"""NaN and infinity in rows of the norm, in 16 bits and in 8."""
import pytest
import torch

from mini_nangila_b200.ops import norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", [40, 2048, 2051])
@pytest.mark.parametrize("residual", [False, True])
def test_special_rows(dtype, width, residual):
    """The norm of a row with a NaN is NaN everywhere; of a row with an infinity,
    whose root-mean-square is infinite, NaN there and 0 beside it.  codes * scale
    are the same, and quantize_rows keeps a NaN in its place and makes a row with
    an infinity NaN.  Other rows do not notice."""
    x = torch.randn(4, width, device="cuda").to(dtype)
    clean = x.clone()
    x[1, 3], x[2, 5] = float("nan"), -float("inf")
    w = torch.ones(width, device="cuda", dtype=dtype)
    kw = dict(residual=torch.randn(4, width, device="cuda").to(dtype)) if residual else {}
    y, codes, scale = (norm.rms_norm(x, w, **kw), *norm.rms_norm_fp8(x, w, **kw)[:2])
    want, wcodes, wscale = (norm.rms_norm(clean, w, **kw), *norm.rms_norm_fp8(clean, w, **kw)[:2])
    if residual:
        y, want = y[0], want[0]
    for v, c in ((y.float(), want.float()),
                 (codes.float() * scale[:, None], wcodes.float() * wscale[:, None])):
        assert v[1].isnan().all() and v[2, 5].isnan() and not v[2, :5].any() and not v[2, 6:].any()
        assert torch.equal(v[0], c[0]) and torch.equal(v[3], c[3])
    codes, scale = norm.quantize_rows(x)
    wcodes, wscale = norm.quantize_rows(clean)
    v, c = codes.float() * scale[:, None], wcodes.float() * wscale[:, None]
    assert v[1, 3].isnan() and v[1, :3].isfinite().all() and v[1, 4:].isfinite().all() and v[2].isnan().all()
    assert torch.equal(v[0], c[0]) and torch.equal(v[3], c[3])
