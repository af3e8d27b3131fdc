"""CPU tests of the bounds in weight_bounds: they reject an output that lacks one tile of V, at any length in use."""
import pytest
import torch

import quant_reference as ref
import weight_bounds


@pytest.mark.parametrize("kind,n,bits,dtype", [("int8", 20000, 11, torch.bfloat16), ("fp8", 40001, 11, torch.float16),
                                               ("int4", 1300, 11, torch.bfloat16), ("int8", 40001, 11, torch.bfloat16),
                                               ("int8", 9300, 8, torch.bfloat16)])
def test_a_missing_tile_is_rejected(kind, n, bits, dtype):
    g = torch.Generator().manual_seed(1)
    q = torch.randn(4, 64, generator=g).to(dtype)
    k, ks = ref.quantise(torch.randn(n, 2, 64, generator=g), kind)
    v, vs = ref.quantise(torch.randn(n, 2, 64, generator=g) * torch.exp(0.5 * torch.randn(n, 2, 1, generator=g)), kind)
    found = weight_bounds.attend(q, k, ks, v, vs)
    tol, tol_lse = weight_bounds.random_bounds(found, n, bits, dtype)
    assert (tol <= weight_bounds.bounds(found, n, bits, dtype)[0]).double().mean() > 0.9
    assert ((found["o"].to(dtype).double() - found["o"]).abs() <= tol).all()
    at = n // 2 // 128 * 128
    for change in (0.0, -1.0):
        less = v.clone()
        less[at:at + 128] *= change
        off = (weight_bounds.attend(q, k, ks, less, vs)["o"] - found["o"]).abs()
        assert (off > tol).double().mean() > 0.3, (off / tol).median()
    assert (found["o"].abs() > tol).double().mean() > 0.8  # an output of zeros
    assert (tol_lse < 1e-2).all()
