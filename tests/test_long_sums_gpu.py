"""GPU tests of the longest sequences against bounds under which a tile of V that is left out, or taken twice, shows."""
import pytest
import torch

import test_quant_cache_gpu as quant
import test_shared_prefix_gpu as shared
import weight_bounds

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def api():
    import decoding_attention_b200
    return decoding_attention_b200


def check(o, lse, q, k, v, bits, alibi=False, what=""):
    ones = torch.ones(k.shape[:2], device=k.device)
    found = weight_bounds.attend(q, k, ones, v, ones, alibi=alibi)
    tol, tol_lse = weight_bounds.random_bounds(found, len(k), bits, o.dtype)
    assert ((lse.double() - found["lse"]).abs() <= tol_lse).all(), f"{what} lse: off by {(lse.double() - found['lse']).abs().max()}"
    over = (o.double() - found["o"]).abs() / tol
    assert (over <= 1.0).all(), f"{what}: {over.max().item():.3g} of the bound"


@pytest.mark.parametrize("hq,hk,dim", [(16, 4, 128), (8, 8, 96), (32, 2, 128), (8, 2, 64), (8, 8, 256)])
@pytest.mark.parametrize("kind", ["fp8", "int8", "int4"])
def test_decode_over_codes(api, kind, hq, hk, dim):
    for dt, lens, page, alibi in (("fp16", [40001], 64, False), ("bf16", [20000, 300, 7000], 0, False), ("fp16", [9000, 12345], 16, True),
                                  ("fp16", [1300 + 7 * i for i in range(160)], 0, False)):
        pr = quant.problem(kind, DTYPES[dt], lens, hq, hk, dim, 50, page=page)
        o, lse = api.quantized_fwd(pr["q"], pr["kc"], pr["vc"], pr["ks"], pr["vs"], pr["cu"], is_alibi=alibi, return_lse=True,
                                   block_table=pr["table"])
        for b in range(0, len(lens), 1 + len(lens) // 5):
            check(o[b], lse[b], pr["q"][b], pr["k"][b], pr["v"][b], 11, alibi, f"{kind} {hq}/{hk} {dim} {lens[:3]} sequence {b}")


@pytest.mark.parametrize("hq,hk,dim,batch", [(16, 4, 128, 200), (32, 1, 64, 60), (12, 4, 96, 7), (32, 8, 128, 1)])
@pytest.mark.parametrize("kind", [None, "fp8", "int4"])
@pytest.mark.parametrize("dt,bits", [("fp16", 11), ("bf16", 8)])
def test_decode_behind_a_prefix(api, dt, bits, kind, hq, hk, dim, batch):
    for prefix, top, page in ((9000, 300, 0), (4096, 3000, 64)):
        lens = [(i * 129) % (top + 1) for i in range(1, batch + 1)]
        pr = shared.problem(DTYPES[dt], prefix, lens, hq, hk, dim, 51, kind=kind, page=page, prefix_page=page)
        o, lse = shared.call(api, pr)
        for b in range(0, batch, 1 + batch // 5):
            check(o[b], lse[b], pr["q"][b], pr["keys"][0][b], pr["keys"][1][b], bits, False, f"{dt} {kind} {prefix}+{lens[b]} sequence {b}")
