"""GPU tests of decode behind a shared prefix where one key leads many: the small weights of the others are kept."""
import pytest
import torch

import weight_bounds

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def api():
    import decoding_attention_b200
    return decoding_attention_b200


def lead_and_check(api, dtype, bits, dim, hq, hk, batch, prefix, own, leads, nats):
    """`leads`: (part, key) of the leading keys, one call each.  Checked for the last sequence, some of its heads."""
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(1, 1, dim, device=DEV, generator=g).to(dtype).expand(batch, hq, -1).contiguous()
    cu = (torch.arange(batch + 1, device=DEV) * own).to(torch.int32)
    k = [(0.05 * torch.randn(n, hk, dim, device=DEV, generator=g)).to(dtype) for n in (prefix, own * batch)]
    v = [(0.5 + torch.randn(n, hk, dim, device=DEV, generator=g)).to(dtype) for n in (prefix, own * batch)]
    row = q[0, 0].float()
    lead = (row * (nats * dim ** 0.5 / (row @ row))).to(dtype)
    b, group = batch - 1, hq // hk
    for side, j in leads:
        at = j + (own * b if side else 0)
        k[side][at], v[side][at, :, ::2] = lead, 0.0
        o, lse = api.shared_prefix_fwd(q, k[0], v[0], k[1], v[1], cu, return_lse=True)
        mine = [torch.cat((x[0], x[1][own * b:])) for x in (k, v)]
        ones = torch.ones(prefix + own, hk, device=DEV)
        found = weight_bounds.attend(q[b], mine[0], ones, mine[1], ones)
        tol, tol_lse = weight_bounds.bounds(found, prefix + own, bits, dtype)
        assert ((lse[b].double() - found["lse"]).abs() <= tol_lse).all(), (lse[b].double() - found["lse"]).abs().max()
        over = (o[b].double() - found["o"]).abs() / tol
        assert (over <= 1.0).all(), f"key {j} of part {side}: {over.max().item():.3g} of the bound"
        k[side][at] = 0.0


TYPES = [(torch.float16, 11), (torch.bfloat16, 8)]


@pytest.mark.parametrize("dim,hq,hk,batch", [(128, 32, 8, 40), (64, 16, 16, 9), (96, 12, 1, 3)])
@pytest.mark.parametrize("dtype,bits", TYPES)
def test_one_key_far_ahead(api, dtype, bits, dim, hq, hk, batch):
    """The leading key's V row is zero in half of the dims, where the output is what the many small weights come to."""
    lead_and_check(api, dtype, bits, dim, hq, hk, batch, 8000, 50, [(0, 1), (0, 700), (0, 7999)], 16.0)
    lead_and_check(api, dtype, bits, dim, hq, hk, batch, 200, 3000, [(1, 1), (1, 700), (1, 2999)], 16.0)


@pytest.mark.parametrize("dtype,bits", TYPES)
def test_one_key_far_ahead_in_a_block_with_many(api, dtype, bits):
    """Enough rows that a block has most of the prefix, or all keys of a sequence, in one sum."""
    for dim in (64, 128):
        lead_and_check(api, dtype, bits, dim, 64, 8, 512, 4000, 1, [(0, 0), (0, 2500)], 16.3)
        lead_and_check(api, dtype, bits, dim, 8, 8, 300, 100, 3000, [(1, 0), (1, 1777)], 16.3)


@pytest.mark.parametrize("prefix,own", [(0, 40), (150, 0), (150, 40)])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_scores_near_the_end_of_fp32(api, sign, prefix, own):
    """Keys that are all alike, with scores of +-2^122: the output is the mean of V."""
    dim, hq, hk = 128, 8, 2
    g = torch.Generator(device=DEV).manual_seed(4)
    k = [torch.full((n, hk, dim), 2.0 ** 62, device=DEV, dtype=torch.bfloat16) for n in (prefix, own)]
    v = [torch.randn(n, hk, dim, device=DEV, generator=g).to(torch.bfloat16) for n in (prefix, own)]
    q = torch.full((1, hq, dim), sign * 2.0 ** 60 / dim, device=DEV, dtype=torch.bfloat16)
    cu = torch.tensor([0, own], dtype=torch.int32, device=DEV)
    o, lse = api.shared_prefix_fwd(q, k[0], v[0], k[1], v[1], cu, softmax_scale=1.0, return_lse=True)
    ones = torch.ones(prefix + own, hk, device=DEV)
    found = weight_bounds.attend(q[0], torch.cat(k), ones, torch.cat(v), ones, softmax_scale=1.0)
    tol, tol_lse = weight_bounds.bounds(found, prefix + own, 8, q.dtype)
    assert ((lse[0].double() - found["lse"]).abs() <= tol_lse).all() and ((o[0].double() - found["o"]).abs() <= tol).all()
