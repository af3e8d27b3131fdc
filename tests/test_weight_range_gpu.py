"""GPU tests of decode attention where softmax weights and V scales differ by many powers of two: a key that takes nearly
all of the weight next to many that share the rest, V rows of zeros, V rows of any size."""
import math

import pytest
import torch

import quant_reference as ref
import weight_bounds

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
KINDS = ["fp8", "int8", "int4"]
# Formats and head layouts: codes as tensor-core operands, codes widened in registers.
CODES = [("fp8", 8, 2, 128), ("int8", 8, 2, 128), ("fp8", 8, 8, 96), ("int8", 8, 8, 96)]
STREAM = [("int4", 8, 2, 128), ("int4", 32, 1, 96), ("int8", 8, 2, 64), ("int8", 32, 2, 128), ("fp8", 4, 1, 256), ("fp8", 16, 1, 64)]
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def api():
    import decoding_attention_b200
    return decoding_attention_b200


def cache_of(n, hk, dim, kind, seed, k_spread=0.1):
    """Codes and scales of a sequence whose scores stay small: K rows of about 0.05, V rows of about one."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = []
    for size in (0.05, 1.0):
        x = size * torch.randn(n, hk, dim, device=DEV, generator=g) + (0.5 if size == 1.0 else 0.0)
        codes, s = ref.quantise(x, kind)
        out += [codes, s]
    return out


def raise_key(q, k_code, k_scale, j, nats):
    """Gives key j a score of about `nats` in all heads (q is the same in all of them)."""
    row = q[0].double()
    top = 112.0 if k_code.abs().max() > 7 else 7.0
    code = torch.round(row / row.abs().max() * top)
    # (numbers that e4m3 has too)
    code = torch.where(code.abs() > 16, torch.round(code / 16) * 16, code) if top == 112.0 else code
    k_code[j] = code
    k_scale[j] = nats * math.sqrt(len(row)) / float(row @ code)


def run(api, q, parts, kind, alibi=False, softmax_scale=None):
    k_code, k_scale, v_code, v_scale = parts
    cu = torch.tensor([0, len(k_code)], dtype=torch.int32, device=DEV)
    return api.quantized_fwd(q[None], ref.pack(k_code, kind), ref.pack(v_code, kind), k_scale.float(), v_scale.float(), cu,
                             is_alibi=alibi, softmax_scale=softmax_scale, return_lse=True)


def check(api, q, parts, kind, alibi=False, softmax_scale=None, what=""):
    parts = [parts[0], parts[1].float(), parts[2], parts[3].float()]
    o, lse = run(api, q, parts, kind, alibi, softmax_scale)
    found = weight_bounds.attend(q, *parts, alibi=alibi, softmax_scale=softmax_scale)
    tol, tol_lse = weight_bounds.bounds(found, len(parts[0]), 11, o.dtype)
    assert ((lse[0].double() - found["lse"]).abs() <= tol_lse).all(), f"{what} lse: off by {(lse[0].double() - found['lse']).abs().max()}"
    over = (o[0].double() - found["o"]).abs() / tol
    assert (over <= 1.0).all(), f"{what}: {over.max().item():.3g} of the bound"  # (NaN is over it)


def query(hq, dim, dtype, seed=5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(1, dim, device=DEV, generator=g).to(dtype).expand(hq, -1).contiguous()


@pytest.mark.parametrize("kind,hq,hk,dim", CODES + STREAM)
def test_the_leading_key_has_a_v_row_of_zeros(api, kind, hq, hk, dim):
    """By so much that the weights of all others are below what fp32 holds, and by less."""
    q = query(hq, dim, torch.bfloat16)
    for nats in (200.0, 95.0, 82.0, 60.0, 12.0):
        for n in (300, 3000):
            for j in (0, 130, n - 1):
                parts = cache_of(n, hk, dim, kind, 6)
                raise_key(q, parts[0], parts[1], j, nats)
                parts[2][j], parts[3][j] = 0.0, 0.0
                check(api, q, parts, kind, what=f"{kind} {hq}/{hk} {dim} {nats} nats, {n} keys, key {j}")


@pytest.mark.parametrize("kind,hq,hk,dim", CODES + STREAM)
def test_zero_v_rows_at_the_end_under_alibi(api, kind, hq, hk, dim):
    n = 700
    parts = cache_of(n, hk, dim, kind, 7)
    parts[2][-300:], parts[3][-300:] = 0.0, 0.0
    check(api, query(hq, dim, torch.bfloat16), parts, kind, alibi=True, what=kind)


def test_all_v_rows_are_zeros(api):
    for kind in KINDS:
        parts = cache_of(400, 2, 128, kind, 8)
        parts[2].zero_()
        parts[3].zero_()
        q = query(8, 128, torch.float16)
        check(api, q, parts, kind, what=kind)
        assert (run(api, q, parts, kind)[0] == 0).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("kind,hq,hk,dim", CODES + STREAM)
def test_one_key_far_ahead_of_many(api, kind, hq, hk, dim, dt):
    """The leading key's V row is zero in half of the dims: there the output is what the many small weights come to, and
    none of them may be lost, while the leading weight itself is an ordinary one."""
    q = query(hq, dim, DTYPES[dt])
    for n, nats, j in ((20000, 16.0, 0), (20000, 14.0, 19999), (6000, 17.0, 3000)):
        parts = cache_of(n, hk, dim, kind, 9)
        raise_key(q, parts[0], parts[1], j, nats)
        parts[2][j, :, ::2] = 0.0
        check(api, q, parts, kind, what=f"{kind} {hq}/{hk} {dim} {dt} {nats} nats, key {j} of {n}")


@pytest.mark.parametrize("kind,hq,hk,dim", CODES + STREAM)
def test_v_rows_of_any_size(api, kind, hq, hk, dim):
    """Stretches of a sequence whose V scales are 2^100 apart, next to scores that rise, fall or stay."""
    n = 1000
    q = query(hq, dim, torch.bfloat16)
    for sizes in ((0, -100, 0), (-100, 0, -100, 100), (100, 0, -100), (-60, -100, 40, 100, 0), (0, 0, -100), (60, -60, 60), (0, 112, -100), (112,), (-100,)):
        for slope in (0.0, 2.0, -2.0):
            parts = cache_of(n, hk, dim, kind, 10)
            at = torch.arange(n, device=DEV) * len(sizes) // n
            parts[3] *= torch.exp2(torch.tensor(sizes, device=DEV, dtype=torch.float32)[at]).unsqueeze(-1)
            parts[0][:] = parts[0][:1]  # equal scores, times the ramp
            parts[1][:] = parts[1][:1] * torch.exp2(slope * torch.linspace(-2, 2, n, device=DEV)).unsqueeze(-1) * 8
            check(api, q, parts, kind, what=f"{kind} {hq}/{hk} {dim} {sizes} slope {slope}")


@pytest.mark.parametrize("kind,dim", [("int8", 128), ("fp8", 128), ("int8", 96), ("int4", 64), ("fp8", 64)])
def test_one_key_far_ahead_in_a_block_with_many(api, kind, dim):
    """With as many heads as this a block has thousands of keys, which share its references with the leading one."""
    hk, n = 128, 40000
    q = query(hk, dim, torch.float16)
    parts = cache_of(n, hk, dim, kind, 11)
    for j in (0, 20011):
        raise_key(q, parts[0], parts[1], j, 16.0)
        parts[2][j, :, ::2] = 0.0
    few = slice(0, hk, 41)
    o, lse = run(api, q, parts, kind)
    found = weight_bounds.attend(q[few], parts[0][:, few], parts[1][:, few].float(), parts[2][:, few], parts[3][:, few].float())
    tol, tol_lse = weight_bounds.bounds(found, n, 11, o.dtype)
    assert ((lse[0, few].double() - found["lse"]).abs() <= tol_lse).all()
    over = (o[0, few].double() - found["o"]).abs() / tol
    assert (over <= 1.0).all(), f"{kind} {dim}: {over.max().item():.3g} of the bound"


@pytest.mark.parametrize("kind,hq,hk,dim", CODES + STREAM)
def test_scores_near_the_end_of_fp32(api, kind, hq, hk, dim):
    """Keys that are all alike, with scores of +-2^122: the output is the mean of V."""
    for sign in (-1.0, 1.0):
        for n in (5, 300):
            parts = cache_of(n, hk, dim, kind, 12)
            parts[0][:], parts[1][:] = 4.0, 2.0 ** 60
            q = torch.full((hq, dim), sign * 2.0 ** 60 / dim, device=DEV).to(torch.bfloat16)
            check(api, q, parts, kind, softmax_scale=1.0, what=f"{kind} {sign} {n}")


@pytest.mark.parametrize("kind,hq,hk,dim", CODES + STREAM)
def test_largest_and_smallest_queries(api, kind, hq, hk, dim):
    for at, scale in ((127, 2.0 ** -30), (126, 2.0 ** -30), (-90, 2.0 ** 80)):
        parts = cache_of(200, hk, dim, kind, 13)
        parts[1] *= 2.0 ** (-95 if at > 0 else 5)
        q = (query(hq, dim, torch.float32).clamp(-1.9, 1.9) * 2.0 ** (at - 64) * 2.0 ** 64).to(torch.bfloat16)
        check(api, q, parts, kind, softmax_scale=scale, what=f"{kind} 2^{at}")
