"""GPU tests of caches whose elements and bytes are counted past 2^32: rows at the end give what the same rows give in a small cache."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAGE = 64
CODE = {"fp8": torch.float8_e4m3fn, "int8": torch.int8, "int4": torch.uint8}


@pytest.fixture(scope="module")
def api():
    import decoding_attention_b200
    return decoding_attention_b200


def rows(n, hk, dim, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(n, hk, dim, device=DEV, generator=g).to(torch.bfloat16)


def cache(kind, total, hk, dim):
    width = dim // 2 if kind == "int4" else dim
    return ([torch.zeros(total, hk, width, dtype=torch.uint8, device=DEV).view(CODE[kind]) for _ in range(2)]
            + [torch.zeros(total, hk, device=DEV) for _ in range(2)])


@pytest.mark.parametrize("kind,hq,hk,dim", [("fp8", 32, 8, 128), ("int8", 64, 8, 128), ("int4", 16, 8, 256)])
def test_codes(api, kind, hq, hk, dim):
    n = 640
    width = dim // 2 if kind == "int4" else dim
    total = -(-((1 << 32) // (hk * width) + 4 * n) // PAGE) * PAGE
    first = total - n
    big, small = cache(kind, total, hk, dim), cache(kind, n, hk, dim)
    k, v = rows(n, hk, dim, 1), rows(n, hk, dim, 2)
    slots = torch.arange(n, device=DEV)
    api.kv_cache_write(k, v, *small, slots=slots)
    api.kv_cache_write(k, v, *big, slots=slots + first)
    for a, b in zip(small, big):
        assert torch.equal(a.view(torch.uint8), b[first:].view(torch.uint8)) and not b[:n].view(torch.uint8).any()
    for a, b in zip(api.kv_cache_read(*small), api.kv_cache_read(*big, slots=slots + first)):
        assert torch.equal(a, b)
    q = rows(2, hq, dim, 3)
    lens = torch.tensor([0, 200, n], dtype=torch.int32, device=DEV)
    want = api.quantized_fwd(q, *small, lens)
    assert torch.equal(api.quantized_fwd(q, *big, lens + first), want)
    paged = [[t.view(-1, PAGE, *t.shape[1:]) for t in side] for side in (small, big)]
    table = torch.arange(n // PAGE, device=DEV, dtype=torch.int32).repeat(2, 1)
    cu = torch.tensor([0, 200, 200 + n], dtype=torch.int32, device=DEV)
    want = api.quantized_fwd(q, *paged[0], cu, block_table=table)
    assert torch.equal(api.quantized_fwd(q, *paged[1], cu, block_table=table + first // PAGE), want)


def test_prefix_pool(api):
    hq, hk, dim, n = 32, 8, 128, 640
    total = -(-((1 << 32) // (hk * dim) + 4 * n) // PAGE) * PAGE
    first = total - n
    pools = [torch.zeros(total, hk, dim, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    k, v = rows(n, hk, dim, 1), rows(n, hk, dim, 2)
    pools[0][first:], pools[1][first:] = k, v
    q = rows(3, hq, dim, 3)
    cu = torch.tensor([0, 64, 64, 100], dtype=torch.int32, device=DEV)
    table = torch.tensor([[8, 0], [0, 0], [9, 0]], dtype=torch.int32, device=DEV)
    prefix = torch.arange(8, device=DEV, dtype=torch.int32)
    small = [x.view(-1, PAGE, hk, dim) for x in (k, v)]
    big = [x.view(-1, PAGE, hk, dim) for x in pools]
    for length in (512, 500):
        want = api.shared_prefix_fwd(q, None, None, *small, cu, block_table=table, prefix_table=prefix, prefix_len=length)
        got = api.shared_prefix_fwd(q, None, None, *big, cu, block_table=table + first // PAGE, prefix_table=prefix + first // PAGE,
                                    prefix_len=length)
        assert torch.equal(got, want)
    # rows of their own, a packed batch that begins far into its tensor
    lens = torch.tensor([0, 20, 20, 100], dtype=torch.int32, device=DEV)
    want = api.shared_prefix_fwd(q, k[:512], v[:512], k[512:], v[512:], lens)
    got = api.shared_prefix_fwd(q, pools[0][first:first + 512], pools[1][first:first + 512], *pools, lens + first + 512)
    assert torch.equal(got, want)
