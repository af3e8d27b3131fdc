"""GPU tests of tensors whose rows share memory (expanded over tokens or sequences): inputs give what their copies give,
outputs are refused.  The unquantised calls are held to the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def api():
    import decoding_attention_b200
    return decoding_attention_b200


def rand(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def cache(n, hk, dim):
    return [torch.zeros(n, hk, dim, dtype=torch.int8, device=DEV) for _ in range(2)] + [torch.zeros(n, hk, device=DEV) for _ in range(2)]


def one_and_overlapping(n, heads, dim, seed, dtype=torch.bfloat16):
    """Rows that are all the same one, and rows that start half a row behind the one before."""
    yield rand(1, heads, dim, seed=seed, dtype=dtype).expand(n, -1, -1)
    flat = rand((n + 1) * heads * dim // 2, seed=seed, dtype=dtype)
    yield flat.as_strided((n, heads, dim), (heads * dim // 2, dim, 1))


@pytest.mark.parametrize("tokens", [2, 37])
def test_write_of_expanded_rows(api, tokens):
    for k, v in zip(one_and_overlapping(tokens, 4, 128, 1), one_and_overlapping(tokens, 4, 128, 2)):
        got, want = cache(tokens, 4, 128), cache(tokens, 4, 128)
        api.kv_cache_write(k, v, *got)
        api.kv_cache_write(k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format), *want)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[2].min() > 0


def test_decode_of_one_query_for_many_sequences(api):
    lens = [40, 0, 300, 7, 1]
    caches = cache(sum(lens), 2, 128)
    api.kv_cache_write(rand(sum(lens), 2, 128, seed=1), rand(sum(lens), 2, 128, seed=2), *caches)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)
    for q in one_and_overlapping(len(lens), 8, 128, 3):
        want = api.quantized_fwd(q.clone(memory_format=torch.contiguous_format), *caches, cu)
        assert torch.equal(api.quantized_fwd(q, *caches, cu), want)


@pytest.mark.parametrize("batch", [2, 64])
def test_prefix_call_with_expanded_inputs(api, batch):
    hq, hk, dim, n = 16, 4, 128, 500
    cu = (torch.arange(batch + 1, device=DEV) * 3).to(torch.int32)
    pk, pv, k, v = [rand(m, hk, dim, seed=i) for i, m in enumerate((n, n, 3 * batch, 3 * batch))]
    for q in one_and_overlapping(batch, hq, dim, 9):
        want = api.shared_prefix_fwd(q.clone(memory_format=torch.contiguous_format), pk, pv, k, v, cu)
        assert torch.equal(api.shared_prefix_fwd(q, pk, pv, k, v, cu), want)
    q = rand(batch, hq, dim, seed=9)
    for a, b in zip(one_and_overlapping(n, hk, dim, 5), one_and_overlapping(n, hk, dim, 6)):
        want = api.shared_prefix_fwd(q, *[x.clone(memory_format=torch.contiguous_format) for x in (a, b)], k, v, cu)
        assert torch.equal(api.shared_prefix_fwd(q, a, b, k, v, cu), want)
    for a, b in zip(one_and_overlapping(3 * batch, hk, dim, 7), one_and_overlapping(3 * batch, hk, dim, 8)):
        want = api.shared_prefix_fwd(q, pk, pv, *[x.clone(memory_format=torch.contiguous_format) for x in (a, b)], cu)
        assert torch.equal(api.shared_prefix_fwd(q, pk, pv, a, b, cu), want)


def test_expanded_query_in_a_captured_call(api):
    cu = torch.tensor([0, 5, 9, 9, 30], dtype=torch.int32, device=DEV)
    q1 = rand(1, 16, 128, seed=1)
    rest = [rand(m, 4, 128, seed=i) for i, m in enumerate((200, 200, 30, 30))]
    out = torch.zeros(4, 16, 128, dtype=torch.bfloat16, device=DEV)
    api.shared_prefix_fwd(q1.expand(4, -1, -1), *rest, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.shared_prefix_fwd(q1.expand(4, -1, -1), *rest, cu, out=out)
    q1.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, api.shared_prefix_fwd(q1.repeat(4, 1, 1), *rest, cu))


def test_outputs_whose_rows_overlap_are_refused(api):
    caches = cache(20, 2, 128)
    api.kv_cache_write(rand(20, 2, 128, seed=1), rand(20, 2, 128, seed=2), *caches)
    cu = torch.tensor([0, 8, 20], dtype=torch.int32, device=DEV)
    q = rand(2, 8, 128, seed=3)
    pk, pv = rand(50, 2, 128, seed=4), rand(50, 2, 128, seed=5)
    k, v = api.kv_cache_read(*caches)
    for bad in one_and_overlapping(2, 8, 128, 6):
        with pytest.raises(RuntimeError, match="rows of its own"):
            api.quantized_fwd(q, *caches, cu, out=bad)
        with pytest.raises(RuntimeError, match="rows of its own"):
            api.shared_prefix_fwd(q, pk, pv, k, v, cu, out=bad)
    for bad in one_and_overlapping(20, 2, 128, 7):
        with pytest.raises(RuntimeError, match="rows of its own"):
            api.kv_cache_read(*caches, out=(bad, torch.empty_like(v)))
        with pytest.raises(RuntimeError, match="rows of its own"):
            api.kv_cache_read(*caches, out=(torch.empty_like(k), bad))
    # one row overlaps with none, whatever its stride
    o = torch.empty(8, 128, dtype=torch.bfloat16, device=DEV).as_strided((1, 8, 128), (0, 128, 1))
    assert torch.equal(api.quantized_fwd(q[:1], *caches, cu[:2], out=o), api.quantized_fwd(q[:1], *caches, cu[:2]))


def copied(x):
    return x.clone(memory_format=torch.contiguous_format)


@pytest.mark.parametrize("hq,hk", [(8, 8), (16, 4), (32, 1)])
def test_unquantised_calls_with_expanded_inputs(api, hq, hk):
    lens = [40, 0, 300, 7, 1]
    n, batch, dim = sum(lens), len(lens), 128
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)
    q, k, v = rand(batch, hq, dim, seed=1), rand(n, hk, dim, seed=2), rand(n, hk, dim, seed=3)
    for x in one_and_overlapping(batch, hq, dim, 4):
        assert torch.equal(api.dmha_fwd(x, k, v, cu, 300), api.dmha_fwd(copied(x), k, v, cu, 300))
        assert torch.equal(api.decoding_attn_fwd(x, k, v, cu, 300, dim, False), api.dmha_fwd(copied(x), k, v, cu, 300))
    for a, b in zip(one_and_overlapping(n, hk, dim, 5), one_and_overlapping(n, hk, dim, 6)):
        assert torch.equal(api.dmha_fwd(q, a, b, cu, 300), api.dmha_fwd(q, copied(a), copied(b), cu, 300))
    table = torch.arange(batch * 20, device=DEV).to(torch.int32).view(batch, 20)
    pools = rand(batch * 20, 16, hk, dim, seed=7), rand(batch * 20, 16, hk, dim, seed=8)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for x in one_and_overlapping(batch, hq, dim, 9):
        assert torch.equal(api.paged_fwd(x, *pools, lengths, table), api.paged_fwd(copied(x), *pools, lengths, table))
    for bad in one_and_overlapping(batch, hq, dim, 10):
        with pytest.raises(RuntimeError, match="rows of its own"):
            api.dmha_fwd(q, k, v, cu, 300, out=bad)
        with pytest.raises(RuntimeError, match="rows of its own"):
            api.paged_fwd(q, *pools, lengths, table, out=bad)


def test_latent_cache_with_expanded_inputs(api):
    cu = torch.tensor([0, 50, 50, 90], dtype=torch.int32, device=DEV)
    q, kv = rand(3, 16, 576, seed=1), rand(90, 1, 576, seed=2)
    for x in one_and_overlapping(3, 16, 576, 3):
        assert torch.equal(api.dmla_fwd(x, kv, cu, 50), api.dmla_fwd(copied(x), kv, cu, 50))
    for x in one_and_overlapping(90, 1, 576, 4):
        assert torch.equal(api.dmla_fwd(q, x, cu, 50), api.dmla_fwd(q, copied(x), cu, 50))
    for bad in one_and_overlapping(3, 16, 512, 5):
        with pytest.raises(RuntimeError, match="rows of its own"):
            api.dmla_fwd(q, kv, cu, 50, out=bad)
