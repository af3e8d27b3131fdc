"""GPU tests of decode attention behind a prefix that the batch shares, against a plain 64-bit form."""
import pytest
import torch

import quant_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
BITS = {torch.float16: 11, torch.bfloat16: 8}


@pytest.fixture(scope="module")
def api():
    import decoding_attention_b200
    return decoding_attention_b200


def rows(n, hk, dim, dtype, gen, spread=0.5):
    x = torch.randn(n, hk, dim, device=DEV, generator=gen)
    return (x * torch.exp(spread * torch.randn(n, hk, 1, device=DEV, generator=gen))).to(dtype)


def problem(dtype, prefix, lens, hq, hk, dim, seed, kind=None, page=0, prefix_page=0, one_pool=False):
    """The call's tensors, and each sequence's keys in 64 bits.  Rows that are no keys hold NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    batch = len(lens)
    q = torch.randn(batch, hq, dim, device=DEV, generator=g).to(dtype)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)
    pre = [rows(prefix, hk, dim, dtype, g) for _ in range(2)]
    own = [rows(sum(lens), hk, dim, dtype, g) for _ in range(2)]
    args = dict(k_scale=None, v_scale=None, block_table=None, prefix_table=None, prefix_len=None)
    wide = [x.double() for x in own]
    blocks = [-(-n // page) for n in lens] if page else []
    shared = -(-prefix // prefix_page) if prefix_page else 0
    pool_pages = (sum(blocks) + (shared if one_pool else 0) + 2) if page else 0
    order = torch.randperm(max(pool_pages, 1), device=DEV, generator=g).to(torch.int32)
    if page:
        table = torch.full((batch, max(blocks + [1])), 1 << 29, dtype=torch.int32, device=DEV)
        at = 0
        for b, n in enumerate(blocks):
            table[b, :n] = order[at:at + n]
            at += n
        args["block_table"] = table
        where = torch.cat([(table[b, :blocks[b]].long().repeat_interleave(page) * page
                            + torch.arange(page, device=DEV).repeat(blocks[b]))[:n] for b, n in enumerate(lens)])
        total = pool_pages * page
    else:
        where = torch.arange(sum(lens), device=DEV)
        total = sum(lens) + 3
    store = []
    for i, t in enumerate(("k", "v")):
        if kind:
            codes, s = ref.quantise(own[i], kind)
            packed = ref.pack(codes, kind)
            wide[i] = codes * s.double().unsqueeze(-1)
            cache = torch.full((total, *packed.shape[1:]), 0x7F, dtype=torch.uint8, device=DEV)
            cache[where] = packed.view(torch.uint8)
            scale = torch.full((total, hk), float("nan"), device=DEV)
            scale[where] = s
            cache = cache.view(packed.dtype)
            args[t + "_scale"] = scale.view(-1, page, hk) if page else scale
        else:
            cache = torch.full((total, hk, dim), float("nan"), dtype=dtype, device=DEV)
            cache[where] = own[i]
        store.append(cache.view(-1, page, *cache.shape[1:]) if page else cache)
    pk, pv = pre
    if prefix_page:
        args["prefix_len"] = prefix
        if one_pool:
            ids = order[sum(blocks):sum(blocks) + shared].contiguous()
            pools = store
        else:
            ids = torch.randperm(shared + 2, device=DEV, generator=g)[:shared].to(torch.int32).contiguous()
            pools = [torch.full((shared + 2, prefix_page, hk, dim), float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
        at = (ids.long().repeat_interleave(prefix_page) * prefix_page + torch.arange(prefix_page, device=DEV).repeat(shared))[:prefix]
        for pool, x in zip(pools, pre):
            pool.view(-1, hk, dim)[at] = x
        args["prefix_table"] = ids
        pk, pv = (None, None) if one_pool else pools
    at = cu.tolist()
    keys = [[torch.cat((pre[i].double(), wide[i][at[b]:at[b + 1]])) for b in range(batch)] for i in range(2)]
    return dict(q=q, pk=pk, pv=pv, k=store[0], v=store[1], cu=cu, args=args, keys=keys)


def call(api, pr, **more):
    return api.shared_prefix_fwd(pr["q"], pr["pk"], pr["pv"], pr["k"], pr["v"], pr["cu"], return_lse=True, **pr["args"], **more)


def check(api, pr, alibi=False, softmax_scale=None, what=""):
    o, lse = call(api, pr, is_alibi=alibi, softmax_scale=softmax_scale)
    assert o.shape == pr["q"].shape and o.dtype == pr["q"].dtype
    for b in range(len(pr["q"])):
        k, v = pr["keys"][0][b], pr["keys"][1][b]
        if len(k) == 0:
            assert (o[b] == 0).all() and torch.isneginf(lse[b]).all(), f"{what} row {b}"
            continue
        e_o, e_lse, spread, scores, top = ref.attend(pr["q"][b], k, v, alibi, softmax_scale)
        tol_o, tol_lse = ref.bounds(e_o, e_lse, spread, scores, top, len(k), BITS[o.dtype], o.dtype)
        assert ((lse[b].double() - e_lse).abs() <= tol_lse).all(), f"{what} lse of {b}: {(lse[b].double() - e_lse).abs().max()}"
        over = ((o[b].double() - e_o).abs() - tol_o).max().item()
        assert over <= 0, f"{what} sequence {b}: over the bound by {over}"
    return o, lse


LENS = [0, 1, 17, 64, 200, 0, 33]


@pytest.mark.parametrize("prefix", [1, 15, 127, 128, 129, 256, 1000, 5003])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
def test_prefix_lengths(api, dt, prefix):
    check(api, problem(DTYPES[dt], prefix, LENS, 32, 8, 128, prefix), what=f"{prefix}")


@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 4), (6, 2), (5, 1), (16, 2), (32, 1), (33, 1), (100, 1), (128, 1), (12, 4), (64, 2)])
def test_head_layouts(api, hq, hk, dim):
    for batch in (1, 5):
        lens = [(7 * i) % 50 for i in range(batch)]
        check(api, problem(torch.bfloat16, 700, lens, hq, hk, dim, 3), alibi=dim == 96, what=f"{hq}/{hk} {dim} batch {batch}")


@pytest.mark.parametrize("batch", [2, 31, 32, 33, 64, 65, 100, 129])
def test_batches_around_a_row_tile(api, batch):
    """One row tile, two, an odd number of them; the last one full or with a single sequence."""
    lens = [(13 * i) % 70 for i in range(batch)]
    check(api, problem(torch.float16, 900, lens, 8, 2, 64, 4), what=f"batch {batch}")
    check(api, problem(torch.bfloat16, 333, lens, 3, 1, 128, 5), alibi=True, what=f"batch {batch}, 3 heads")


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("one_pool", [False, True])
def test_paged_prefix(api, page, one_pool):
    for prefix in (1, 100, 777, 1024):
        pr = problem(torch.bfloat16, prefix, LENS, 16, 4, 128, 6, page=page, prefix_page=page, one_pool=one_pool)
        check(api, pr, what=f"page {page} prefix {prefix}")
    pr = problem(torch.float16, 600, LENS, 8, 4, 96, 7, page=1, prefix_page=page)
    check(api, pr, alibi=True, what="own keys in pages of one")


@pytest.mark.parametrize("kind", ["fp8", "int8", "int4"])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_own_keys_as_codes(api, kind, dim):
    check(api, problem(torch.bfloat16, 500, LENS, 16, 2, dim, 8, kind=kind), what=kind)
    check(api, problem(torch.float16, 300, LENS, 40, 2, dim, 9, kind=kind, page=16, prefix_page=64), alibi=True, what=kind + " paged")


def test_no_prefix_and_no_own_keys(api):
    pr = problem(torch.bfloat16, 0, LENS, 16, 4, 128, 10)
    check(api, pr, what="no prefix")
    pr = problem(torch.bfloat16, 500, [0, 0, 0], 16, 4, 128, 11)
    check(api, pr, what="no own keys")
    pr = problem(torch.float16, 0, [0, 0], 16, 4, 64, 12)
    check(api, pr, what="nothing")
    pr = problem(torch.bfloat16, 200, LENS, 16, 4, 128, 13)
    pr["args"]["prefix_len"] = 150  # fewer than there are
    pr["keys"] = [[torch.cat((x[:150], x[200:])) for x in side] for side in pr["keys"]]
    check(api, pr, what="part of the rows")


def test_long_prefix_many_sequences(api):
    lens = [(i * 29) % 300 for i in range(200)]
    check(api, problem(torch.bfloat16, 9000, lens, 16, 4, 128, 14), what="bf16")
    check(api, problem(torch.float16, 3300, lens, 32, 1, 64, 15), alibi=True, what="MQA")


# Enough key tiles to fill the GPU: the SMs are divided by the lengths that the device finds.
@pytest.mark.parametrize("hq,hk,dim,batch", [(32, 8, 128, 70), (16, 16, 64, 130), (24, 3, 96, 150), (64, 1, 128, 90)])
@pytest.mark.parametrize("kind", [None, "fp8", "int8", "int4"])
def test_own_keys_next_to_a_long_prefix(api, hq, hk, dim, batch, kind):
    prefix = 2500 if hk > 1 else 5000
    for top in (3, 130, 900):  # hardly any own keys, some, more than the prefix
        lens = [(i * 37) % (top + 1) for i in range(batch)]
        page = 64 if top == 130 else 0
        check(api, problem(torch.bfloat16, prefix, lens, hq, hk, dim, 30, kind=kind, page=page), alibi=top == 900, what=f"{kind} {top}")


def test_two_streams_with_work_for_all_sms(api):
    """Calls that divide the SMs, next to one another and to calls with codes: each result is that of the call alone."""
    prs = [problem(torch.bfloat16, 3000, [(i * 41) % 700 for i in range(90)], 32, 8, 128, 32 + j, kind=kind)
           for j, kind in enumerate((None, "fp8"))]
    want = [check(api, pr) for pr in prs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for turn in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(((turn + i) % 2, call(api, prs[(turn + i) % 2])))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[j][0]) and torch.equal(lse, want[j][1]) for j, (o, lse) in got)


def test_replay_with_other_lengths(api):
    """A captured call is used with lengths that change which SMs do what."""
    batch, hq, hk, dim, prefix = 70, 32, 8, 128, 2500
    pr = problem(torch.bfloat16, prefix, [800] * batch, hq, hk, dim, 31)
    full = pr["cu"].clone()
    keys = pr["keys"]
    buf = torch.zeros_like(pr["q"])
    call(api, pr)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, lse = call(api, pr, out=buf)
    for n in (800, 0, 1, 300, 20, 799):
        pr["cu"].copy_((torch.arange(batch + 1, device=DEV) * n).to(torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        o2, lse2 = call(api, pr)
        assert torch.equal(buf, o2) and torch.equal(lse, lse2)
        own = [[torch.cat([x[prefix:] for x in side]) for side in keys]][0]
        pr["keys"] = [[torch.cat((side[b][:prefix], own[i][b * n:(b + 1) * n])) for b in range(batch)] for i, side in enumerate(keys)]
        check(api, pr, what=f"{n} own keys")
    pr["cu"].copy_(full)


@pytest.mark.parametrize("alibi", [False, True])
def test_scores_that_rise_and_fall(api, alibi):
    """Row maxima that move by far more than the lazy reference allows, in either direction, and a long softmax scale."""
    for order in (1.0, -1.0):
        pr = problem(torch.bfloat16, 1500, [40, 0, 300], 32, 4, 128, 16)
        ramp = torch.exp2(order * torch.linspace(-4, 4, 1500, device=DEV)).view(-1, 1, 1)
        pr["pk"] = (pr["pk"].float() * ramp).to(torch.bfloat16)
        for b in range(3):
            pr["keys"][0][b][:1500] = pr["pk"].double()
        check(api, pr, alibi=alibi, softmax_scale=0.5, what=f"ramp {order}")


def test_nan_in_the_prefix_reaches_all_and_in_own_keys_one(api):
    pr = problem(torch.bfloat16, 300, [40, 0, 100], 8, 2, 128, 17)
    pr["v"][41 + 20, 1, 5] = float("nan")
    o, lse = call(api, pr)
    assert torch.isnan(o[2, 4:, 5]).all() and torch.isfinite(o[2, :4]).all() and torch.isfinite(o[:2]).all()
    pr["pk"][7, 0] = float("nan")
    o, lse = call(api, pr)
    assert torch.isnan(o[:, :4]).all() and torch.isnan(lse[:, :4]).all() and torch.isfinite(o[:2, 4:]).all()


def test_prefix_pages_outside_the_pool_read_as_zeros(api):
    pr = problem(torch.bfloat16, 256, [10, 20], 8, 2, 128, 18, page=64, prefix_page=64)
    pr["args"]["prefix_table"][1] = -1
    pr["args"]["prefix_table"][3] = 1 << 20
    for side in pr["keys"]:
        for x in side:
            x[64:128] = 0
            x[192:256] = 0
    check(api, pr, what="bad pages")


def test_strides_out_streams_and_graphs(api):
    pr = problem(torch.bfloat16, 1100, [40, 0, 300, 7], 16, 4, 128, 19)
    o1, lse1 = check(api, pr)
    wide_q = torch.randn(4, 24, 128, device=DEV).to(torch.bfloat16)
    wide_q[:, :16] = pr["q"]
    both = torch.cat((pr["pk"], pr["pv"]), 1)  # K and V rows of a token side by side
    own = torch.cat((pr["k"], pr["v"]), 1)
    out = torch.full((4, 20, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    o2, lse2 = api.shared_prefix_fwd(wide_q[:, :16], both[:, :4], both[:, 4:], own[:, :4], own[:, 4:], pr["cu"], out=out[:, :16],
                                     return_lse=True)
    assert torch.equal(o1, o2) and torch.equal(lse1, lse2) and (out[:, 16:] == 3.0).all()
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(call(api, pr))
    torch.cuda.synchronize()
    assert all(torch.equal(o, o1) and torch.equal(l, lse1) for o, l in outs)
    buf = torch.zeros_like(o1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(api, pr, out=buf)
    for _ in range(3):
        buf.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(buf, o1)
    pr["q"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(buf, o1) and torch.equal(buf, call(api, pr)[0])


def test_agrees_with_the_unshared_call(api):
    """The same keys, laid out once per sequence, through dmha_fwd."""
    pr = problem(torch.float16, 640, [40, 1, 300], 32, 8, 128, 20)
    o, lse = check(api, pr)
    k = torch.cat([x.half() for x in pr["keys"][0]])
    v = torch.cat([x.half() for x in pr["keys"][1]])
    lens = [len(x) for x in pr["keys"][0]]
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)
    o2, lse2 = api.dmha_fwd(pr["q"], k, v, cu, max(lens), return_lse=True)
    assert (o.float() - o2.float()).abs().max().item() <= 4e-3 and (lse - lse2).abs().max().item() <= 1e-4


def test_a_server_with_a_quantised_context(api):
    """A prompt is stored as codes; its rows are read back once as the shared prefix of a batch whose new tokens are
    written, quantised, behind it."""
    g = torch.Generator(device=DEV).manual_seed(30)
    hk, hq, dim, n, batch = 4, 16, 128, 700, 9
    k, v = rows(n, hk, dim, torch.bfloat16, g), rows(n, hk, dim, torch.bfloat16, g)
    kc, vc = [torch.zeros(n, hk, dim, dtype=torch.int8, device=DEV) for _ in range(2)]
    ks, vs = [torch.zeros(n, hk, device=DEV) for _ in range(2)]
    api.kv_cache_write(k, v, kc, vc, ks, vs)
    pk, pv = api.kv_cache_read(kc, vc, ks, vs, dtype=torch.bfloat16)
    page = 16
    pool = [torch.zeros(batch + 2, page, hk, dim, dtype=torch.int8, device=DEV) for _ in range(2)]
    scales = [torch.zeros(batch + 2, page, hk, device=DEV) for _ in range(2)]
    table = torch.randperm(batch + 2, device=DEV)[:batch].to(torch.int32).view(batch, 1)
    held = [[pk.double()] * batch, [pv.double()] * batch]
    for step in range(3):
        new = [rows(batch, hk, dim, torch.bfloat16, g) for _ in range(2)]
        api.kv_cache_write(*new, *pool, *scales, slots=table[:, 0].long() * page + step)
        for i in range(2):
            codes, s = ref.quantise(new[i], "int8")
            x = codes * s.double().unsqueeze(-1)
            held[i] = [torch.cat((held[i][b], x[b:b + 1])) for b in range(batch)]
        pr = dict(q=torch.randn(batch, hq, dim, device=DEV, generator=g).to(torch.bfloat16), pk=pk, pv=pv, k=pool[0], v=pool[1],
                  cu=(torch.arange(batch + 1, device=DEV) * (step + 1)).to(torch.int32),
                  args=dict(k_scale=scales[0], v_scale=scales[1], block_table=table, prefix_table=None, prefix_len=None), keys=held)
        check(api, pr, what=f"step {step}")


def test_refusals(api):
    pr = problem(torch.bfloat16, 100, [20, 30], 8, 2, 128, 25)
    paged = problem(torch.bfloat16, 100, [20, 30], 8, 2, 128, 25, page=16, prefix_page=16, one_pool=True)
    q, pk, pv, k, v, cu = [pr[t] for t in ("q", "pk", "pv", "k", "v", "cu")]
    t = paged["args"]["prefix_table"]
    bt = paged["args"]["block_table"]
    f = api.shared_prefix_fwd
    bad = [
        lambda: f(q.float(), pk.float(), pv.float(), k.float(), v.float(), cu),
        lambda: f(q, pk.half(), pv.half(), k, v, cu),
        lambda: f(q, pk, pv, k.half(), v.half(), cu),
        lambda: f(q, pk, None, k, v, cu),
        lambda: f(q, None, None, k, v, cu),
        lambda: f(q, pk[:, :1], pv[:, :1], k, v, cu),
        lambda: f(q, pk, pv[:50], k, v, cu),
        lambda: f(q, pk, pv, k, v[:-1], cu),
        lambda: f(q, pk, pv, k, v, cu.long()),
        lambda: f(q, pk, pv, k, v, cu[:2]),
        lambda: f(q[:, :7], pk, pv, k, v, cu),
        lambda: f(q, pk, pv, k, v, cu, prefix_len=101),
        lambda: f(q, pk, pv, k, v, cu, prefix_len=-1),
        lambda: f(q, pk, pv, k, v, cu, k_scale=torch.ones(53, 2, device=DEV)),
        lambda: f(q, pk, pv, k, v, cu, block_table=bt),
        lambda: f(q, pk, pv, paged["k"], paged["v"], cu),
        lambda: f(q, None, None, paged["k"], paged["v"], cu, block_table=bt, prefix_table=t),
        lambda: f(q, None, None, paged["k"], paged["v"], cu, block_table=bt, prefix_table=t, prefix_len=16 * len(t) + 1),
        lambda: f(q, None, None, paged["k"], paged["v"], cu, block_table=bt, prefix_table=t.long(), prefix_len=100),
        lambda: f(q, pk.view(-1, 10, 2, 128), pv.view(-1, 10, 2, 128), k, v, cu, prefix_table=t, prefix_len=20),
        lambda: f(q, pk, pv, k, v, cu, out=torch.empty(2, 8, 128, device=DEV)),
        lambda: f(torch.randn(2, 2, 256, device=DEV).bfloat16(), torch.zeros(9, 1, 256, device=DEV).bfloat16(),
                  torch.zeros(9, 1, 256, device=DEV).bfloat16(), torch.zeros(50, 1, 256, device=DEV).bfloat16(),
                  torch.zeros(50, 1, 256, device=DEV).bfloat16(), cu),
        lambda: f(torch.randn(2, 129, 64, device=DEV).half(), *[torch.zeros(50, 1, 64, device=DEV).half() for _ in range(4)], cu),
    ]
    for i, run in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError)):
            run()
            pytest.fail(f"call {i} was not refused")
