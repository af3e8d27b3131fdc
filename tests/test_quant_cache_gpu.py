"""GPU tests of the quantised cache with a scale per (token, KV head): writing rows, reading them back, decode
attention over them, against plain 64-bit forms."""
import math

import pytest
import torch

import quant_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
KINDS = ["fp8", "int8", "int4"]
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def api():
    import decoding_attention_b200
    return decoding_attention_b200


def rows(n, hk, dim, dtype, seed, spread=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, hk, dim, device=DEV, generator=g)
    x *= torch.exp(spread * torch.randn(n, hk, 1, device=DEV, generator=g))
    return x.to(dtype)


def empty_cache(n, hk, dim, kind, seed=99):
    """A cache full of stale rows."""
    c, s = ref.quantise(rows(n, hk, dim, torch.float32, seed), kind)
    return ref.pack(c, kind), s


def same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


# ---- writing and reading ---------------------------------------------------------------------

@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
def test_write_is_the_definition_bit_by_bit(api, kind, dt, dim):
    for n, hk in ((1, 1), (37, 5), (2500, 8)):
        k, v = rows(n, hk, dim, DTYPES[dt], 1), rows(n, hk, dim, DTYPES[dt], 2)
        total = n + 61
        kc, ks = empty_cache(total, hk, dim, kind)
        vc, vs = empty_cache(total, hk, dim, kind, 98)
        slots = torch.randperm(total, device=DEV)[:n]
        expect = []
        for x, cache, scale in ((k, kc, ks), (v, vc, vs)):
            codes, s = ref.quantise(x, kind)
            e_c, e_s = cache.clone(), scale.clone()
            e_c.view(torch.uint8)[slots] = ref.pack(codes, kind).view(torch.uint8)
            e_s[slots] = s
            expect += [e_c, e_s]
        api.kv_cache_write(k, v, kc, vc, ks, vs, slots=slots)
        for got, want, what in zip((kc, ks, vc, vs), expect, ("k codes", "k scales", "v codes", "v scales")):
            # (e4m3 has two zeros; a value of either sign that rounds to zero keeps its sign in both)
            assert same(got, want), f"{what} n={n} hk={hk}"


@pytest.mark.parametrize("kind", KINDS)
def test_write_skips_padding_and_slots_outside_and_takes_strided_rows(api, kind):
    n, hk, dim, total = 40, 4, 128, 64
    fused = rows(n, 3 * hk, dim, torch.bfloat16, 3)  # q, k and v of a token side by side
    k, v = fused[:, hk:2 * hk], fused[:, 2 * hk:]
    kc, ks = empty_cache(total, hk, dim, kind)
    vc, vs = empty_cache(total, hk, dim, kind, 98)
    before = [t.clone() for t in (kc, ks, vc, vs)]
    slots = torch.randperm(total, device=DEV)[:n]
    slots[::5] = -1
    slots[1], slots[2], slots[3] = total, 1 << 40, -(1 << 62)
    paged = [t.view(4, 16, *t.shape[1:]) for t in (kc, vc, ks, vs)]
    api.kv_cache_write(k, v, *paged, slots=slots)
    kept = (slots >= 0) & (slots < total)
    for x, cache, scale, c0, s0 in ((k, kc, ks, before[0], before[1]), (v, vc, vs, before[2], before[3])):
        codes, s = ref.quantise(x[kept], kind)
        c0.view(torch.uint8)[slots[kept]] = ref.pack(codes, kind).view(torch.uint8)
        s0[slots[kept]] = s
        assert same(cache, c0) and torch.equal(scale, s0)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
def test_special_rows(api, kind, dt):
    """Zeros, the smallest and largest numbers, infinities and NaN; rows that tie between two codes."""
    dtype = DTYPES[dt]
    fin = torch.finfo(dtype)
    x = rows(12, 2, 64, dtype, 4)
    x[0] = 0
    x[1] = fin.smallest_normal / 2 ** 4
    x[2, :, ::2] = fin.max
    x[3, 0, 5] = math.inf
    x[4, 1, 63] = -math.inf
    x[5, 0, 0] = math.nan
    x[6] = fin.min
    x[7] = 0
    x[7, :, 3] = fin.tiny
    x[8] = -0.0
    # the largest is Q, so the scale is 1 and halves tie
    half = torch.arange(64, device=DEV, dtype=torch.float32) / 2
    x[9] = (half % 7).to(dtype)
    x[9, :, 0] = ref.QMAX[kind]
    if dt == "bf16":
        x[10] = 2.0 ** -101  # below the smallest row that is kept
        x[11] = 2.0 ** -100
    kc, ks = empty_cache(12, 2, 64, kind)
    vc, vs = empty_cache(12, 2, 64, kind)
    api.kv_cache_write(x, x, kc, vc, ks, vs)
    codes, s = ref.quantise(x, kind)
    assert same(kc, ref.pack(codes, kind)) and same(vc, kc)
    assert torch.equal(torch.nan_to_num(ks, nan=-1.0), torch.nan_to_num(s, nan=-1.0)) and same(ks, vs)
    k, _ = api.kv_cache_read(kc, vc, ks, vs, dtype=dtype)
    bad = torch.isnan(s)
    assert bad.sum() == 3 and torch.isnan(k[bad]).all() and torch.isfinite(k[~bad]).all()


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", KINDS)
def test_read(api, kind, dtype, dim):
    for n, hk in ((1, 1), (33, 3), (3001, 8)):
        total = 2 * n + 5
        kc, ks = empty_cache(total, hk, dim, kind, 7)
        vc, vs = empty_cache(total, hk, dim, kind, 8)
        slots = torch.randint(0, total, (n,), device=DEV)  # a row may be read twice
        if n > 4:
            slots[2], slots[3] = -1, total
        k, v = api.kv_cache_read(kc, vc, ks, vs, slots=slots, dtype=dtype)
        inside = ((slots >= 0) & (slots < total)).view(-1, 1, 1)
        for got, cache, scale in ((k, kc, ks), (v, vc, vs)):
            at = slots.clamp(0, total - 1)
            want = (ref.unpack(cache, kind)[at].float() * scale[at].unsqueeze(-1)).to(dtype)
            assert got.dtype == dtype and torch.equal(got, torch.where(inside, want, torch.zeros_like(want)))
        full_k, _ = api.kv_cache_read(kc, vc, ks, vs, dtype=dtype)
        assert torch.equal(full_k, (ref.unpack(kc, kind).float() * ks.unsqueeze(-1)).to(dtype))


def test_read_into_given_tensors(api):
    kc, ks = empty_cache(50, 4, 128, "int8", 7)
    vc, vs = empty_cache(50, 4, 128, "int8", 8)
    both = torch.full((50, 8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    k, v = api.kv_cache_read(kc, vc, ks, vs, out=(both[:, :4], both[:, 4:]))
    assert k.data_ptr() == both.data_ptr()
    k2, v2 = api.kv_cache_read(kc, vc, ks, vs)
    assert torch.equal(both, torch.cat((k2, v2), 1))


# ---- decode attention ------------------------------------------------------------------------

def problem(kind, dtype, lens, hq, hk, dim, seed, page=0, k_spread=0.5, v_spread=0.5, poison=True):
    """q, caches (packed or paged) whose unused rows hold NaN, and each sequence's rows in 64 bits."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(len(lens), hq, dim, device=DEV, generator=g).to(dtype)
    cu = torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)
    table = None
    if page:
        blocks = [-(-n // page) for n in lens]
        pages = sum(blocks) + 2
        order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
        table = torch.full((len(lens), max(blocks + [1])), 1 << 30, dtype=torch.int32, device=DEV)  # (unused entries: no page)
        at = 0
        for b, nb in enumerate(blocks):
            table[b, :nb] = order[at:at + nb]
            at += nb
        total = pages * page
        where = [(table[b].long().clamp(max=pages - 1).repeat_interleave(page) * page
                  + torch.arange(page, device=DEV).repeat(table.shape[1]))[:n] for b, n in enumerate(lens)]
    else:
        total = sum(lens) + 9
        where = [torch.arange(int(cu[b]), int(cu[b]) + n, device=DEV) for b, n in enumerate(lens)]
    out = []
    used = torch.zeros(total, dtype=torch.bool, device=DEV)
    for w in where:
        used[w] = True
    for i, spread in ((1, k_spread), (2, v_spread)):
        codes, s = ref.quantise(rows(total, hk, dim, dtype, seed + i, spread), kind)
        cache = ref.pack(codes, kind)
        wide = ref.unpack(cache, kind) * s.double().unsqueeze(-1)
        if poison:
            cache.view(torch.uint8)[~used] = 0x7F
            s = torch.where(used.unsqueeze(-1), s, torch.full_like(s, math.nan))
        out.append((cache, s, [wide[w] for w in where]))
    (kc, ks, k), (vc, vs, v) = out
    if page:
        kc, ks, vc, vs = [t.view(-1, page, *t.shape[1:]) for t in (kc, ks, vc, vs)]
    return dict(q=q, cu=cu, table=table, kc=kc, ks=ks, vc=vc, vs=vs, k=k, v=v, lens=lens)


def check(api, pr, alibi=False, softmax_scale=None, what=""):
    o, lse = api.quantized_fwd(pr["q"], pr["kc"], pr["vc"], pr["ks"], pr["vs"], pr["cu"], is_alibi=alibi,
                               softmax_scale=softmax_scale, return_lse=True, block_table=pr["table"])
    assert o.shape == pr["q"].shape and o.dtype == pr["q"].dtype
    compare(o, lse, pr, alibi, softmax_scale, what)
    return o, lse


def compare(o, lse, pr, alibi=False, softmax_scale=None, what=""):
    for b, n in enumerate(pr["lens"]):
        e_o, e_lse, spread, scores, top = ref.attend(pr["q"][b], pr["k"][b], pr["v"][b], alibi, softmax_scale)
        if n == 0:
            assert (o[b] == 0).all() and torch.isneginf(lse[b]).all(), f"{what} empty row {b}"
            continue
        tol_o, tol_lse = ref.bounds(e_o, e_lse, spread, scores, top, n, 11, o.dtype)
        assert ((lse[b].double() - e_lse).abs() <= tol_lse).all(), f"{what} lse of {b}: {(lse[b].double() - e_lse).abs().max()}"
        over = ((o[b].double() - e_o).abs() - tol_o).max().item()
        assert over <= 0, f"{what} sequence {b} of {n} keys: over the bound by {over}"


LENS = [0, 1, 15, 16, 17, 31, 32, 33, 700, 0, 64, 1300, 3, 257]


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("kind", KINDS)
def test_decode_kinds_and_dims(api, kind, dim):
    for dt, hq, hk in (("fp16", 8, 8), ("bf16", 32, 8), ("bf16", 20, 2)):
        pr = problem(kind, DTYPES[dt], LENS, hq, hk, dim, 11)
        check(api, pr, what=f"{kind} {dim} {dt} {hq}/{hk}")


@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 1), (8, 1), (9, 1), (16, 1), (17, 1), (32, 1), (64, 1), (100, 1), (10, 5),
                                   (6, 3), (21, 7), (64, 64), (12, 12)])
def test_decode_head_layouts(api, hq, hk):
    for kind, alibi in (("int8", True), ("int4", False)):
        pr = problem(kind, torch.bfloat16, [300, 0, 1, 2100], hq, hk, 64, 12)
        check(api, pr, alibi=alibi, what=f"{kind} {hq}/{hk}")


@pytest.mark.parametrize("page", [1, 2, 16, 64, 256])
@pytest.mark.parametrize("kind", KINDS)
def test_decode_paged(api, kind, page):
    pr = problem(kind, torch.float16, LENS, 16, 4, 128, 13, page=page)
    check(api, pr, alibi=page == 16, what=f"page {page}")


def test_decode_masks_bad_pages_and_rows(api):
    """Pages and rows outside the cache are masked, not read."""
    pr = problem("fp8", torch.bfloat16, [200, 130, 64], 8, 2, 128, 14, page=16)
    pr["table"][0, 3] = -1
    pr["table"][0, 5] = 1 << 20
    pr["table"][2, :4] = -5
    keep = torch.ones(200, dtype=torch.bool, device=DEV)
    keep[48:64] = False
    keep[80:96] = False
    pr["k"][0], pr["v"][0] = pr["k"][0][keep], pr["v"][0][keep]
    pr["k"][2], pr["v"][2] = pr["k"][2][:0], pr["v"][2][:0]
    pr["lens"] = [168, 130, 0]
    check(api, pr, what="bad pages")
    # a table narrower than the lengths say: the keys behind it are masked
    pr = problem("int8", torch.bfloat16, [200, 40], 8, 2, 128, 15, page=16)
    pr["table"] = pr["table"][:, :4].contiguous()
    pr["k"][0], pr["v"][0], pr["lens"] = pr["k"][0][:64], pr["v"][0][:64], [64, 40]
    check(api, pr, what="narrow table")
    # packed: lengths that run past the cache
    pr = problem("int8", torch.float16, [50, 60], 8, 2, 128, 16)
    n = 80
    for t in ("kc", "ks", "vc", "vs"):
        pr[t] = pr[t][:n].contiguous()
    pr["k"][1], pr["v"][1], pr["lens"] = pr["k"][1][:30], pr["v"][1][:30], [50, 30]
    check(api, pr, what="short cache")


@pytest.mark.parametrize("kind", KINDS)
def test_decode_many_and_long_sequences(api, kind):
    """Sequences that span several CTAs next to ones that do not; a table with a row stride."""
    pr = problem(kind, torch.bfloat16, [5000, 20000, 1, 0, 7, 9000], 32, 8, 128, 17)
    check(api, pr, what="long")
    pr = problem(kind, torch.float16, [(i * 37) % 190 for i in range(300)], 8, 2, 64, 18, page=16)
    wide = torch.full((300, pr["table"].shape[1] + 5), 1 << 29, dtype=torch.int32, device=DEV)
    wide[:, :-5] = pr["table"]
    pr["table"] = wide[:, :-5]
    check(api, pr, alibi=True, what="many")


@pytest.mark.parametrize("kind", KINDS)
def test_decode_scales_that_differ_widely(api, kind):
    """V rows whose scales differ by 2^20 and more, the row that decides among the smallest; K scores that rise to the end
    or start at their largest."""
    pr = problem(kind, torch.bfloat16, [400, 900], 8, 2, 128, 19, v_spread=6.0, poison=False)
    check(api, pr, softmax_scale=0.02, what="v spread")
    for order in (1.0, -1.0):
        pr = problem(kind, torch.float16, [600], 4, 1, 64, 20, v_spread=3.0, poison=False)
        ramp = torch.exp2(order * torch.linspace(-6, 6, 609, device=DEV)).view(-1, 1)
        pr["ks"] = pr["ks"] * ramp
        pr["k"][0] = (ref.unpack(pr["kc"], kind) * pr["ks"].double().unsqueeze(-1))[:600]
        small = pr["vs"].clone()
        big = (pr["q"].double()[0, 0] @ pr["k"][0][:, 0].T).argmax()
        small[big] = 2.0 ** -30
        pr["vs"] = small
        pr["v"][0] = (ref.unpack(pr["vc"], kind) * pr["vs"].double().unsqueeze(-1))[:600]
        check(api, pr, what=f"ramp {order}")


def test_decode_queries_of_extreme_size(api):
    """q is brought to fp16 by a power of two per head: heads of any magnitude, zero heads among them."""
    pr = problem("int8", torch.bfloat16, [100, 333], 8, 2, 128, 21)
    size = torch.tensor([2.0 ** -60, 2.0 ** -20, 1.0, 0.0, 2.0 ** 10, 2.0 ** -5, 2.0 ** -126, 2.0 ** 3], device=DEV).view(1, 8, 1)
    pr["q"] = (pr["q"].float() * size).to(torch.bfloat16)
    check(api, pr, what="q sizes")


@pytest.mark.parametrize("dim", [96, 128])
@pytest.mark.parametrize("kind", KINDS)
def test_decode_many_short_sequences_of_every_head_layout(api, kind, dim):
    """More (sequence, KV head) pairs than the GPU holds blocks, a few keys each."""
    lens = [(i * 53) % 97 for i in range(150)]
    for hq, hk, page in ((32, 8, 0), (8, 8, 16), (12, 4, 1)):
        check(api, problem(kind, torch.bfloat16, lens, hq, hk, dim, 26, page=page), alibi=page == 1, what=f"{kind} {hq}/{hk} page {page}")


@pytest.mark.parametrize("page", [16, 64, 512])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_decode_long_ragged_pages_with_bias(api, kind, page):
    """Tiles of several pages, pages of several tiles, cuts and ends inside both, walked from the end."""
    for lens, hq, hk, dim in (([6001, 0, 129, 12345, 128, 2], 8, 4, 96), ([40001], 16, 4, 128), ([3000] * 5 + [1], 5, 5, 128)):
        check(api, problem(kind, torch.float16, lens, hq, hk, dim, 28, page=page), alibi=True, what=f"{lens} {hq}/{hk}")


@pytest.mark.parametrize("kind", KINDS)
def test_lengths_that_are_not_cumulative_stay_inside(api, kind):
    """What comes out is unspecified then; nothing around the output changes and the next call is right."""
    pr = problem(kind, torch.bfloat16, [700, 20, 300, 5, 60], 32, 8, 128, 29)
    for cu in ([0, 900, 100, 2000, 50, 1085], [500, 400, 300, 200, 100, 0], [-7, 3, 2 ** 31 - 1, 0, 5, 9], [2 ** 31 - 1] * 5 + [-2 ** 31]):
        wide = torch.full((5, 40, 128), 3.0, dtype=torch.bfloat16, device=DEV)
        api.quantized_fwd(pr["q"], pr["kc"], pr["vc"], pr["ks"], pr["vs"], torch.tensor(cu, dtype=torch.int32, device=DEV),
                          out=wide[:, 4:36])
        assert (wide[:, :4] == 3.0).all() and (wide[:, 36:] == 3.0).all()
    check(api, pr)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_calls_right_behind_the_writes_of_their_inputs(api, kind):
    """Fresh caches, memory traffic just before the call (late tiles), long and short sequences in one block."""
    for seed in range(12):
        pr = problem(kind, torch.bfloat16, [5000, 20000, 1, 0, 7, 9000], 32, 8, 128, 200 + seed, poison=seed % 2 == 0)
        junk = torch.full((48 << 20,), float(seed), device=DEV)
        del junk
        check(api, pr, what=f"seed {seed}")


def test_more_keys_in_a_block_than_its_integers_hold(api):
    """Equal scores and the largest codes: every weight counts, sums pass 2^31 unless they are taken over in time."""
    n, hk = 101000, 128
    g = torch.Generator(device=DEV).manual_seed(27)
    kc = torch.zeros(n, hk, 128, dtype=torch.int8, device=DEV)
    vc = torch.full((n, hk, 128), 127, dtype=torch.int8, device=DEV)
    vc[:, 1::2] = -127
    ks, vs = torch.ones(n, hk, device=DEV), torch.full((n, hk), 0.5, device=DEV)
    q = torch.randn(1, hk, 128, device=DEV, generator=g).to(torch.bfloat16)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    o, lse = api.quantized_fwd(q, kc, vc, ks, vs, cu, return_lse=True)
    want = torch.full((hk, 1), 63.5, device=DEV)
    want[1::2] = -63.5
    assert (o[0].float() == want).all() and (lse - math.log(n)).abs().max() <= 2e-5


def test_nan_and_infinity_reach_the_sequences_that_hold_them_only(api):
    pr = problem("int8", torch.bfloat16, [100, 333, 50], 8, 2, 128, 22, poison=False)
    pr["vs"][100 + 200, 1] = math.nan
    o, lse = api.quantized_fwd(pr["q"], pr["kc"], pr["vc"], pr["ks"], pr["vs"], pr["cu"], return_lse=True)
    assert torch.isnan(o[1, 4:]).all() and torch.isfinite(o[1, :4]).all()
    assert torch.isfinite(o[0]).all() and torch.isfinite(o[2]).all() and torch.isfinite(lse).all()
    pr["ks"][7, 0] = math.nan
    o, lse = api.quantized_fwd(pr["q"], pr["kc"], pr["vc"], pr["ks"], pr["vs"], pr["cu"], return_lse=True)
    assert torch.isnan(o[0, :4]).all() and torch.isnan(lse[0, :4]).all() and torch.isfinite(o[0, 4:]).all()


def test_results_do_not_depend_on_what_else_is_in_the_batch_layout(api):
    """Two runs agree bit for bit; an out tensor with a row stride, q rows inside a fused tensor."""
    pr = problem("fp8", torch.bfloat16, [513, 4000, 0, 9], 32, 8, 128, 23)
    o1, lse1 = check(api, pr)
    fused = torch.randn(4, 48, 128, device=DEV).to(torch.bfloat16)
    fused[:, :32] = pr["q"]
    wide = torch.full((4, 40, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    out = wide[:, :32]
    o2, lse2 = api.quantized_fwd(fused[:, :32], pr["kc"], pr["vc"], pr["ks"], pr["vs"], pr["cu"], out=out, return_lse=True)
    assert o2.data_ptr() == wide.data_ptr() and torch.equal(o1, o2) and torch.equal(lse1, lse2)
    assert (wide[:, 32:] == 3.0).all()


def test_inputs_whose_elements_are_apart(api):
    pr = problem("int8", torch.float16, [40, 0, 300], 8, 2, 64, 34)
    o, _ = check(api, pr)
    apart = torch.stack((pr["q"], torch.full_like(pr["q"], math.nan)), -1).flatten(-2)[..., ::2]
    assert apart.stride(-1) == 2 and torch.equal(api.quantized_fwd(apart, pr["kc"], pr["vc"], pr["ks"], pr["vs"], pr["cu"]), o)
    x = rows(7, 2, 64, torch.float16, 35)
    a, b = [[torch.zeros(7, 2, 64, dtype=torch.int8, device=DEV) for _ in range(2)] + [torch.zeros(7, 2, device=DEV) for _ in range(2)]
            for _ in range(2)]
    api.kv_cache_write(x, 2 * x, *a)
    api.kv_cache_write(torch.stack((x, x), -1)[..., 0], x.transpose(0, 2).contiguous().transpose(0, 2) * 2, *b)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_two_streams_and_graph_replay(api):
    pr = problem("int8", torch.bfloat16, [513, 4000, 0, 9, 77], 32, 8, 128, 24)
    args = (pr["q"], pr["kc"], pr["vc"], pr["ks"], pr["vs"], pr["cu"])
    want = api.quantized_fwd(*args)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(api.quantized_fwd(*args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    out = torch.zeros_like(want)
    k_new, v_new = rows(3, 8, 128, torch.bfloat16, 31), rows(3, 8, 128, torch.bfloat16, 32)
    slots = torch.tensor([600, -1, 2], device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        api.kv_cache_write(k_new, v_new, pr["kc"], pr["vc"], pr["ks"], pr["vs"], slots=slots)
        api.quantized_fwd(*args, out=out)
    graph.replay()
    torch.cuda.synchronize()
    first = out.clone()
    assert not torch.equal(first, want)
    assert torch.equal(first, api.quantized_fwd(*args))
    k_new.copy_(rows(3, 8, 128, torch.bfloat16, 33))
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(out, first) and torch.equal(out, api.quantized_fwd(*args))


@pytest.mark.parametrize("kind", KINDS)
def test_write_decode_and_read_as_a_server_uses_them(api, kind):
    """Prompts are written page by page, a few tokens are decoded and appended, the context is read back."""
    hq, hk, dim, page, batch = 16, 4, 128, 16, 5
    lens = [33, 16, 0, 100, 1]
    steps = 3
    width = -(-(max(lens) + steps) // page)
    pages = batch * width
    table = torch.randperm(pages, device=DEV).to(torch.int32).view(batch, width)
    code = {"fp8": torch.float8_e4m3fn, "int8": torch.int8, "int4": torch.uint8}[kind]
    cd = dim // 2 if kind == "int4" else dim
    kc = torch.zeros(pages, page, hk, cd, dtype=torch.uint8, device=DEV).view(code)
    vc = torch.zeros_like(kc)
    ks, vs = torch.zeros(pages, page, hk, device=DEV), torch.zeros(pages, page, hk, device=DEV)

    def slot(b, j):
        return int(table[b, j // page]) * page + j % page

    held = [([], []) for _ in range(batch)]

    def append(k, v, where):
        api.kv_cache_write(k, v, kc, vc, ks, vs, slots=torch.tensor([slot(b, j) for b, j in where], device=DEV))
        for i, (b, _) in enumerate(where):
            for x, keep in ((k, held[b][0]), (v, held[b][1])):
                codes, s = ref.quantise(x[i], kind)
                keep.append(codes * s.double().unsqueeze(-1))

    n = sum(lens)
    append(rows(n, hk, dim, torch.bfloat16, 41), rows(n, hk, dim, torch.bfloat16, 42),
           [(b, j) for b in range(batch) for j in range(lens[b])])
    for step in range(steps):
        append(rows(batch, hk, dim, torch.bfloat16, 50 + step), rows(batch, hk, dim, torch.bfloat16, 60 + step),
               [(b, lens[b]) for b in range(batch)])
        lens = [x + 1 for x in lens]
        pr = dict(q=torch.randn(batch, hq, dim, device=DEV).to(torch.bfloat16), table=table, kc=kc, ks=ks, vc=vc, vs=vs,
                  cu=torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32), lens=lens,
                  k=[torch.stack(h[0]) for h in held], v=[torch.stack(h[1]) for h in held])
        check(api, pr, what=f"step {step}")
    slots = torch.tensor([slot(b, j) for b in range(batch) for j in range(lens[b])], device=DEV)
    k, v = api.kv_cache_read(kc, vc, ks, vs, slots=slots, dtype=torch.float32)
    assert torch.equal(k.double(), torch.cat(pr["k"]).float().double())
    assert torch.equal(v.double(), torch.cat(pr["v"]).float().double())


# ---- refusals --------------------------------------------------------------------------------

def test_refusals(api):
    pr = problem("int8", torch.bfloat16, [20, 30], 8, 2, 128, 25)
    q, kc, vc, ks, vs, cu = [pr[t] for t in ("q", "kc", "vc", "ks", "vs", "cu")]
    n = 4
    k = rows(n, 2, 128, torch.bfloat16, 1)
    slots = torch.arange(n, device=DEV)
    bad = [
        lambda: api.quantized_fwd(q.float(), kc, vc, ks, vs, cu),
        lambda: api.quantized_fwd(q, kc.float(), vc.float(), ks, vs, cu),
        lambda: api.quantized_fwd(q, kc, vc.view(torch.float8_e4m3fn), ks, vs, cu),
        lambda: api.quantized_fwd(q, kc, vc, ks.half(), vs.half(), cu),
        lambda: api.quantized_fwd(q, kc, vc, ks[:-1], vs, cu),
        lambda: api.quantized_fwd(q, kc, vc, ks, vs, cu.long()),
        lambda: api.quantized_fwd(q, kc, vc, ks, vs, cu[:-1]),
        lambda: api.quantized_fwd(q, kc, vc, ks, vs, cu.cpu()),
        lambda: api.quantized_fwd(q[:, :7], kc, vc, ks, vs, cu),
        lambda: api.quantized_fwd(q[..., :64].contiguous(), kc, vc, ks, vs, cu),
        lambda: api.quantized_fwd(q, kc.transpose(0, 1), vc.transpose(0, 1), ks, vs, cu),
        lambda: api.quantized_fwd(q, kc, vc, ks, vs, cu, block_table=torch.zeros(2, 3, dtype=torch.int32, device=DEV)),
        lambda: api.quantized_fwd(q, kc[:56].view(-1, 8, 2, 128), vc[:56].view(-1, 8, 2, 128), ks[:56].view(-1, 8, 2), vs[:56].view(-1, 8, 2), cu),
        lambda: api.quantized_fwd(q, kc[:57].view(-1, 3, 2, 128), vc[:57].view(-1, 3, 2, 128), ks[:57].view(-1, 3, 2),
                                  vs[:57].view(-1, 3, 2), cu, block_table=torch.zeros(2, 3, dtype=torch.int32, device=DEV)),
        lambda: api.quantized_fwd(q, kc, vc, ks, vs, cu, out=torch.empty(2, 8, 128, device=DEV)),
        lambda: api.quantized_fwd(q, kc, vc, ks, vs, cu, out=torch.empty(2, 8, 64, dtype=q.dtype, device=DEV)),
        lambda: api.kv_cache_write(k.float(), k.float(), kc, vc, ks, vs, slots=slots),
        lambda: api.kv_cache_write(k, k.half(), kc, vc, ks, vs, slots=slots),
        lambda: api.kv_cache_write(k, k[:3], kc, vc, ks, vs, slots=slots),
        lambda: api.kv_cache_write(k, k, kc, vc, ks, vs, slots=slots.int()),
        lambda: api.kv_cache_write(k, k, kc, vc, ks, vs, slots=slots[:3]),
        lambda: api.kv_cache_write(k[:, :1], k[:, :1], kc, vc, ks, vs, slots=slots),
        lambda: api.kv_cache_write(rows(100, 2, 128, torch.bfloat16, 1), rows(100, 2, 128, torch.bfloat16, 1), kc, vc, ks, vs),
        lambda: api.kv_cache_read(kc, vc, ks, vs, dtype=torch.float64),
        lambda: api.kv_cache_read(kc, vc, ks, vs, slots=slots.cpu()),
        lambda: api.kv_cache_read(kc, vc, ks, vs, out=(torch.empty(3, 2, 128, dtype=torch.bfloat16, device=DEV),) * 2),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((RuntimeError, TypeError)):
            call()
            pytest.fail(f"call {i} was not refused")
    # nothing to do is not an error
    api.kv_cache_write(k[:0], k[:0], kc, vc, ks, vs, slots=slots[:0])
    a, b = api.kv_cache_read(kc, vc, ks, vs, slots=slots[:0])
    assert a.shape == (0, 2, 128) and b.shape == (0, 2, 128)
    o, lse = api.quantized_fwd(q, kc[:0], vc[:0], ks[:0], vs[:0], torch.zeros_like(cu), return_lse=True)
    assert (o == 0).all() and torch.isneginf(lse).all()
