"""Workloads of the operators around a quantised or shared KV cache, each with its plain form.

write   quantise the K and V rows of new tokens into a cache, one scale per (token, KV head)
read    the rows of such a cache, back in 16 bits
decode  decode attention over such a cache, packed or paged
prefix  decode attention of a batch whose sequences share a prefix, which is computed once for all of them

With ``own = False`` ``run`` computes an operator with elementary torch operations in 32 bits (the codes of
``write`` in 64: a product next to the border between two codes has to fall on the right side), with
``own = True`` it calls this package.  ``exact`` has the definitions again, in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
QMAX = {"fp8": 448.0, "int8": 127.0, "int4": 7.0}   # the largest code of a format
BYTES = {"fp8": 1.0, "int8": 1.0, "int4": 0.5, "none": 2.0}
TINY = 2.0 ** -100                                  # a row whose largest magnitude is below this is stored as zeros


# ---- the cases -------------------------------------------------------------------------------

def listed():
    return [
        # One decoding step of 256 sequences (32/8 heads of 128): 256 tokens go to scattered rows of a paged pool.
        {"name": "write_step_fp8", "op": "write", "kind": "fp8", "dtype": "bf16", "tokens": 256, "head_k": 8, "dim": 128,
         "rows": 16384, "scatter": True, "padding": 5},
        # A 32 768-token prompt is stored after its forward pass.
        {"name": "write_prompt_int8", "op": "write", "kind": "int8", "dtype": "fp16", "tokens": 32768, "head_k": 8,
         "dim": 128, "rows": 32768, "scatter": False, "padding": 0},
        # The context of 16 sequences of 8 192 tokens is brought back to bf16, page by page, for a prompt's next chunk.
        {"name": "read_context_fp8", "op": "read", "kind": "fp8", "dtype": "bf16", "tokens": 131072, "head_k": 8,
         "dim": 128, "rows": 140000, "scatter": True, "padding": 0},
        # A short piece of one sequence, odd in length, in the smallest format and an odd head dim.
        {"name": "read_piece_int4", "op": "read", "kind": "int4", "dtype": "fp16", "tokens": 1111, "head_k": 8,
         "dim": 96, "rows": 2048, "scatter": True, "padding": 3},
        # The small MHA workload: 4 sequences of 1 024 keys, 32 heads.
        {"name": "decode_mha_int8", "op": "decode", "kind": "int8", "dtype": "fp16", "batch": 4, "lo": 1024, "hi": 1024,
         "head_q": 32, "head_k": 32, "dim": 128, "alibi": False, "page": 0, "lens": 1},
        # The headline workload of the framework with an FP8 cache: 256 sequences of 512..4096 keys, 32/8 heads.
        {"name": "decode_gqa_fp8", "op": "decode", "kind": "fp8", "dtype": "bf16", "batch": 256, "lo": 512, "hi": 4096,
         "head_q": 32, "head_k": 8, "dim": 128, "alibi": False, "page": 0, "lens": 2},
        # The MQA workload with ALiBi and a 4-bit cache.
        {"name": "decode_mqa_int4", "op": "decode", "kind": "int4", "dtype": "fp16", "batch": 128, "lo": 2048, "hi": 2048,
         "head_q": 32, "head_k": 1, "dim": 128, "alibi": True, "page": 0, "lens": 3},
        # One long sequence of 131 072 keys, 32 heads, in 64-key pages.
        {"name": "decode_long_int8", "op": "decode", "kind": "int8", "dtype": "bf16", "batch": 1, "lo": 131072, "hi": 131072,
         "head_q": 32, "head_k": 32, "dim": 128, "alibi": False, "page": 64, "lens": 4},
        # A few sequences that just started behind a system prompt of 1 024 tokens: latency.
        {"name": "prefix_small", "op": "prefix", "kind": "none", "dtype": "bf16", "batch": 8, "prefix": 1024, "lo": 0, "hi": 64,
         "head_q": 32, "head_k": 8, "dim": 128, "alibi": False, "page": 0, "lens": 5},
        # An ordinary serving batch: 64 sequences behind 8 192 shared tokens, everything in one pool of 64-key pages.
        {"name": "prefix_paged", "op": "prefix", "kind": "none", "dtype": "bf16", "batch": 64, "prefix": 8192, "lo": 64,
         "hi": 1024, "head_q": 32, "head_k": 8, "dim": 128, "alibi": False, "page": 64, "lens": 6},
        # The same with MQA, ALiBi, an odd prefix and the sequences' own keys in FP8.
        {"name": "prefix_mqa_fp8", "op": "prefix", "kind": "fp8", "dtype": "fp16", "batch": 33, "prefix": 5003, "lo": 1,
         "hi": 700, "head_q": 32, "head_k": 1, "dim": 128, "alibi": True, "page": 0, "lens": 7},
        # The largest: 256 sequences sampled from one long context.
        {"name": "prefix_large", "op": "prefix", "kind": "none", "dtype": "bf16", "batch": 256, "prefix": 16384, "lo": 128,
         "hi": 1024, "head_q": 32, "head_k": 8, "dim": 128, "alibi": False, "page": 0, "lens": 8},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "prefix", "prefix"])
    dtype = rng.choice(["fp16", "bf16"])
    if op in ("write", "read"):
        head_k, dim = rng.choice([1, 2, 4, 8, 12, 32]), rng.choice([64, 96, 128, 256])
        most = (33554432 if op == "write" else 134217728) // (head_k * dim)
        tokens = _spread(rng, 1, min(most, 262144))
        scatter = rng.random() < 0.7
        rows = tokens + (rng.randrange(tokens // 4 + 64) if scatter else 0)
        return {"op": op, "kind": rng.choice(["fp8", "int8", "int4"]), "dtype": dtype, "tokens": tokens, "head_k": head_k,
                "dim": dim, "rows": rows, "scatter": scatter, "padding": rng.randrange(8) if scatter and tokens > 8 else 0}
    head_k = rng.choice([1, 1, 2, 4, 5, 8, 32])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16, 32])
    if head_k * group > 64:
        group = 64 // head_k
    case = {"op": op, "dtype": dtype, "head_q": head_k * group, "head_k": head_k, "alibi": rng.random() < 0.3,
            "page": rng.choice([0, 0, 16, 64, 128]), "lens": rng.randrange(1 << 30), "batch": _spread(rng, 1, 256)}
    if op == "decode":
        dim = rng.choice([64, 96, 128, 256])
        # no more padded cache elements than 256 x 4096 x 8 x 128, no more score elements than 256 x 4096 x 32
        most = max(1, min(131072, (1 << 30) // (case["batch"] * head_k * dim), (1 << 25) // (case["batch"] * case["head_q"])))
        hi = _spread(rng, 1, most)
        return {**case, "kind": rng.choice(["fp8", "int8", "int4"]), "dim": dim, "lo": rng.choice([hi, hi // 2, hi // 8]), "hi": hi}
    dim = rng.choice([64, 96, 128])
    most = max(1, min(32768, (1 << 34) // (case["batch"] * case["head_q"] * dim)))
    prefix = _spread(rng, 1, most)
    hi = _spread(rng, 1, max(1, min(1024, (1 << 28) // (case["batch"] * head_k * dim))))
    return {**case, "kind": rng.choice(["none", "none", "fp8", "int8", "int4"]), "dim": dim, "prefix": prefix,
            "lo": rng.choice([0, hi // 2, hi // 8]), "hi": hi}


def _lengths(case):
    r = random.Random(case["lens"])
    return [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]


def work(case):
    hk, d, b = case["head_k"], case["dim"], BYTES[case["kind"]]
    if case["op"] in ("write", "read"):
        n = 2 * case["tokens"] * hk
        return {"bytes": n * (2 * d + d * b + 4) + (8 * case["tokens"] if case["scatter"] else 0), "flops": 2 * n * d}
    keys, hq, batch = sum(_lengths(case)), case["head_q"], case["batch"]
    moved = keys * hk * (2 * d * b + (8 if case["kind"] != "none" else 0)) + batch * hq * (4 * d + 4)
    flops = 4 * keys * hq * d
    if case["op"] == "prefix":
        moved += case["prefix"] * hk * 4 * d
        flops += 4 * batch * case["prefix"] * hq * d
    return {"bytes": moved, "flops": flops}


# ---- what a program has in hand --------------------------------------------------------------

def _rows(n, heads, dim, dtype, gen):
    """K or V rows as a model makes them: normal values, rows of unequal magnitude, a few strong channels."""
    x = torch.randn(n, heads, dim, device=DEV, generator=gen)
    x *= torch.exp(0.5 * torch.randn(n, heads, 1, device=DEV, generator=gen))
    x *= 1.0 + 3.0 * (torch.rand(1, heads, dim, device=DEV, generator=gen) < 0.03)
    return (0.5 * x).to(dtype)


def _codes(x, kind):
    """(codes as float64, fp32 scales) of rows x."""
    amax = x.double().abs().amax(-1)
    fine, most = amax >= TINY, torch.full_like(amax, QMAX[kind])
    # both quotients are rounded once to 32 bits: they are part of the format
    scale = torch.where(fine, amax / most, 0.0).float()
    inverse = torch.where(fine, most / torch.where(fine, amax, 1.0), 0.0).float()
    y = x.double() * inverse.double().unsqueeze(-1)
    if kind != "fp8":
        return torch.round(y), scale
    # e4m3: three bits behind the leading one down to 2^-6, steps of 2^-9 below
    step = torch.exp2(torch.clamp(torch.frexp(y)[1].double() - 1.0, min=-6.0) - 3.0)
    return torch.round(y / step) * step, scale


def _pack(codes, kind):
    """Codes as they lie in the cache."""
    if kind == "fp8":
        return codes.float().to(torch.float8_e4m3fn)
    codes = codes.to(torch.int8)
    if kind == "int8":
        return codes
    return ((codes[..., 0::2] & 15) | ((codes[..., 1::2] & 15) << 4)).view(torch.uint8)


def _unpack(cache, kind):
    """What is stored, as numbers: int8, or float8 values."""
    if kind != "int4":
        return cache
    low, high = (cache << 4).view(torch.int8) >> 4, cache.view(torch.int8) >> 4
    return torch.stack((low, high), -1).flatten(-2)


def _cache(x, kind):
    """A quantised copy of rows x, made piece by piece."""
    parts = [_codes(p, kind) for p in x.split(1 << 16)]
    return torch.cat([_pack(c, kind) for c, _ in parts]), torch.cat([s for _, s in parts])


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, hk, dim, kind = DTYPES[case["dtype"]], case["head_k"], case["dim"], case["kind"]
    if case["op"] in ("write", "read"):
        n, rows = case["tokens"], case["rows"]
        state = {"case": case, "dtype": dtype, "slots": None}
        if case["scatter"]:
            state["slots"] = torch.randperm(rows, device=DEV, generator=gen)[:n].contiguous()
            if case["padding"]:  # a batch that is padded to a fixed size: the last tokens have no row
                state["slots"][n - case["padding"]:] = -1
        if case["op"] == "write":
            state["k"], state["v"] = _rows(n, hk, dim, dtype, gen), _rows(n, hk, dim, dtype, gen)
        for t in ("k", "v"):  # a cache that holds earlier rows
            state[t + "_cache"], state[t + "_scale"] = _cache(_rows(rows, hk, dim, dtype, gen), kind)
        return state
    lens = _lengths(case)
    batch, total, page = case["batch"], sum(lens), case["page"]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    state = {"case": case, "cu_seq_k": cu, "longest": max(lens), "block_table": None, "prefix_table": None,
             "k_prefix": None, "v_prefix": None, "k_scale": None, "v_scale": None,
             "q": torch.randn(batch, case["head_q"], dim, device=DEV, generator=gen).to(dtype)}
    prefix = case.get("prefix", 0)
    blocks = [-(-n // page) for n in lens] if page else []
    if page:
        pages = sum(blocks)
        shared = -(-prefix // page) if kind == "none" else 0  # a 16-bit prefix lies in the same pool
        order = torch.randperm(pages + shared + 3, device=DEV, generator=gen).to(torch.int32)
        table = torch.zeros(batch, max(1, max(blocks)), dtype=torch.int32)
        at = 0
        order_host = order.cpu()
        for b, n in enumerate(blocks):
            table[b, :n] = order_host[at:at + n]
            at += n
        state["block_table"] = table.to(DEV)
        if shared:
            state["prefix_table"] = order[at:at + shared].contiguous()
        total = (pages + shared + 3) * page
    for t in ("k", "v"):
        x = _rows(max(1, total), hk, dim, dtype, gen)
        if kind != "none":
            x, s = _cache(x, kind)
            state[t + "_scale"] = s.view(-1, page, hk) if page else s
        state[t] = x.view(-1, page, hk, x.shape[-1]) if page else x
        if prefix and state["prefix_table"] is None:
            state[t + "_prefix"] = _rows(prefix, hk, dim, dtype, gen)
    return state


# ---- the plain forms -------------------------------------------------------------------------

def _plain_write(state):
    kind, slots = state["case"]["kind"], state["slots"]
    out = {}
    rows = state["case"]["rows"]
    for t in ("k", "v"):
        codes, scale = _codes(state[t], kind)
        cache, scales = _unpack(state[t + "_cache"], kind), state[t + "_scale"]
        codes = codes.float().to(torch.float8_e4m3fn).view(torch.uint8) if kind == "fp8" else codes.to(torch.int8)
        if kind == "fp8":
            cache = cache.view(torch.uint8)
        at = torch.arange(rows, device=DEV) if slots is None else torch.where(slots < 0, rows, slots)  # row `rows` is dropped
        cache = torch.cat((cache, cache[:1])).index_put((at,), codes)[:rows]
        out[t] = cache.view(torch.float8_e4m3fn) if kind == "fp8" else cache
        out[t + "_scale"] = torch.cat((scales, scales[:1])).index_put((at,), scale)[:rows]
    return out


def _plain_read(state):
    kind, slots, out = state["case"]["kind"], state["slots"], {}
    for t in ("k", "v"):
        cache, scales = state[t + "_cache"], state[t + "_scale"]
        if slots is not None:
            at = slots.clamp(min=0)
            cache, scales = cache.view(torch.uint8)[at].view(cache.dtype), scales[at]
        x = _unpack(cache, kind).float() * scales.unsqueeze(-1)
        if slots is not None:
            x = torch.where((slots < 0).view(-1, 1, 1), 0.0, x)
        out[t] = x.to(state["dtype"])
    return out


def _own_keys(state, t):
    """(K or V of every sequence in fp32 [batch, longest, head_k, dim], which of them are keys)."""
    case, cu, table, page = state["case"], state["cu_seq_k"].long(), state["block_table"], state["case"]["page"]
    j = torch.arange(max(1, state["longest"]), device=DEV)
    valid = j < (cu[1:] - cu[:-1]).unsqueeze(1)
    if page:
        rows = table.long()[:, torch.clamp(j // page, max=table.shape[1] - 1)] * page + j % page
    else:
        rows = cu[:-1].unsqueeze(1) + j
    cache = state[t].flatten(0, 1) if page else state[t]
    rows = torch.where(valid, rows, 0)
    x = _unpack(cache.view(torch.uint8)[rows].view(cache.dtype) if case["kind"] == "fp8" else cache[rows], case["kind"]).float()
    if case["kind"] != "none":
        scale = state[t + "_scale"]
        x *= (scale.flatten(0, 1) if page else scale)[rows].unsqueeze(-1)
    return x, valid


def _prefix_rows(state, t):
    if state["prefix_table"] is None:
        return state[t + "_prefix"].float()
    return state[t][state["prefix_table"].long()].flatten(0, 1)[:state["case"]["prefix"]].float()


def _plain_attention(state):
    case = state["case"]
    hq, hk, dim, batch = case["head_q"], case["head_k"], case["dim"], case["batch"]
    group = hq // hk
    q = state["q"].float().view(batch, hk, group, dim)
    cu = state["cu_seq_k"].long()
    prefix = case.get("prefix", 0)
    last = prefix + cu[1:] - cu[:-1] - 1
    slope = torch.exp2(-8.0 * torch.arange(1, hq + 1, device=DEV, dtype=torch.float32) / hq).view(1, hk, group, 1)
    k, valid = _own_keys(state, "k")
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(dim)                                 # [batch, hk, group, keys]
    del k
    if case["alibi"]:
        s += slope * (prefix + torch.arange(s.shape[-1], device=DEV) - last.unsqueeze(1)).view(batch, 1, 1, -1)
    s.masked_fill_(~valid.view(batch, 1, 1, -1), -math.inf)
    top = s.amax(-1, keepdim=True)
    if prefix:
        # the prefix is one matrix for all rows of a KV head
        rows = q.permute(1, 0, 2, 3).reshape(hk, batch * group, dim)
        sp = torch.matmul(rows, _prefix_rows(state, "k").permute(1, 2, 0)).view(hk, batch, group, prefix)
        sp /= math.sqrt(dim)
        sp = sp.permute(1, 0, 2, 3)
        if case["alibi"]:
            sp = sp + slope * (torch.arange(prefix, device=DEV) - last.unsqueeze(1)).view(batch, 1, 1, -1)
        top = torch.maximum(top, sp.amax(-1, keepdim=True))
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    v, _ = _own_keys(state, "v")
    o = torch.matmul(p, v.permute(0, 2, 1, 3))
    del v
    if prefix:
        p = torch.exp(sp - top)
        del sp
        total = total + p.sum(-1, keepdim=True)
        p = p.permute(1, 0, 2, 3).reshape(hk, batch * group, prefix)
        o = o + torch.matmul(p, _prefix_rows(state, "v").permute(1, 0, 2)).view(hk, batch, group, dim).permute(1, 0, 2, 3)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total)).view(batch, hq)
    return {"o": o.reshape(batch, hq, dim).to(state["q"].dtype), "lse": lse}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "decode": _plain_attention, "prefix": _plain_attention}[op](state)
    import decoding_attention_b200 as da
    if op == "write":
        kind = state["case"]["kind"]
        da.kv_cache_write(state["k"], state["v"], state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"],
                          slots=state["slots"])
        return {"k": _unpack(state["k_cache"], kind), "k_scale": state["k_scale"],
                "v": _unpack(state["v_cache"], kind), "v_scale": state["v_scale"]}
    if op == "read":
        k, v = da.kv_cache_read(state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"], slots=state["slots"],
                                dtype=state["dtype"])
        return {"k": k, "v": v}
    if op == "decode":
        o, lse = da.quantized_fwd(state["q"], state["k"], state["v"], state["k_scale"], state["v_scale"], state["cu_seq_k"],
                                  is_alibi=state["case"]["alibi"], return_lse=True, block_table=state["block_table"])
    else:
        o, lse = da.shared_prefix_fwd(state["q"], state["k_prefix"], state["v_prefix"], state["k"], state["v"],
                                      state["cu_seq_k"], is_alibi=state["case"]["alibi"], return_lse=True,
                                      k_scale=state["k_scale"], v_scale=state["v_scale"], block_table=state["block_table"],
                                      prefix_table=state["prefix_table"], prefix_len=state["case"]["prefix"])
    return {"o": o, "lse": lse}


# ---- the definitions in 64 bits --------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "write":
        out = {}
        for t in ("k", "v"):
            x = state[t].double()
            scale = x.abs().max(dim=-1).values / QMAX[case["kind"]]
            ratio = x / torch.where(scale > 0, scale, 1.0)[..., None]
            cache, scales = _unpack(state[t + "_cache"], case["kind"]).to(torch.float64), state[t + "_scale"].double()
            slots = torch.arange(len(x), device=DEV) if state["slots"] is None else state["slots"]
            kept = slots >= 0
            cache[slots[kept]], scales[slots[kept]] = ratio[kept], scale[kept]
            out[t], out[t + "_scale"] = cache if case["kind"] == "fp8" else None, scales
        return out
    if case["op"] == "read":
        out = {}
        for t in ("k", "v"):
            x = _unpack(state[t + "_cache"], case["kind"]).to(torch.float64) * state[t + "_scale"].double()[..., None]
            if state["slots"] is not None:
                x = x[state["slots"]]
                x[state["slots"] < 0] = 0.0
            out[t] = x
        return out
    if work(case)["flops"] > 2e11:
        return None
    hq, hk, dim, page = case["head_q"], case["head_k"], case["dim"], case["page"]
    group, prefix = hq // hk, case.get("prefix", 0)
    cu = state["cu_seq_k"].tolist()
    slopes = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=DEV, dtype=torch.float64) / hq)
    shared = {}
    for t in ("k", "v"):
        if prefix and state["prefix_table"] is None:
            shared[t] = state[t + "_prefix"].double()
        elif prefix:
            shared[t] = torch.cat([state[t][i] for i in state["prefix_table"].tolist()])[:prefix].double()
    o = torch.zeros(case["batch"], hq, dim, device=DEV, dtype=torch.float64)
    lse = torch.full((case["batch"], hq), -math.inf, device=DEV, dtype=torch.float64)
    for b in range(case["batch"]):
        n = cu[b + 1] - cu[b]
        if n + prefix == 0:
            continue
        mine = {}
        for t in ("k", "v"):
            if page:
                ids = state["block_table"][b, :-(-n // page)].long()
                x = _unpack(state[t].view(torch.uint8)[ids].view(state[t].dtype) if case["kind"] == "fp8" else state[t][ids],
                            case["kind"]).flatten(0, 1)[:n].double()
                if case["kind"] != "none":
                    x = x * state[t + "_scale"][ids].flatten(0, 1)[:n, :, None].double()
            else:
                x = _unpack(state[t][cu[b]:cu[b + 1]], case["kind"]).double()
                if case["kind"] != "none":
                    x = x * state[t + "_scale"][cu[b]:cu[b + 1], :, None].double()
            mine[t] = torch.cat((shared[t], x)) if prefix else x
        position = torch.arange(n + prefix, device=DEV, dtype=torch.float64) - (n + prefix - 1)
        for h in range(hk):
            heads = slice(h * group, (h + 1) * group)
            s = state["q"][b, heads].double() @ mine["k"][:, h].T / dim ** 0.5
            if case["alibi"]:
                s = s + slopes[heads, None] * position
            lse[b, heads] = torch.logsumexp(s, 1)
            o[b, heads] = torch.exp(s - lse[b, heads, None]) @ mine["v"][:, h]
    return {"o": o, "lse": lse}
