"""The FP8 key/value cache and the attention that reads it: what is measured.

Four operators: ``write`` (quantise new tokens' K and V into a paged e4m3 cache),
``read`` (gather cached tokens back to fp16 / bf16), ``decode`` (attention of a few
new tokens per sequence over the cache) and ``prefix`` (the same for a batch whose
sequences share their first tokens).

A cache is k, v: e4m3 codes (pages, kv heads, page size, head dim) and k_exp, v_exp:
uint8 (pages, kv heads, page size); a token's head has the value code * 2^(exp - 127).
A new row takes the least power of two that brings its largest magnitude to 448 or
less (2^-63 at least, 1 for a row of zeros); a row with an infinity or a NaN is
marked with 255 and reads as NaN. Sequence b holds seqlens[b] tokens, token t in page
page_table[b, t // page size].
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # One new token for each of 32 running sequences, written between two decode steps.
        {"name": "write-step", "op": "write", "batch": 32, "new": 1, "past": 4096, "heads_kv": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "salt": 1},
        # Packed prompts of different lengths, head dimension 64, a page of 64.
        {"name": "write-prompts", "op": "write", "batch": 7, "new": 1111, "past": 0, "heads_kv": 8, "dim": 64,
         "page": 64, "dtype": "fp16", "salt": 2},
        # A full prefill batch: the largest write.
        {"name": "write-prefill", "op": "write", "batch": 16, "new": 8192, "past": 0, "heads_kv": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "salt": 3},
        # One sequence's tokens read back, odd length.
        {"name": "read-one", "op": "read", "batch": 1, "new": 777, "past": 0, "heads_kv": 8, "dim": 128,
         "page": 16, "dtype": "fp16", "salt": 4},
        # A batch's tokens read back to be handed to another step.
        {"name": "read-batch", "op": "read", "batch": 16, "new": 8192, "past": 100, "heads_kv": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "salt": 5},
        # One user, a short prompt: latency.
        {"name": "decode-one", "op": "decode", "batch": 1, "heads": 32, "heads_kv": 8, "queries": 1, "dim": 128,
         "keys": 512, "page": 16, "dtype": "fp16", "salt": 6},
        # A ragged batch of running sequences, one K/V head per query head, head dimension 64.
        {"name": "decode-mha", "op": "decode", "batch": 16, "heads": 16, "heads_kv": 16, "queries": 1, "dim": 64,
         "keys": 4097, "page": 64, "dtype": "fp16", "salt": 7},
        # A large ragged batch with grouped heads: the usual server step.
        {"name": "decode-batch", "op": "decode", "batch": 64, "heads": 32, "heads_kv": 8, "queries": 1, "dim": 128,
         "keys": 16384, "page": 16, "dtype": "bf16", "salt": 8},
        # Five drafted tokens per sequence are checked at once.
        {"name": "decode-draft", "op": "decode", "batch": 8, "heads": 32, "heads_kv": 8, "queries": 5, "dim": 128,
         "keys": 8192, "page": 32, "dtype": "bf16", "salt": 9},
        # One sequence of 128K tokens.
        {"name": "decode-long", "op": "decode", "batch": 1, "heads": 32, "heads_kv": 4, "queries": 1, "dim": 128,
         "keys": 131072, "page": 128, "dtype": "fp16", "salt": 10},
        # A few samples of one short prompt.
        {"name": "prefix-few", "op": "prefix", "batch": 4, "heads": 16, "heads_kv": 16, "queries": 1, "dim": 64,
         "keys": 129, "prefix": 1000, "page": 16, "dtype": "fp16", "salt": 11},
        # Many users behind one long system prompt.
        {"name": "prefix-many", "op": "prefix", "batch": 64, "heads": 32, "heads_kv": 8, "queries": 1, "dim": 128,
         "keys": 512, "prefix": 16384, "page": 16, "dtype": "bf16", "salt": 12},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "prefix"])
    case = {"op": op, "dim": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128, 256]),
            "dtype": rng.choice(["fp16", "bf16"]), "salt": rng.randrange(1 << 20)}
    if op in ("write", "read"):
        batch = _log(rng, 1, 64)
        return dict(case, batch=batch, new=_log(rng, 1, 131072 // batch // 2), past=rng.randrange(4096),
                    heads_kv=rng.choice([1, 2, 3, 4, 5, 8]))
    heads_kv = rng.choice([1, 2, 4, 5, 8])
    heads = heads_kv * rng.choice([1, 2, 3, 4, 8])
    batch, queries = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 3, 7])
    case = dict(case, batch=batch, heads=min(heads, 32) // heads_kv * heads_kv, heads_kv=heads_kv, queries=queries)
    if op == "decode":
        return dict(case, keys=max(queries, _log(rng, 16, 65536 // batch + 16)))
    return dict(case, keys=max(queries, _log(rng, 8, 1024)), prefix=_log(rng, 32, min(16384, (1 << 20) // (batch * queries))))


def _lens(case):
    """(tokens held, of them new or behind the prefix) of each sequence; goes by the case alone."""
    rng = random.Random(case["salt"])
    op = case["op"]
    if op in ("write", "read"):
        if case["new"] == 1:
            new = [1] * case["batch"]
        else:  # ragged; the longest as the case says
            new = [case["new"]] + [rng.randint(1, case["new"]) for _ in range(case["batch"] - 1)]
        return [n + (rng.randint(0, case["past"]) if case["past"] else 0) for n in new], new
    low = case["queries"]
    own_keys = [case["keys"]] + [rng.randint(low, case["keys"]) for _ in range(case["batch"] - 1)]
    rng.shuffle(own_keys)
    return [n + case.get("prefix", 0) for n in own_keys], own_keys


def _quantise(x):
    """Codes (e4m3) and exponent bytes of rows x (..., dim), by the rule at the head of this file."""
    x = x.float()
    amax = x.abs().amax(-1)
    fine = torch.isfinite(amax)
    part, power = torch.frexp(torch.where(fine, amax, torch.zeros_like(amax)))  # amax = part * 2^power
    e = power - 9 + (part > 0.875).int()
    e = torch.where(amax == 0, torch.zeros_like(e), e.clamp(min=-63))
    codes = torch.ldexp(x, -e.unsqueeze(-1))
    codes = torch.where(fine.unsqueeze(-1), codes, torch.zeros_like(codes)).to(E4M3)
    byte = torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)
    return codes, byte


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 1000003 + case["salt"])
    total, new = _lens(case)
    batch, heads_kv, dim, page = case["batch"], case["heads_kv"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    prefix = case.get("prefix", 0)
    shared = prefix // page  # whole pages that all sequences share
    need = [-(-n // page) - shared for n in total]
    pages = shared + sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=dev).int()
    width = shared + max(need)
    need_t = torch.tensor(need, device=dev)
    first = torch.cat([need_t.new_zeros(1), need_t.cumsum(0)[:-1]])
    col = torch.arange(width - shared, device=dev)
    at = shared + first[:, None] + col[None, :]
    table = torch.where(col[None, :] < need_t[:, None], order[at.clamp(max=pages - 1).long()].int(),
                        torch.full((), -1, dtype=torch.int32, device=dev))
    table = torch.cat([order[:shared].expand(batch, shared), table], 1).contiguous()
    if prefix % page:  # the page in which the prefix ends is each sequence's own: it holds the same tokens
        edge = table[:, shared].long()
    seqlens = torch.tensor(total, dtype=torch.int32, device=dev)

    def cache_part(spread):
        # Keys and values as a projection gives them: unit rows of the model, some channels
        # several times larger than the rest, tokens of different size.
        codes = torch.empty(pages, heads_kv, page, dim, dtype=E4M3, device=dev)
        byte = torch.empty(pages, heads_kv, page, dtype=torch.uint8, device=dev)
        channel = torch.exp(spread * torch.randn(heads_kv, 1, dim, generator=gen, device=dev))
        step = max(1, (1 << 25) // (heads_kv * page * dim))
        for p0 in range(0, pages, step):
            n = min(step, pages - p0)
            x = torch.randn(n, heads_kv, page, dim, generator=gen, device=dev) * channel
            x = x * torch.exp(0.3 * torch.randn(n, heads_kv, page, 1, generator=gen, device=dev))
            codes[p0:p0 + n], byte[p0:p0 + n] = _quantise(x)
        if prefix % page:
            codes.view(torch.uint8)[edge, :, :prefix % page] = codes.view(torch.uint8)[edge[:1], :, :prefix % page]
            byte[edge, :, :prefix % page] = byte[edge[:1], :, :prefix % page]
        return codes, byte

    state = {"case": case, "table": table, "seqlens": seqlens, "width": width}
    state["k"], state["k_exp"] = cache_part(0.4)
    state["v"], state["v_exp"] = cache_part(0.2)
    if case["op"] in ("write", "read"):
        state["cu"] = torch.tensor([0] + new, device=dev).cumsum(0).int()
        state["total"] = sum(new)
    if case["op"] == "write":
        shape = (sum(new), heads_kv, dim)
        for name in ("new_k", "new_v"):
            x = torch.randn(shape, generator=gen, device=dev)
            state[name] = (x * torch.exp(0.5 * torch.randn(shape[0], shape[1], 1, generator=gen, device=dev))).to(dtype)
    if case["op"] in ("decode", "prefix"):
        q = torch.randn(batch, case["heads"], case["queries"], dim, generator=gen, device=dev)
        state["q"] = (1.5 * q).to(dtype)
    return state


def _places(state):
    """Page and slot of every token of the packed order, and which of them are held."""
    case = state["case"]
    cu, n = state["cu"].long(), state["total"]
    row = torch.arange(n, device=cu.device)
    b = torch.searchsorted(cu, row, right=True) - 1
    pos = state["seqlens"].long()[b] - (cu[b + 1] - row)
    return state["table"].long()[b, pos // case["page"]], pos % case["page"]


def _write(state):
    page, slot = _places(state)
    for name in ("k", "v"):
        codes, byte = _quantise(state["new_" + name])
        state[name].view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)
        state[name + "_exp"][page, :, slot] = byte
    return state["k"], state["v"], state["k_exp"], state["v_exp"]


def _value(codes, byte):
    e = torch.where(byte == 255, torch.full((), math.nan, device=byte.device), torch.ldexp(
        torch.ones((), device=byte.device), byte.int() - 127))
    return codes.float() * e.unsqueeze(-1)


def _read(state):
    page, slot = _places(state)
    dtype = DTYPES[state["case"]["dtype"]]
    top = torch.finfo(dtype).max
    return tuple(_value(state[n].view(torch.uint8)[page, :, slot].view(E4M3), state[n + "_exp"][page, :, slot])
                 .clamp(-top, top).to(dtype) for n in ("k", "v"))


def _gather(state, name, table, first, last):
    """Tokens first..last-1 of each row of the table as fp32 (rows, kv heads, last - first, dim)."""
    page = state["case"]["page"]
    p0, p1 = first // page, -(-last // page)
    at = table[:, p0:p1].clamp(min=0).long()
    x = _value(state[name].view(torch.uint8)[at].view(E4M3), state[name + "_exp"][at])  # rows, pages, heads, slots, dim
    x = x.transpose(1, 2).flatten(2, 3)
    return x[:, :, first - p0 * page:last - p0 * page]


def _attend(state):
    """Attention over the cached tokens; the shared ones are gathered and multiplied once."""
    case, q = state["case"], state["q"]
    batch, heads, queries, dim = q.shape
    group, prefix = heads // case["heads_kv"], case.get("prefix", 0)
    longest = prefix + case["keys"]
    qs = q.float().reshape(batch, case["heads_kv"], group * queries, dim) * dim ** -0.5
    own_k = _gather(state, "k", state["table"], prefix, longest)
    s = torch.matmul(qs, own_k.transpose(2, 3))
    del own_k
    pos = state["seqlens"].view(-1, 1) - queries + torch.arange(queries, device=q.device)
    key = torch.arange(prefix, longest, device=q.device)
    seen = (key <= pos.unsqueeze(2)).repeat(1, group, 1).unsqueeze(1)  # batch, 1, group * queries, keys
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    if prefix:
        shared_k = _gather(state, "k", state["table"][:1], 0, prefix)[0]  # kv heads, prefix, dim
        qp = qs.transpose(0, 1).flatten(1, 2)
        sp = torch.matmul(qp, shared_k.transpose(1, 2)).view(case["heads_kv"], batch, group * queries, prefix)
        top = torch.maximum(top, sp.amax(-1, keepdim=True).transpose(0, 1))
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    own_v = _gather(state, "v", state["table"], prefix, longest)
    # A slot behind a sequence's end holds whatever was there: no product may see it.
    own_v = torch.where((key < state["seqlens"].view(-1, 1)).view(batch, 1, -1, 1), own_v, torch.zeros_like(own_v))
    o = torch.matmul(p, own_v)
    del own_v, s, p
    if prefix:
        pp = torch.exp(sp - top.transpose(0, 1))
        total = total + pp.sum(-1, keepdim=True).transpose(0, 1)
        shared_v = _gather(state, "v", state["table"][:1], 0, prefix)[0]
        o = o + torch.matmul(pp.flatten(1, 2), shared_v).view(case["heads_kv"], batch, -1, dim).transpose(0, 1)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = torch.where(total > 0, top + torch.log(total), torch.full_like(top, -math.inf))
    return o.reshape(q.shape).to(q.dtype), lse.reshape(batch, heads, queries)


def run(state):
    op = state["case"]["op"]
    if own:
        import ada_cute_fp8_flash_attention_b200 as fa8

        cache = fa8.KVCacheFP8(state["k"], state["v"], state["k_exp"], state["v_exp"])
        table, seqlens = state["table"], state["seqlens"]
        if op == "write":
            fa8.kv_cache_write(cache, state["new_k"], state["new_v"], table, seqlens, cu_seqlens=state["cu"])
            return cache.k, cache.v, cache.k_exp, cache.v_exp
        if op == "read":
            return fa8.kv_cache_read(cache, table, seqlens, state["cu"], state["total"],
                                     dtype=state["case"]["dtype"])
        if op == "decode":
            return fa8.flash_attn_fp8_decode(state["q"], cache, table, seqlens, return_lse=True)
        return fa8.flash_attn_fp8_shared_prefix(state["q"], cache, table, seqlens, state["case"]["prefix"],
                                                return_lse=True)
    return {"write": _write, "read": _read, "decode": _attend, "prefix": _attend}[op](state)


def work(case):
    total, new = _lens(case)
    dim, heads_kv = case["dim"], case["heads_kv"]
    row = heads_kv * (dim + 1)  # codes and exponents of a token's K, or V
    if case["op"] in ("write", "read"):
        n = sum(new)
        return {"bytes": 2 * n * (row + heads_kv * dim * 2), "flops": 0}
    rows = case["batch"] * case["heads"] * case["queries"]
    cached = case.get("prefix", 0) + sum(new) if case["op"] == "prefix" else sum(total)
    pairs = case["heads"] * case["queries"] * sum(total)
    return {"bytes": 2 * cached * row + rows * (2 * dim * 2 + 4), "flops": 4 * dim * pairs}


def _round_e4m3(x):
    """The e4m3 value nearest to x (64 bits, |x| <= 448), ties to the even one."""
    power = torch.frexp(x)[1] - 1  # 2^power <= |x| < 2^(power + 1)
    step = torch.ldexp(torch.ones_like(x), power.clamp(min=-6) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    state = prepare(case, seed)
    total, new = _lens(case)
    page, dev = case["page"], state["table"].device
    table = state["table"].long()

    def tokens(name, b, first, last):
        """Values (last - first, kv heads, dim) of sequence b's tokens first..last-1, and where they are."""
        pos = torch.arange(first, last, device=dev)
        p, s = table[b, pos // page], pos % page
        codes = state[name].view(torch.uint8)[p, :, s].view(E4M3).double()
        return codes * torch.exp2(state[name + "_exp"][p, :, s].double() - 127).unsqueeze(-1), p, s

    if case["op"] == "write":
        out = []
        for name in ("k", "v"):
            codes = state[name].double()
            for b in range(case["batch"]):
                first = sum(new[:b])
                x = state["new_" + name][first:first + new[b]].double()
                amax = x.abs().amax(-1)
                e = torch.ceil(torch.log2(amax / 448) - 1e-9)  # 16-bit inputs: no ratio lies this near above a power of two
                e = torch.where(amax == 0, torch.zeros_like(e), e.clamp(min=-63))
                pos = torch.arange(total[b] - new[b], total[b], device=dev)
                codes[table[b, pos // page], :, pos % page] = _round_e4m3(x * torch.exp2(-e).unsqueeze(-1))
            out.append(codes)
        return out[0], out[1], None, None
    if case["op"] == "read":
        return tuple(torch.cat([tokens(n, b, total[b] - new[b], total[b])[0] for b in range(case["batch"])])
                     for n in ("k", "v"))
    heads, queries, dim = case["heads"], case["queries"], case["dim"]
    if 4 * dim * heads * queries * sum(total) > 4e12:
        return None
    out = torch.empty(state["q"].shape, dtype=torch.float64, device=dev)
    lse = torch.empty(state["q"].shape[:3], dtype=torch.float64, device=dev)
    group = heads // case["heads_kv"]
    for b in range(case["batch"]):
        k, v = tokens("k", b, 0, total[b])[0], tokens("v", b, 0, total[b])[0]
        for i in range(queries):
            n = total[b] - queries + i + 1  # keys that this query sees
            q = state["q"][b, :, i].double().view(case["heads_kv"], group, dim)
            s = torch.einsum("hgd,nhd->hgn", q, k[:n]) / math.sqrt(dim)
            out[b, :, i] = torch.einsum("hgn,nhd->hgd", torch.softmax(s, -1), v[:n]).reshape(heads, dim)
            lse[b, :, i] = torch.logsumexp(s, -1).reshape(heads)
    return out, lse
