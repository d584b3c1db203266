"""GPU parity of the paged e4m3 cache (write, read) and of the attention over it
(decode, shared prefix) against the 64-bit oracle.

Tolerances. Codes and exponents are whole numbers: equal. A value read back is
rounded once: equal. Attention, with u = eps / 2 of q's type (2^-11 fp16, 2^-8
bf16), A = sum p|v| / sum p, B = the largest sum_d |q_d k_d| * scale of a key and
w = sum p / max p:
* the result is rounded once: u |o|;
* each p is rounded once to u (fp16: 11 bits, bf16: 8 bits): u A;
* scores are sums of D products in fp32, whose additions may each lose 2^-22 of
  the largest partial sum (truncating accumulation): ds = D 2^-22 B, which moves
  every p by ds and the quotient by 2 ds A; exp2 and the sum of p in fp32 add
  2^-20 A;
* small p meet a floor: the least step of e4m3 is 2^-9, half of it 2^-10; the last
  of 2 (bf16) or 3 (fp16) terms weighs 16^-1 or 16^-2, and 1 stands for 8: 2^-17 or
  2^-21 of the largest p * 2^e of the row, times n keys of magnitude vmax or less,
  over w.
lse: ds + 2^-20 (1 + |lse|).
"""
import math
import random

import pytest

from oracle import kv_cache_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def fa8(cuda):
    import ada_cute_fp8_flash_attention_b200 as m
    return m


def make_cache(fa8, pages, heads_kv, page_size, D, layout="phsd", seed=0, spread=1.0):
    """A cache of quantised normal rows; every code and byte defined."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def part():
        x = torch.randn(pages, heads_kv, page_size, D, generator=g, device="cuda")
        x = x * torch.exp(spread * torch.randn(pages, heads_kv, page_size, 1, generator=g,
                                               device="cuda"))
        values, byte = ref.quantise(x)
        codes = values.float().to(E4M3)
        if layout == "pshd":
            codes = codes.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(E4M3)
        return codes, byte
    (k, ke), (v, ve) = part(), part()
    return fa8.KVCacheFP8(k, v, ke, ve)


def u8(t):
    return t.view(torch.uint8)


def make_table(lens, page_size, pages, seed=0, width=None, fill=-1):
    """Distinct random pages for every sequence; unused entries hold `fill`."""
    rng = random.Random(seed)
    free = list(range(pages))
    rng.shuffle(free)
    need = [-(-n // page_size) for n in lens]
    width = width or max(need + [1])
    rows = [[free.pop() for _ in range(n)] + [fill] * (width - n) for n in need]
    return (torch.tensor(rows, dtype=torch.int32, device="cuda"),
            torch.tensor(lens, dtype=torch.int32, device="cuda"))


def pages_for(lens, page_size):
    return sum(-(-n // page_size) for n in lens) + 2


def clone(cache):
    # .clone() keeps the strides of a dense tensor, whatever its order
    return type(cache)(*(u8(t).clone().view(t.dtype) for t in cache))


def check_written(fa8, cache, before, k, v, table, lens, new):
    """Every slot holds the oracle's row of its token, all others what they held."""
    want = clone(before)
    ps = cache.k.shape[2]
    for name, rows in (("k", k), ("v", v)):
        codes, exps = u8(getattr(want, name)), getattr(want, name + "_exp")
        for b, n in enumerate(new):
            x = rows[b]  # (H_kv, n, D)
            values, byte = ref.quantise(x)
            pos = torch.arange(lens[b] - n, lens[b], device="cuda")
            page, slot = table[b].long()[pos // ps], pos % ps
            codes[page, :, slot] = u8(values.float().to(E4M3)).transpose(0, 1)
            exps[page, :, slot] = byte.transpose(0, 1)
    for name in ("k", "v"):
        got, exp = u8(getattr(cache, name)), u8(getattr(want, name))
        # -0 and 0 are one value: compare the codes' values
        assert torch.equal(torch.where(got == 128, 0, got), torch.where(exp == 128, 0, exp)), name
        assert torch.equal(getattr(cache, name + "_exp"), getattr(want, name + "_exp")), name


@pytest.mark.parametrize("layout", ["phsd", "pshd"])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,heads_kv,page_size", [(128, 8, 16), (64, 3, 64), (128, 1, 256),
                                                  (64, 5, 32), (128, 2, 128)])
def test_write_packed(fa8, D, heads_kv, page_size, dtype, layout):
    new = [1, 37, 0, 130, 64]
    lens = [1, 40, 19, 130, 300]
    pages = pages_for(lens, page_size)
    cache = make_cache(fa8, pages, heads_kv, page_size, D, layout)
    before = clone(cache)
    table, seqlens = make_table(lens, page_size, pages)
    lead, tail = 3, 5  # rows before the first and behind the last sequence
    total = lead + sum(new) + tail
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(total, heads_kv, D, generator=g, device="cuda").mul(5).to(DTYPES[dtype])
    v = torch.randn(total, heads_kv, D, generator=g, device="cuda").mul(0.02).to(DTYPES[dtype])
    cu = torch.tensor([lead] + new, device="cuda").cumsum(0).int()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    fa8.kv_cache_write(cache, k, v, table, seqlens, cu_seqlens=cu, status=status)
    assert int(status) == 0
    split = lambda x: [x[a:b].transpose(0, 1) for a, b in zip(cu.tolist(), cu.tolist()[1:])]  # noqa: E731
    check_written(fa8, cache, before, split(k), split(v), table, lens, new)


@pytest.mark.parametrize("case", ["contiguous", "fused", "shifted", "broadcast"])
def test_write_dense_strides(fa8, case):
    B, Hkv, n, D, ps = 3, 4, 7, 128, 16
    lens = [7, 100, 33]
    pages = pages_for(lens, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D)
    before = clone(cache)
    table, seqlens = make_table(lens, ps, pages)
    if case == "contiguous":
        k, v = torch.randn(2, B, Hkv, n, D, device="cuda").half()
    elif case == "fused":  # views into one projection, tokens before heads
        qkv = torch.randn(B, n, 3 * Hkv * D, device="cuda").half()
        k, v = (t.view(B, n, Hkv, D).transpose(1, 2) for t in qkv.split(Hkv * D, 2)[1:])
    elif case == "shifted":  # an odd start: not 16-byte aligned
        k, v = (torch.randn(B * Hkv * n * D + 3, device="cuda").half()[3:].view(B, Hkv, n, D)
                for _ in range(2))
    else:
        k, v = (torch.randn(B, 1, n, D, device="cuda").half().expand(B, Hkv, n, D)
                for _ in range(2))
    fa8.kv_cache_write(cache, k, v, table, seqlens)
    check_written(fa8, cache, before, k, v, table, lens, [n] * B)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_write_and_read_special_rows(fa8, dtype):
    dt = DTYPES[dtype]
    D, ps = 64, 16
    info = torch.finfo(dt)
    rows = torch.zeros(14, D, dtype=torch.float64)
    rows[1] = info.max
    rows[2, 5] = -info.max
    rows[3, 0], rows[3, 1] = math.inf, 1
    rows[4, 0], rows[4, 1] = math.nan, 1
    rows[5, 7], rows[5, 8] = info.smallest_normal, -info.smallest_normal
    rows[6, 0] = info.smallest_normal * info.eps  # the least subnormal
    rows[7, :3] = torch.tensor([448.0, 1.0, -2.0 ** -9])
    rows[8, :3] = torch.tensor([448.0 * (1 + info.eps), 1.0, 2.0 ** -9])
    rows[9, :3] = torch.tensor([1.75, 0.0595703125, -1.0625])  # ties of e4m3
    rows[10] = torch.linspace(-448, 448, D)
    rows[11] = torch.exp2(torch.arange(D).double().clamp(max=30) - 20)
    rows[12, 0] = -0.0
    rows[13] = -math.inf
    x = rows.to(dt).cuda().view(1, 1, -1, D)
    n = x.shape[2]
    cache = make_cache(fa8, 2, 1, ps, D)
    before = clone(cache)
    table, seqlens = make_table([n], ps, 2)
    fa8.kv_cache_write(cache, x, -x, table, seqlens)
    check_written(fa8, cache, before, x, -x, table, [n], [n])
    for back in ("fp16", "bf16"):
        k, v = fa8.kv_cache_read(cache, table, seqlens, None, n, dtype=back)
        for got, name in ((k, "k"), (v, "v")):
            want = ref.to_16bit(ref.tokens(u8(getattr(cache, name)), getattr(cache, name + "_exp"),
                                           table[0], 0, n), DTYPES[back])
            assert torch.equal(got[0].isnan(), want.isnan())
            assert torch.equal(got[0].nan_to_num(7.0), want.nan_to_num(7.0))
            assert bool(got[0, 0, 3].isnan().all()) and bool(got[0, 0, 4].isnan().all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,heads_kv,page_size,layout", [(128, 8, 16, "phsd"), (64, 3, 64, "pshd"),
                                                         (128, 1, 128, "pshd"), (64, 2, 32, "phsd")])
def test_read_packed(fa8, D, heads_kv, page_size, layout, dtype):
    lens, take = [5, 0, 200, 64, 131], [5, 0, 77, 1, 131]
    pages = pages_for(lens, page_size)
    cache = make_cache(fa8, pages, heads_kv, page_size, D, layout, spread=3.0)
    table, seqlens = make_table(lens, page_size, pages)
    cu = torch.tensor([0] + take, device="cuda").cumsum(0).int()
    total = sum(take) + 9
    out = tuple(torch.full((total, heads_kv, D), 3.0, dtype=DTYPES[dtype], device="cuda")
                for _ in range(2))
    got = fa8.kv_cache_read(cache, table, seqlens, cu, total, dtype=dtype, out=out)
    assert got[0].data_ptr() == out[0].data_ptr()
    for t, name in zip(got, ("k", "v")):
        want = [ref.tokens(u8(getattr(cache, name)), getattr(cache, name + "_exp"), table[b],
                           lens[b] - take[b], lens[b]).transpose(0, 1) for b in range(len(lens))]
        assert torch.equal(t[:sum(take)], ref.to_16bit(torch.cat(want), DTYPES[dtype]))
        assert bool((t[sum(take):] == 3.0).all())  # behind the last sequence: as it was
    fresh = fa8.kv_cache_read(cache, table, seqlens, cu, sum(take), dtype=dtype)
    assert torch.equal(fresh[0], got[0][:sum(take)]) and torch.equal(fresh[1], got[1][:sum(take)])


def test_copy_status_bits(fa8):
    """Bad lengths and pages are flagged, the other sequences served."""
    D, Hkv, ps = 64, 2, 16
    lens = [20, 70, 2, 33]  # table rows hold 64; 70 does not fit, 2 < 3 new tokens
    cache = make_cache(fa8, 12, Hkv, ps, D)
    before = clone(cache)
    table = torch.arange(16, dtype=torch.int32, device="cuda").view(4, 4) % 12
    table[3, 2] = 12  # token 32 of the last sequence: no such page
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.randn(4, Hkv, 3, D, device="cuda").half()
    fa8.kv_cache_write(cache, x, x, table, seqlens, status=status)
    assert int(status) == 4 | 8
    table2 = table.clone()
    table2[3, 2] = 0
    want = clone(before)
    for name in ("k", "v"):
        for b, toks in ((0, [17, 18, 19]), (3, [30, 31])):
            for i, t in zip(range(3), toks):
                values, byte = ref.quantise(x[b, :, i])
                page = int(table2[b, t // ps])
                u8(getattr(want, name))[page, :, t % ps] = u8(values.float().to(E4M3))
                getattr(want, name + "_exp")[page, :, t % ps] = byte
        got, exp = u8(getattr(cache, name)), u8(getattr(want, name))
        assert torch.equal(torch.where(got == 128, 0, got), torch.where(exp == 128, 0, exp))
        assert torch.equal(getattr(cache, name + "_exp"), getattr(want, name + "_exp"))
    status.zero_()
    out = tuple(torch.full((4, Hkv, 3, D), 9.0, dtype=torch.float16, device="cuda")
                for _ in range(2))
    table[3, 2] = -7
    k, v = fa8.kv_cache_read(cache, table, seqlens, None, 3, out=out, status=status)
    assert int(status) == 4 | 8
    assert bool((k[1:3] == 9).all()) and bool((v[1:3] == 9).all())
    assert bool(k[3, :, 2].isnan().all()) and not bool(k[3, :, :2].isnan().any())


def test_copy_first_offset_far_below_zero(fa8):
    """cu[1] - cu[0] does not fit 32 bits: refused, nothing is written on either side."""
    cache = make_cache(fa8, 4, 2, 16, 64)
    before = clone(cache)
    table = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4)
    seqlens = torch.tensor([2], dtype=torch.int32, device="cuda")
    cu = torch.tensor([-2**31, 10], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = torch.randn(10, 2, 64, device="cuda").half()
    fa8.kv_cache_write(cache, x, x, table, seqlens, cu, status=status)
    assert int(status) == 4
    assert all(torch.equal(u8(t), u8(o)) for t, o in zip(cache, before))
    status.zero_()
    out = tuple(torch.full((10, 2, 64), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    k, v = fa8.kv_cache_read(cache, table, seqlens, cu, 10, out=out, status=status)
    assert int(status) == 4 and bool((k == 9).all()) and bool((v == 9).all())


# ------------------------------------------------------------------ attention

def oracle_attention(q, cache, table, lens, scale=None, prefix=0):
    """Per sequence from the oracle: out, lse and the tolerances of both."""
    B, H, Sq, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    outs, lses, tols, ltols = [], [], [], []
    for b in range(B):
        row = table[b].clone()
        if prefix:
            ps = cache.k.shape[2]
            assert bool((row[:prefix // ps] == table[0][:prefix // ps]).all())
        k = ref.tokens(u8(cache.k), cache.k_exp, row, 0, lens[b])
        v = ref.tokens(u8(cache.v), cache.v_exp, row, 0, lens[b])
        out, lse, A, w, big = ref.attention(q[b].double(), k, v, scale)
        ds = (D * 2.0 ** -22 * big).unsqueeze(-1)
        vmax = float(v.abs().nan_to_num(0).max()) if lens[b] else 0.0
        least = 2.0 ** (-21 if q.dtype == torch.float16 else -17)
        floor = (lens[b] * least * vmax / w.clamp(min=1)).unsqueeze(-1)
        tols.append(u * out.abs() + (u + 2 * ds + 2.0 ** -20) * A + floor)
        ltols.append(ds.squeeze(-1) + 2.0 ** -20 * (1 + lse.abs()))
        outs.append(out)
        lses.append(lse)
    return tuple(torch.stack(t) for t in (outs, lses, tols, ltols))


def assert_attention(got, q, cache, table, lens, scale=None, prefix=0):
    out, lse = got
    want, wlse, tol, ltol = oracle_attention(q, cache, table, lens, scale, prefix)
    assert out.dtype == q.dtype and out.shape == q.shape
    assert torch.equal(out.isnan(), want.isnan())
    fine = ~want.isnan()
    over = ((out.double() - want).abs() - tol)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"out: over by {float(over.max()):.3g}"
    none = wlse == -math.inf
    assert torch.equal(lse == -math.inf, none)
    assert bool((out[none] == 0).all())
    fine = ~none & ~wlse.isnan()
    assert torch.equal(lse.isnan(), wlse.isnan())
    over = ((lse.double() - wlse).abs() - ltol)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, f"lse: over by {float(over.max()):.3g}"


def make_q(B, H, Sq, D, dtype, seed=5, size=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (size * torch.randn(B, H, Sq, D, generator=g, device="cuda")).to(DTYPES[dtype])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv,Sq", [(8, 8, 1), (8, 1, 1), (32, 4, 1), (6, 2, 1), (4, 2, 5),
                                      (48, 1, 1), (16, 2, 3), (128, 1, 1), (1, 1, 2), (8, 2, 33)])
def test_decode(fa8, H, Hkv, Sq, D, dtype):
    lens = [1, 128, 0, 300, 129, 17, 1025]
    ps = 32
    pages = pages_for(lens, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.5)
    table, seqlens = make_table(lens, ps, pages)
    q = make_q(len(lens), H, Sq, D, dtype)
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_attention(got, q, cache, table, lens)
    again = fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
    assert torch.equal(again, got[0])  # bit-identical, with and without lse


@pytest.mark.parametrize("layout", ["phsd", "pshd"])
@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256, 384])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_pages(fa8, ps, D, layout):
    lens = [ps, ps + 1, 3 * ps - 1, 700]
    pages = pages_for(lens, ps)
    cache = make_cache(fa8, pages, 3, ps, D, layout, spread=0.5)
    table, seqlens = make_table(lens, ps, pages, width=4 + 700 // ps)
    q = make_q(4, 6, 2, D, "fp16")
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_attention(got, q, cache, table, lens)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,Hkv", [([40000], 2), ([8191, 1, 4096, 20000, 7], 4),
                                      ([600] * 150, 2)])
def test_decode_long_and_many(fa8, lens, Hkv, D):
    """Ranges that are split over many blocks and joined, and more work than blocks."""
    ps = 64
    pages = pages_for(lens, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    table, seqlens = make_table(lens, ps, pages)
    q = make_q(len(lens), 4 * Hkv, 1, D, "fp16", size=0.7)
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_attention(got, q, cache, table, lens)


def test_decode_many_sequences(fa8):
    """A thousand short sequences, empty ones among them; pages used twice."""
    rng = random.Random(4)
    lens = [rng.choice([0, 1, 5, 16, 17, 40]) for _ in range(1000)]
    cache = make_cache(fa8, 64, 1, 16, 64)
    table = torch.randint(0, 64, (1000, 3), dtype=torch.int32, device="cuda")
    table[::7, 1] = table[::7, 0]  # the same page at two places of a sequence
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = make_q(1000, 2, 1, 64, "bf16")
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_attention(got, q, cache, table, lens)


@pytest.mark.parametrize("D,H,Sq", [(128, 2, 1), (64, 8, 3), (128, 32, 1), (128, 64, 2)])
def test_decode_wait_that_runs_out(fa8, D, H, Sq):
    """A limit of one clock: the kernel reports it, ends, and the next call is right."""
    from ada_cute_fp8_flash_attention_b200 import c_abi
    lens = [3000, 900]
    cache = make_cache(fa8, pages_for(lens, 64), 1, 64, D)
    table, seqlens = make_table(lens, 64, pages_for(lens, 64))
    q = make_q(2, H, Sq, D, "fp16")
    want = fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = c_abi.decode_params(cache.k.shape[0], 1, 64, D, 2, table.shape[1], H, Sq)
    c = p.cache
    c.k, c.v = cache.k.data_ptr(), cache.v.data_ptr()
    c.k_exp, c.v_exp = cache.k_exp.data_ptr(), cache.v_exp.data_ptr()
    c.page_table, c.seqlens, c.status = table.data_ptr(), seqlens.data_ptr(), status.data_ptr()
    out = torch.zeros_like(q)
    p.q, p.o = q.data_ptr(), out.data_ptr()
    size = c_abi.decode_workspace_size(p)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert c_abi.decode(p, ws.data_ptr(), size - 1, stream) == c_abi.FA8_ERR_INVALID_ARG
    assert c_abi.decode(p, ws.data_ptr() + 16, size, stream) == c_abi.FA8_ERR_INVALID_ARG
    p.wait_timeout_cycles = 1
    c_abi.check(c_abi.decode(p, ws.data_ptr(), size, stream))
    torch.cuda.synchronize()
    assert int(status) == 1
    status.zero_()
    p.wait_timeout_cycles = 0
    c_abi.check(c_abi.decode(p, ws.data_ptr(), size, stream))
    torch.cuda.synchronize()
    assert int(status) == 0 and torch.equal(out, want)


def test_prefix_wait_that_runs_out(fa8):
    """Blocks that give up have not said where all their items are: whatever the
    workspace holds there, the joining kernel stays inside it."""
    from ada_cute_fp8_flash_attention_b200 import c_abi
    B, H, D, ps, prefix = 64, 16, 64, 64, 1000
    lens = [prefix + 1 + (11 * b) % 140 for b in range(B)]
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, H, ps, D, spread=0.3)
    same_prefix(cache, table, lens, prefix)
    q = make_q(B, H, 1, D, "fp16")
    want = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = c_abi.decode_params(pages, H, ps, D, B, table.shape[1], H, 1)
    c = p.cache
    c.k, c.v = cache.k.data_ptr(), cache.v.data_ptr()
    c.k_exp, c.v_exp = cache.k_exp.data_ptr(), cache.v_exp.data_ptr()
    c.page_table, c.seqlens, c.status = table.data_ptr(), seqlens.data_ptr(), status.data_ptr()
    out = torch.zeros_like(q)
    p.q, p.o, p.prefix_len = q.data_ptr(), out.data_ptr(), prefix
    size = c_abi.decode_workspace_size(p)
    assert size % 16 == 0
    ws = torch.empty(size // 4, dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for places in ((2**31 - 1, 2**31 - 1, 2**31 - 1), (0, 2**31 - 1, 0), (-5, 3, -9), (7, 2, 0)):
        ws.view(-1, 4)[:] = torch.tensor(places + (2,), dtype=torch.int32, device="cuda")
        status.zero_()
        p.wait_timeout_cycles = 1
        c_abi.check(c_abi.decode(p, ws.data_ptr(), size, stream))
        torch.cuda.synchronize()
        assert int(status) == 1
        status.zero_()
        p.wait_timeout_cycles = 0
        c_abi.check(c_abi.decode(p, ws.data_ptr(), size, stream))
        torch.cuda.synchronize()
        assert int(status) == 0 and torch.equal(out, want)


def test_decode_many_rows_without_keys(fa8):
    """More 16-byte pieces of results than 31 bits count, all of them zeros."""
    H, Sq = 2056, 65535
    cache = make_cache(fa8, 1, 8, 16, 128)
    table, seqlens = make_table([0], 16, 1, width=1)
    q = make_q(1, 1, 1, 128, "fp16").expand(1, H, Sq, 128)
    out = torch.full((1, H, Sq, 128), 3.0, dtype=torch.float16, device="cuda")
    fa8.flash_attn_fp8_decode(q, cache, table, seqlens, out=out)
    bits = out.view(torch.int32)
    assert int(bits.amax()) == 0 and int(bits.amin()) == 0


def test_decode_long_query(fa8):
    """A chunk of a prompt: more query rows than one block holds."""
    lens = [700, 150, 260]
    cache = make_cache(fa8, pages_for(lens, 16), 2, 16, 128, spread=0.5)
    table, seqlens = make_table(lens, 16, pages_for(lens, 16))
    q = make_q(3, 8, 201, 128, "bf16")  # the second sequence's first 51 queries see nothing
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_attention(got, q, cache, table, lens)


@pytest.mark.parametrize("case", ["bshd", "shifted", "sliced"])
def test_decode_strides(fa8, case):
    lens, B, H, Sq, D = [50, 200], 2, 8, 3, 128
    cache = make_cache(fa8, 20, 4, 16, D)
    table, seqlens = make_table(lens, 16, 20)
    base = make_q(B, H, Sq, D, "fp16")
    if case == "bshd":
        q = base.transpose(1, 2).contiguous().transpose(1, 2)
    elif case == "shifted":
        q = torch.empty(base.numel() + 1, dtype=base.dtype, device="cuda")[1:].view(base.shape)
        q.copy_(base)
    else:
        q = torch.empty(B, H, Sq, 2 * D, dtype=base.dtype, device="cuda")[..., D:]
        q.copy_(base)
    wide = torch.full((4, 6), -1, dtype=torch.int64)  # int64 on the host, a wider table
    wide[:2, :table.shape[1]] = table.cpu()[:, :6]
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens.long(), return_lse=True)
    assert_attention(got, base, cache, table, lens)
    out = torch.empty(B, Sq, H, D, dtype=torch.float16, device="cuda").transpose(1, 2)
    fa8.flash_attn_fp8_decode(q, cache, table, seqlens, out=out)
    assert torch.equal(out, got[0])


def test_decode_scale_and_extremes(fa8):
    """Scores that differ by thousands, tiny and large rows, an explicit scale."""
    lens = [400, 400, 400]
    cache = make_cache(fa8, pages_for(lens, 16), 2, 16, 128, spread=3.0)
    table, seqlens = make_table(lens, 16, pages_for(lens, 16))
    q = make_q(3, 8, 1, 128, "fp16")
    q[1] *= 100
    q[2] *= 1e-6
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, softmax_scale=0.3, return_lse=True)
    assert_attention(got, q, cache, table, lens, scale=0.3)
    # A growing ramp of scores: the running maximum moves in every block of keys.
    k = torch.zeros(1, 2, 1000, 128, device="cuda")
    k[..., 0] = torch.arange(1000, device="cuda") * 0.1
    cache = make_cache(fa8, 63, 2, 16, 128)
    table, seqlens = make_table([1000], 16, 63)
    fa8.kv_cache_write(cache, k.half(), torch.randn_like(k).half(), table, seqlens)
    for sign in (1.0, -1.0):
        q = torch.zeros(1, 4, 1, 128, dtype=torch.float16, device="cuda")
        q[..., 0] = sign * torch.tensor([0.0, 0.5, 5.0, 50.0], device="cuda").view(1, 4, 1)
        got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, softmax_scale=1.0,
                                        return_lse=True)
        assert_attention(got, q, cache, table, [1000], scale=1.0)


def test_decode_ignores_what_no_query_sees(fa8):
    """NaN codes, NaN exponents and infinite ones behind a sequence's end change nothing."""
    lens = [1, 130, 77, 256]
    for D in (64, 128):
        cache = make_cache(fa8, pages_for(lens, 64), 2, 64, D)
        table, seqlens = make_table(lens, 64, pages_for(lens, 64))
        q = make_q(4, 4, 1, D, "fp16")
        want = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
        for code, byte in ((0x7f, 255), (0xff, 254), (0x7e, 255)):
            dirty = fa8.KVCacheFP8(*(torch.full_like(u8(t), code).view(E4M3) if t.dtype == E4M3
                                     else torch.full_like(t, byte) for t in cache))
            for b, n in enumerate(lens):
                pos = torch.arange(n, device="cuda")
                page, slot = table[b].long()[pos // 64], pos % 64
                for a, c in zip(dirty, cache):
                    u8(a)[page, :, slot] = u8(c)[page, :, slot]
            got = fa8.flash_attn_fp8_decode(q, dirty, table, seqlens, return_lse=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("where", ["k", "v"])
def test_decode_nan_row_reaches_its_queries_only(fa8, where):
    """A token that was NaN makes the queries that see it NaN, not the ones before it."""
    lens, Sq = [140, 140], 4
    cache = make_cache(fa8, pages_for(lens, 16), 2, 16, 128)
    table, seqlens = make_table(lens, 16, pages_for(lens, 16))
    x = torch.randn(2, 2, 2, 128, device="cuda").half()
    bad = x.clone()
    bad[0, 1, 0, 3] = math.nan  # position 138 of sequence 0, K/V head 1
    fa8.kv_cache_write(cache, bad if where == "k" else x, bad if where == "v" else x, table, seqlens)
    q = make_q(2, 4, Sq, 128, "fp16")
    out, lse = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_attention((out, lse), q, cache, table, lens)
    assert bool(out[0, 2:, 2:].isnan().all()) and not bool(out[0, :2].isnan().any())
    assert not bool(out[0, :, :2].isnan().any()) and not bool(out[1].isnan().any())


def test_decode_nan_query(fa8):
    cache = make_cache(fa8, 10, 2, 16, 64)
    table, seqlens = make_table([100, 30], 16, 10)
    q = make_q(2, 4, 1, 64, "fp16")
    clean = fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
    q[0, 1, 0, 5] = math.nan
    q[1, 3, 0, 0] = math.inf
    out = fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
    assert bool(out[0, 1].isnan().all()) and bool(out[1, 3].isnan().all())
    keep = torch.ones(2, 4, dtype=torch.bool, device="cuda")
    keep[0, 1] = keep[1, 3] = False
    assert torch.equal(out[keep], clean[keep])


def test_decode_status_bits(fa8):
    lens = [100, 300, 64, -3, 90]  # a row holds 256: 300 does not fit
    cache = make_cache(fa8, 40, 2, 64, 64)
    table = torch.arange(20, dtype=torch.int32, device="cuda").view(5, 4)
    table[4, 1] = 40
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = make_q(5, 4, 1, 64, "bf16")
    out = torch.full_like(q, 5.0)
    fa8.flash_attn_fp8_decode(q, cache, table, seqlens, out=out, status=status)
    assert int(status) == 4 | 8
    assert bool((out[1] == 5).all()) and bool((out[3] == 5).all())
    assert bool(out[4].isnan().all())
    good = [0, 2]
    want = fa8.flash_attn_fp8_decode(q[good], cache, table[good], seqlens[good])
    tol = torch.finfo(q.dtype).eps * want.abs() + 2 * torch.finfo(q.dtype).eps
    assert bool(((out[good] - want).abs() <= tol).all())  # other shares of the work: other sums


def shared_table(lens, prefix, ps, seed=0):
    """Whole prefix pages shared; the page it ends in is each sequence's own."""
    shared = prefix // ps
    own = [max(0, n - shared * ps) for n in lens]
    pages = shared + pages_for(own, ps) + len(lens)
    table, _ = make_table(own, ps, pages - shared, seed)
    table = torch.where(table >= 0, table + shared, table)
    head = torch.arange(shared, dtype=torch.int32, device="cuda").expand(len(lens), shared)
    seqlens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    return torch.cat([head, table], 1).contiguous(), seqlens, pages


def same_prefix(cache, table, lens, prefix):
    """Copies row 0's tokens of the page the prefix ends in to the other rows' pages."""
    ps = cache.k.shape[2]
    n = prefix % ps
    if n:
        col = prefix // ps
        for b in range(1, len(lens)):
            if lens[b] > col * ps:
                for t in cache:
                    u8(t)[int(table[b, col]), :, :n] = u8(t)[int(table[0, col]), :, :n]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("D,H,Hkv,Sq,prefix,ps", [
    (128, 8, 2, 1, 256, 16), (64, 4, 4, 1, 1000, 64), (128, 32, 8, 1, 129, 128),
    (64, 6, 2, 3, 1, 32), (128, 4, 1, 1, 5000, 64), (128, 16, 1, 2, 47, 16)])
def test_shared_prefix(fa8, D, H, Hkv, Sq, prefix, ps, dtype):
    own = [1, 40, 130, 5, 300, 17, 64, 9, 3, 77, 11]
    lens = [prefix + max(n, Sq) for n in own]
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.5)
    same_prefix(cache, table, lens, prefix)
    q = make_q(len(lens), H, Sq, D, dtype)
    got = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, return_lse=True)
    assert_attention(got, q, cache, table, lens, prefix=prefix)
    again = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix)
    assert torch.equal(again, got[0])


def test_shared_prefix_many_rows(fa8):
    """More query rows than one block holds, and a prefix split over blocks."""
    prefix, ps, B = 3000, 64, 40
    lens = [prefix + 1 + (7 * b) % 90 for b in range(B)]
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, 2, ps, 128, spread=0.3)
    same_prefix(cache, table, lens, prefix)
    q = make_q(B, 16, 1, 128, "fp16")
    got = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, return_lse=True)
    assert_attention(got, q, cache, table, lens, prefix=prefix)


@pytest.mark.parametrize("B,H,Hkv,Sq,D,prefix,dtype", [
    (64, 16, 16, 1, 64, 1000, "fp16"), (48, 32, 8, 1, 128, 1100, "bf16"),
    (40, 32, 2, 1, 128, 5000, "fp16"), (20, 8, 8, 3, 64, 4100, "bf16"),
    (3, 64, 1, 1, 64, 65537, "bf16")])
def test_shared_prefix_apart(fa8, B, H, Hkv, Sq, D, prefix, dtype):
    """Prefixes long enough that they are met by all queries together."""
    ps = 64
    lens = [prefix + Sq + (11 * b) % 140 for b in range(B)]
    lens[1] = prefix - 3  # inside the prefix
    if B > 10:
        lens[5], lens[7] = 0, prefix
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    same_prefix(cache, table, lens, prefix)
    q = make_q(B, H, Sq, D, dtype, size=0.7)
    got = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, return_lse=True)
    assert_attention(got, q, cache, table, lens, prefix=0)
    bad = table.clone()
    bad[1:, :prefix // ps] = -5
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    same = fa8.flash_attn_fp8_shared_prefix(q, cache, bad, seqlens, prefix, status=status)
    assert torch.equal(same, got[0]) and int(status) == 0
    seqlens[2] = table.shape[1] * ps + 1  # refused: left as it was, the others served
    out = torch.full_like(q, 5.0)
    fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, out=out, status=status)
    assert int(status) == 4 and bool((out[2] == 5).all())
    keep = [b for b in range(B) if b != 2]
    tol = 4 * torch.finfo(q.dtype).eps * (got[0].abs() + 1)
    assert bool(((out - got[0]).abs() <= tol)[keep].all())


def test_shared_prefix_edges(fa8):
    """Sequences inside the prefix, empty ones, no prefix, nothing behind it."""
    prefix, ps = 200, 16
    lens = [200, 0, 50, 201, 199, 1, 300]
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, 2, ps, 64)
    same_prefix(cache, table, lens, prefix)
    for Sq in (1, 3):
        q = make_q(len(lens), 4, Sq, 64, "fp16")
        got = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, return_lse=True)
        assert_attention(got, q, cache, table, lens)
    plain = fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
    assert torch.equal(fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, 0), plain)
    bad = table.clone()
    bad[1:, :prefix // ps] = 1 << 30  # whole prefix pages of the other rows are not read
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    same = fa8.flash_attn_fp8_shared_prefix(q, cache, bad, seqlens, prefix, status=status)
    assert torch.equal(same, got[0]) and int(status) == 0
    with pytest.raises(RuntimeError):
        fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, table.shape[1] * ps + 1)


def test_prefix_refused_sequences_are_left_alone(fa8):
    prefix, ps = 64, 16
    lens = [70, 100, 80]
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, 2, ps, 64)
    q = make_q(3, 4, 1, 64, "fp16")
    want = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix)
    seqlens[1] = table.shape[1] * ps + 1
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 5.0)
    fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, out=out, status=status)
    assert int(status) == 4 and bool((out[1] == 5).all())
    tol = torch.finfo(q.dtype).eps * want.abs() + 2 * torch.finfo(q.dtype).eps
    assert bool(((out - want).abs() <= tol)[[0, 2]].all())


def test_decode_follows_the_forward(fa8):
    """The cache's attention and the framework's forward on the same e4m3 codes agree."""
    B, H, Hkv, S, D = 2, 8, 2, 256, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    q8, k8, v8 = (torch.randn(B, h, S, D, generator=g, device="cuda").to(E4M3)
                  for h in (H, Hkv, Hkv))
    o, lse = fa8.flash_attn_fp8_forward_ex(q8, k8, v8, causal=True, v_layout="bhsd",
                                           return_lse=True)
    cache = fa8.kv_cache_alloc(32, Hkv, 16, D)
    table, seqlens = make_table([S, S], 16, 32)
    fa8.kv_cache_write(cache, k8.half(), v8.half(), table, seqlens)
    o2, lse2 = fa8.flash_attn_fp8_decode(q8.half(), cache, table, seqlens, return_lse=True)
    # the values are e4m3 values already, and a power of two brings them to themselves
    # but where the shift reaches subnormal codes (below 2^-6 of the largest's binade)
    assert float((o.float() - o2.float()).abs().max()) <= 2e-2
    assert float((lse - lse2).abs().max()) <= 2e-2


def test_serving_run(fa8):
    """Prompts written, read back, then steps of write + decode, and samples of one prompt."""
    D, H, Hkv, ps, B = 128, 8, 2, 16, 3
    prompts = [33, 1, 80]
    steps = 5
    cap = [n + steps for n in prompts]
    pages = pages_for(cap, ps)
    cache = fa8.kv_cache_alloc(pages, Hkv, ps, D)
    table, _ = make_table(cap, ps, pages)
    g = torch.Generator(device="cuda").manual_seed(9)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    total = sum(prompts)
    k, v = rnd(total, Hkv, D), rnd(total, Hkv, D)
    cu = torch.tensor([0] + prompts, device="cuda").cumsum(0).int()
    seqlens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    fa8.kv_cache_write(cache, k, v, table, seqlens, cu_seqlens=cu, status=status)
    back_k, back_v = fa8.kv_cache_read(cache, table, seqlens, cu, total, dtype="bf16")
    # half a step of e4m3 at the row's factor: 2^-4 of a value, 2^-10 * 2^e below 2^-6 * 2^e
    for x, y in ((k, back_k), (v, back_v)):
        e = ref.factor(ref.quantise(x)[1]).unsqueeze(-1)
        bound = torch.maximum(y.double().abs() * 2.0 ** -4, 2.0 ** -10 * e)
        assert bool(((x.double() - y.double()).abs() <= bound).all())
    lens = list(prompts)
    for _ in range(steps):
        seqlens += 1
        lens = [n + 1 for n in lens]
        fa8.kv_cache_write(cache, rnd(B, Hkv, 1, D), rnd(B, Hkv, 1, D), table, seqlens,
                           status=status)
        q = rnd(B, H, 1, D)
        got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True, status=status)
        assert_attention(got, q, cache, table, lens)
    assert int(status) == 0


def test_graph_replay_and_streams(fa8):
    """A captured step follows its tensors; two captured graphs and a side stream run at once."""
    lens = [90, 2000, 400]
    cache = make_cache(fa8, pages_for([3000] * 3, 64), 2, 64, 128)
    table, seqlens = make_table([3000] * 3, 64, pages_for([3000] * 3, 64))
    seqlens.copy_(torch.tensor(lens))
    q = make_q(3, 8, 1, 128, "fp16")
    new = torch.randn(3, 2, 1, 128, device="cuda").half()
    graphs, outs = [], []
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        fa8.kv_cache_write(cache, new, new, table, seqlens)
        fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
    torch.cuda.current_stream().wait_stream(warm)
    for prefix in (0, 64):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            if prefix == 0:
                fa8.kv_cache_write(cache, new, new, table, seqlens)
                o = fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
            else:
                o = fa8.flash_attn_fp8_shared_prefix(q, cache, table[:1].expand(3, -1), seqlens, 64)
        graphs.append(g)
        outs.append(o)
    for lens in ([91, 2001, 401], [3000, 1, 129]):
        seqlens.copy_(torch.tensor(lens))
        new.normal_()
        graphs[0].replay()
        torch.cuda.synchronize()
        want = fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
        assert torch.equal(outs[0], want)
        wantp = fa8.flash_attn_fp8_shared_prefix(q, cache, table[:1].expand(3, -1), seqlens, 64)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        res = []
        for _ in range(20):  # both graphs and an eager call, nothing waits between
            with torch.cuda.stream(side):
                graphs[1].replay()
            graphs[0].replay()
            res.append(fa8.flash_attn_fp8_decode(q, cache, table, seqlens))
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], wantp)
        assert all(torch.equal(r, want) for r in res)


def test_offsets_past_32_bits(fa8):
    """Pages that begin behind 2^32 bytes of the cache, and exponents with them."""
    ps, Hkv, D = 128, 8, 128
    pages = (1 << 32) // (ps * Hkv * D) + 40
    k = torch.empty(pages, Hkv, ps, D, dtype=torch.uint8, device="cuda")
    v = torch.empty_like(k)
    ke = torch.empty(pages, Hkv, ps, dtype=torch.uint8, device="cuda")
    ve = torch.empty_like(ke)
    big = fa8.KVCacheFP8(k.view(E4M3), v.view(E4M3), ke, ve)
    n = 700
    x = torch.randn(2, 1, Hkv, n, D, device="cuda").bfloat16()
    table = torch.tensor([[pages - 1, 3, pages - 30, pages - 2, pages - 17, 0]],
                         dtype=torch.int32, device="cuda")
    seqlens = torch.tensor([n], dtype=torch.int32, device="cuda")
    fa8.kv_cache_write(big, x[0], x[1], table, seqlens)
    small = fa8.kv_cache_alloc(6, Hkv, ps, D)
    t2 = torch.arange(6, dtype=torch.int32, device="cuda").view(1, 6)
    fa8.kv_cache_write(small, x[0], x[1], t2, seqlens)
    for a, b in zip(fa8.kv_cache_read(big, table, seqlens, None, n),
                    fa8.kv_cache_read(small, t2, seqlens, None, n)):
        assert torch.equal(a, b)
    q = make_q(1, 32, 1, D, "bf16")
    assert torch.equal(fa8.flash_attn_fp8_decode(q, big, table, seqlens),
                       fa8.flash_attn_fp8_decode(q, small, t2, seqlens))


def test_torch_layer_refusals(fa8):
    cache = make_cache(fa8, 4, 2, 16, 64)
    table, seqlens = make_table([20], 16, 4)
    q = make_q(1, 4, 1, 64, "fp16")
    x = torch.randn(1, 2, 1, 64, device="cuda").half()
    bad = [
        lambda: fa8.flash_attn_fp8_decode(q.float(), cache, table, seqlens),
        lambda: fa8.flash_attn_fp8_decode(q[0], cache, table, seqlens),
        lambda: fa8.flash_attn_fp8_decode(q[:, :3], cache, table, seqlens),
        lambda: fa8.flash_attn_fp8_decode(q, cache, table, seqlens[:0]),
        lambda: fa8.flash_attn_fp8_decode(q, cache, table.float(), seqlens),
        lambda: fa8.flash_attn_fp8_decode(q, cache, table[0], seqlens),
        lambda: fa8.flash_attn_fp8_decode(q, cache._replace(k=cache.k_exp), table, seqlens),
        lambda: fa8.flash_attn_fp8_decode(q, cache._replace(v_exp=cache.v_exp[:2]), table, seqlens),
        lambda: fa8.flash_attn_fp8_decode(q, cache, table, seqlens, softmax_scale=-1.0),
        lambda: fa8.flash_attn_fp8_decode(q, cache, table, seqlens, out=q.float()),
        lambda: fa8.flash_attn_fp8_decode(q, cache, table, seqlens,
                                          status=torch.zeros(1, device="cuda")),
        lambda: fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, -1),
        lambda: fa8.kv_cache_write(cache, x.float(), x.float(), table, seqlens),
        lambda: fa8.kv_cache_write(cache, x, x[..., :32], table, seqlens),
        lambda: fa8.kv_cache_write(cache, x.cpu(), x.cpu(), table, seqlens),
        lambda: fa8.kv_cache_write(cache, x, x, table, seqlens, cu_seqlens=seqlens),
        lambda: fa8.kv_cache_read(cache, table, seqlens, None, 1, dtype="fp32"),
        lambda: fa8.kv_cache_read(cache, table, seqlens, None, -1),
        lambda: fa8.kv_cache_read(cache, table, seqlens, None, 1, out=(x, x[..., :32])),
        lambda: fa8.kv_cache_read(cache, table, seqlens, None, 1,
                                  out=(x.expand(1, 2, 1, 64), x[:, :1].expand(1, 2, 1, 64))),
    ]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    odd = torch.zeros(4, 2, 16, 72, dtype=torch.uint8, device="cuda")[..., :64].view(E4M3)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        fa8.flash_attn_fp8_decode(q, cache._replace(k=odd), table, seqlens)
    empty = fa8.flash_attn_fp8_decode(q[:0], cache, table[:0], seqlens[:0])
    assert empty.shape == (0, 4, 1, 64)
    nothing = fa8.flash_attn_fp8_decode(q, fa8.kv_cache_alloc(0, 2, 16, 64), table[:, :0],
                                        torch.zeros_like(seqlens))
    assert bool((nothing == 0).all())
