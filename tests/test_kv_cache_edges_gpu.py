"""GPU checks of the cache's attention where it can go wrong: calls whose waits run
out beside calls of another stream; value rows of zeros, and of very different and
very large or small values; queries with one large element.

Tolerances, with u = eps / 2 of q's type (2^-11 fp16, 2^-8 bf16), p the weights, w
their sum, c_j the codes and 2^e_j the factor of value row j:
* the result is rounded once: u |o|, or half a subnormal step where that is more
  (fp16 values below 2^-14 are multiples of 2^-24: 2^-25); p is rounded once: u A,
  A = sum p |v| / w;
* scores: fp32 sums of D products, each addition off by 2^-22 of the largest partial
  sum B, and q's elements by half the least step of the last term: ds = D 2^-22 B +
  2^-21 (bf16) or 2^-25 (fp16) of the row's largest |q| times the largest scale *
  sum |k| of a key. It moves the quotient by 2 ds A. exp2 and sums: 2^-20 A. Where
  exponents of values differ by E, or are up to E (40 at most) away from -7, that of
  unit normal rows (rows of zeros count as 40 away), weights are exponentials of
  numbers up to E + 8 that were rounded twice, each time by half a unit in the last
  place: ln 2 * 2^-23 (E + 8), of which 8 is within the 2^-20: 2^-23 E A;
* results of parts are joined by their weights, and fp32 holds none under 2^-126
  of the row's largest (rounded up to a power of two): 2^-125 sum |v_j|;
* small p meet a floor, 2^-17 or 2^-21 of the row's largest p_j 2^e_j over rows j
  that are not zero, for every key: that times sum_j |c_j| / w.
lse: ds + 2^-23 E + 2^-20 (1 + |lse|). A result beyond the type's largest is infinite.
"""
import math

import pytest

from oracle import kv_cache_ref as ref
from tests.test_kv_cache_gpu import (E4M3, make_cache, make_q, make_table, pages_for,
                                     same_prefix, shared_table, u8)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa8(cuda):
    import ada_cute_fp8_flash_attention_b200 as m
    return m


def held(codes_u8, exps, row, n):
    """float64 code values (H_kv, n, D) and exponents (H_kv, n) of a sequence's tokens."""
    pos = torch.arange(n, device="cuda")
    page, slot = row.long()[pos // codes_u8.shape[2]], pos % codes_u8.shape[2]
    codes = ref.decode_e4m3(codes_u8[page, :, slot]).transpose(0, 1)
    return codes, exps[page, :, slot].transpose(0, 1).double() - 127


def assert_near(got, q, cache, table, lens, scale=None):
    """Output and lse against 64 bits, by the bounds at the head of this file."""
    out, lse = got
    B, H, Sq, D = q.shape
    G = H // cache.k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    fp16 = q.dtype == torch.float16
    info = torch.finfo(q.dtype)
    u, top, least = info.eps / 2, info.max, info.smallest_normal * info.eps / 2
    for b, n in enumerate(lens):
        kc, ke = held(u8(cache.k), cache.k_exp, table[b], n)
        vc, ve = held(u8(cache.v), cache.v_exp, table[b], n)
        k, c, e = (x.repeat_interleave(G, 0) for x in (kc * torch.exp2(ke).unsqueeze(-1), vc, ve))
        v = c * torch.exp2(e).unsqueeze(-1)
        for i in range(Sq):
            m = n - Sq + i + 1
            if m <= 0:
                assert bool((out[b, :, i] == 0).all()) and bool((lse[b, :, i] == -math.inf).all())
                continue
            x = q[b, :, i].double()
            s = torch.einsum("hd,hnd->hn", x, k[:, :m]) * scale
            mag = torch.einsum("hd,hnd->hn", x.abs(), k[:, :m].abs()) * scale
            ks = k[:, :m].abs().sum(-1).amax(-1) * scale
            ds = D * 2.0 ** -22 * mag.amax(-1) + x.abs().amax(-1) * 2.0 ** (-25 if fp16 else -21) * ks
            p = torch.exp(s - s.amax(-1, keepdim=True))
            w = p.sum(-1)
            want = torch.einsum("hn,hnd->hd", p, v[:, :m]) / w[:, None]
            A = torch.einsum("hn,hnd->hd", p, v[:, :m].abs()) / w[:, None]
            solid = (c[:, :m] != 0).any(-1)
            # in logs: p may be less than a double holds and 2^e as large
            lead = torch.where(solid, s / math.log(2) + e[:, :m], -math.inf).amax(-1)
            lead = torch.exp2(lead - torch.logsumexp(s, -1) / math.log(2))
            floor = lead[:, None] * c[:, :m].abs().sum(1) * 2.0 ** (-21 if fp16 else -17)
            E = (torch.where(solid, e[:, :m], -math.inf).amax(-1)
                 - torch.where(solid, e[:, :m], math.inf).amin(-1)).clamp(min=0).unsqueeze(-1)
            away = torch.where(solid, (e[:, :m] + 7).abs(), 40.0).amax(-1).clamp(max=40)
            E = torch.maximum(E, away.unsqueeze(-1))
            tol = ((u * want.abs()).clamp(min=least)
                   + (u + 2 * ds[:, None] + 2.0 ** -20 + 2.0 ** -23 * E) * A + floor
                   + 2.0 ** -125 * v[:, :m].abs().sum(1))
            err = (out[b, :, i].double() - want).abs()
            far = want.abs() + tol > top  # may be infinite
            bad = (~(err <= tol)) & ~far
            assert not bool(bad.any()), \
                f"out: {float(err[bad].max()):.3g} over {float(tol[bad].min()):.3g}"
            wlse = torch.logsumexp(s, -1)
            ltol = ds + 2.0 ** -23 * E.squeeze(-1) + 2.0 ** -20 * (1 + wlse.abs())
            lerr = (lse[b, :, i].double() - wlse).abs()
            assert bool((lerr <= ltol).all()), \
                f"lse: {float(lerr.max()):.3g} over {float(ltol.min()):.3g}"


def c_decode(cache, table, seqlens, q, out, status=None, prefix=0, lse=None):
    """The C ABI's parameters of a call on contiguous tensors, and its workspace."""
    from ada_cute_fp8_flash_attention_b200 import c_abi
    pages, heads_kv, page_size, D = cache.k.shape
    B, H, Sq, _ = q.shape
    p = c_abi.decode_params(pages, heads_kv, page_size, D, B, table.shape[1], H, Sq)
    c = p.cache
    c.k, c.v = cache.k.data_ptr(), cache.v.data_ptr()
    c.k_exp, c.v_exp = cache.k_exp.data_ptr(), cache.v_exp.data_ptr()
    c.page_table, c.seqlens = table.data_ptr(), seqlens.data_ptr()
    c.status = status.data_ptr() if status is not None else None
    p.q, p.o, p.prefix_len = q.data_ptr(), out.data_ptr(), prefix
    p.lse = lse.data_ptr() if lse is not None else None
    p.dtype = c_abi.FA8_DT_BF16 if q.dtype == torch.bfloat16 else c_abi.FA8_DT_F16
    size = c_abi.decode_workspace_size(p)
    assert size > 0
    return p, torch.empty(size, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("D,Hkv,G,n", [(128, 8, 4, 700), (64, 8, 2, 1000), (128, 4, 64, 500)])
def test_waits_that_run_out_beside_another_stream(fa8, D, Hkv, G, n):
    """Shares of one or two tiles, which fit the ring: the loading warp never waits,
    whoever gives up. Blocks that end early leave nothing behind that lands in the
    shared memory of the calls beside and after them."""
    from ada_cute_fp8_flash_attention_b200 import c_abi
    lens = [n, n // 2, n // 3]
    pages = pages_for(lens, 64)
    cache = make_cache(fa8, pages, Hkv, 64, D)
    table, seqlens = make_table(lens, 64, pages)
    q = make_q(3, Hkv * G, 1, D, "fp16")
    want = fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, good = torch.zeros_like(q), [torch.zeros_like(q) for _ in range(20)]
    p, ws = c_decode(cache, table, seqlens, q, out, status)
    p.wait_timeout_cycles = 1
    fine = [c_decode(cache, table, seqlens, q, o) for o in good]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for pg, wg in fine:
        c_abi.check(c_abi.decode(p, ws.data_ptr(), ws.numel(),
                                 torch.cuda.current_stream().cuda_stream))
        c_abi.check(c_abi.decode(pg, wg.data_ptr(), wg.numel(), side.cuda_stream))
    torch.cuda.synchronize()
    assert int(status) == 1
    assert all(torch.equal(o, want) for o in good)
    p.wait_timeout_cycles = 0
    c_abi.check(c_abi.decode(p, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def put_row(cache, table, page_size, b, pos, k=None, v=None):
    """Token `pos` of sequence b gets these K and V rows (H_kv, D), float64."""
    page, slot = int(table[b, pos // page_size]), pos % page_size
    for name, x in (("k", k), ("v", v)):
        if x is not None:
            values, byte = ref.quantise(x)
            u8(getattr(cache, name))[page, :, slot] = u8(values.float().to(E4M3))
            getattr(cache, name + "_exp")[page, :, slot] = byte


def toward(q, score, heads_kv):
    """A key (H_kv, D) whose score with the mean query row of each group is `score`."""
    D = q.shape[-1]
    x = q.double().view(heads_kv, -1, D).mean(1)
    return x * (score * D ** 0.5 / (x * x).sum(-1, keepdim=True))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("size", [1.0, 0.1, 1e-3])
@pytest.mark.parametrize("D,H,Hkv,Sq,where", [(128, 8, 2, 1, 0), (64, 4, 4, 3, 200),
                                              (128, 32, 1, 2, 511), (128, 64, 1, 2, 130)])
def test_decode_row_of_zeros(fa8, D, H, Hkv, Sq, where, size, dtype):
    """A value row of zeros under the top score leaves the others' precision alone."""
    lens, ps = [512, 512, 40], 16
    pages = pages_for(lens, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    values, byte = ref.quantise(cache.v.double() * ref.factor(cache.v_exp).unsqueeze(-1) * size)
    cache = cache._replace(v=values.float().to(E4M3), v_exp=byte)
    table, seqlens = make_table(lens, ps, pages)
    q = make_q(3, H, Sq, D, dtype, size=1.0)
    zero = torch.zeros(Hkv, D, dtype=torch.float64, device="cuda")
    for b, pos in ((0, where), (1, 5), (1, where), (2, 36)):
        put_row(cache, table, ps, b, pos, toward(q[b], 8.0, Hkv), zero)
    u8(cache.v)[int(table[1, 0]), :, 5] = 128  # minus zeros
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_near(got, q, cache, table, lens)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("size", [1.0, 0.1, 1e-3])
def test_shared_prefix_row_of_zeros(fa8, size, dtype):
    D, H, Hkv, ps, prefix, B = 128, 32, 8, 16, 1040, 48
    lens = [prefix + 1 + (7 * b) % 50 for b in range(B)]
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    values, byte = ref.quantise(cache.v.double() * ref.factor(cache.v_exp).unsqueeze(-1) * size)
    cache = cache._replace(v=values.float().to(E4M3), v_exp=byte)
    same_prefix(cache, table, lens, prefix)
    q = make_q(B, H, 1, D, dtype, size=1.0)
    zero = torch.zeros(Hkv, D, dtype=torch.float64, device="cuda")
    put_row(cache, table, ps, 0, 0, toward(q[0], 8.0, Hkv), zero)
    put_row(cache, table, ps, 0, 777, toward(q[3], 8.0, Hkv), zero)
    put_row(cache, table, ps, 5, lens[5] - 1, toward(q[5], 9.0, Hkv), zero)
    before = fa8.launch_count()
    got = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, return_lse=True)
    assert fa8.launch_count() - before == 3  # the prefix has a launch of its own
    assert_near(got, q, cache, table, lens)


def resized(cache, size, name="v"):
    """The cache with its V (or K) rows multiplied by `size` (pages, heads, slots), float64."""
    x = getattr(cache, name).double() * ref.factor(getattr(cache, name + "_exp")).unsqueeze(-1)
    values, byte = ref.quantise(x * size.unsqueeze(-1))
    return cache._replace(**{name: values.float().to(E4M3), name + "_exp": byte})


SIZES = {  # powers of two that value rows (of about 1) are multiplied by, by position
    "largest": lambda pos, rnd: 110 + 14 * rnd,
    "least": lambda pos, rnd: -60 + 4 * rnd,
    "any": lambda pos, rnd: -64 + 188 * rnd,
    "growing": lambda pos, rnd: -60 + 184 * pos,
    "shrinking": lambda pos, rnd: 124 - 184 * pos,
    "few large": lambda pos, rnd: torch.where(rnd > 0.99, 120.0, 0.0),
    "few small": lambda pos, rnd: torch.where(rnd > 0.99, -60.0, 20.0),
    "late": lambda pos, rnd: torch.where(pos > 0.97, 123.0, -30.0),
    "near": lambda pos, rnd: 48 * rnd,
    "edges": lambda pos, rnd: torch.where(rnd > 0.5, 39.0, -39.0) + 3 * pos,  # of one reference
    "low edge": lambda pos, rnd: -41 + 3 * rnd,
}


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("D,H,Hkv,Sq,spread", [(128, 8, 2, 1, 1.0), (64, 4, 4, 3, 30.0),
                                               (128, 32, 1, 2, 4.0), (128, 64, 1, 1, 60.0),
                                               (64, 16, 2, 1, 1.0)])
def test_decode_range_of_values(fa8, D, H, Hkv, Sq, spread, sizes, dtype):
    """Values of any size beside each other; keys whose scores differ by up to hundreds."""
    lens, ps = [700, 1300, 40, 129], 64
    pages = pages_for(lens, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    table, seqlens = make_table(lens, ps, pages)
    g = torch.Generator(device="cuda").manual_seed(11)
    power = torch.zeros(pages, Hkv, ps, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        for col in range(-(-n // ps)):
            pos = (col * ps + torch.arange(ps, device="cuda").double()) / n
            rnd = torch.rand(Hkv, ps, generator=g, device="cuda").double()
            power[int(table[b, col])] = SIZES[sizes](pos.expand(Hkv, ps), rnd)
    cache = resized(cache, torch.exp2(torch.floor(power)))
    q = make_q(4, H, Sq, D, dtype, size=spread)
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_near(got, q, cache, table, lens)
    again = fa8.flash_attn_fp8_decode(q, cache, table, seqlens)
    assert torch.equal(again.nan_to_num(7.0), got[0].nan_to_num(7.0))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("sizes", ["any", "late", "few large"])
def test_shared_prefix_range_of_values(fa8, sizes, dtype):
    D, H, Hkv, ps, prefix, B = 128, 32, 8, 16, 1040, 48
    lens = [prefix + 1 + (7 * b) % 50 for b in range(B)]
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    g = torch.Generator(device="cuda").manual_seed(12)
    rnd = torch.rand(pages, Hkv, ps, generator=g, device="cuda").double()
    pos = torch.linspace(0, 1, pages * ps, device="cuda").double().view(pages, 1, ps)
    cache = resized(cache, torch.exp2(torch.floor(SIZES[sizes](pos.expand(-1, Hkv, -1), rnd))))
    same_prefix(cache, table, lens, prefix)
    q = make_q(B, H, 1, D, dtype, size=3.0)
    got = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, return_lse=True)
    assert_near(got, q, cache, table, lens)


def test_written_values_near_the_largest(fa8):
    """bf16 rows of 1e30 to 3e38 through the write, beside ordinary ones."""
    D, H, Hkv, ps, n = 128, 8, 2, 16, 300
    g = torch.Generator(device="cuda").manual_seed(4)
    cache = fa8.kv_cache_alloc(2 * 20, Hkv, ps, D)
    table, seqlens = make_table([n, n], ps, 40)
    x = torch.randn(2, 2, Hkv, n, D, generator=g, device="cuda").double()
    power = 10 ** (30 + 8 * torch.rand(2, Hkv, n, 1, generator=g, device="cuda").double())
    v = (x[1].clamp(-3, 3) * power).clamp(-3e38, 3e38)
    v[1, :, ::2] = x[1][1, :, ::2]  # the second sequence: every other row an ordinary one
    fa8.kv_cache_write(cache, x[0].bfloat16(), v.bfloat16(), table, seqlens)
    q = make_q(2, H, 1, D, "bf16")
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert bool(torch.isfinite(got[1]).all())
    assert_near(got, q, cache, table, [n, n])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("k_bytes,v_bytes,code", [
    ((100, 130), (0, 3), 0x7e), ((100, 130), (250, 254), 0x38), ((100, 130), (0, 254), 0x38),
    ((0, 2), (120, 130), 0x7e), ((0, 130), (110, 120), 0x7e)])
def test_bytes_at_both_ends(fa8, k_bytes, v_bytes, code, dtype):
    """A cache that a caller brings: any byte but 255, codes up to `code` for V."""
    D, H, Hkv, ps = 64, 8, 2, 32
    lens = [500, 33]
    pages = pages_for(lens, ps)
    g = torch.Generator(device="cuda").manual_seed(8)
    cache = make_cache(fa8, pages, Hkv, ps, D)
    byte = lambda lo, hi: torch.randint(lo, hi + 1, (pages, Hkv, ps), generator=g,  # noqa: E731
                                        device="cuda", dtype=torch.uint8)
    codes = torch.randint(0, code + 1, cache.v.shape, generator=g, device="cuda", dtype=torch.uint8)
    sign = torch.randint(0, 2, cache.v.shape, generator=g, device="cuda", dtype=torch.uint8) * 128
    cache = cache._replace(v=(codes | sign).view(E4M3), k_exp=byte(*k_bytes), v_exp=byte(*v_bytes))
    table, seqlens = make_table(lens, ps, pages)
    q = make_q(2, H, 1, D, dtype, size=0.02)
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_near(got, q, cache, table, lens)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_query_with_one_large_element(fa8, dtype):
    """The largest element meets zeros of K: the others are what the scores are made of."""
    lens, D, H, Hkv = [600, 200], 128, 8, 2
    cache = make_cache(fa8, pages_for(lens, 16), Hkv, 16, D, spread=0.3)
    u8(cache.k)[..., 5] = 0
    table, seqlens = make_table(lens, 16, pages_for(lens, 16))
    for large in (64.0, 2048.0, 30000.0):
        q = make_q(2, H, 1, D, dtype)
        q[..., 5] = large
        got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
        assert_near(got, q, cache, table, lens)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("above", [5.0, 25.0, 60.0, 300.0])
@pytest.mark.parametrize("H,Hkv,zeros", [(8, 2, 1), (8, 2, 200), (64, 1, 130)])
def test_decode_zeros_far_above(fa8, H, Hkv, zeros, above, dtype):
    """Leading rows of zeros whose scores are far above the others', and far below."""
    lens, ps, D = [640, 300], 16, 128
    pages = pages_for(lens, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    table, seqlens = make_table(lens, ps, pages)
    q = make_q(2, H, 1, D, dtype, size=1.0)
    zero = torch.zeros(Hkv, D, dtype=torch.float64, device="cuda")
    for b, sign in ((0, 1), (1, -1)):
        for pos in range(zeros):
            put_row(cache, table, ps, b, pos, toward(q[b], sign * above, Hkv), zero)
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert_near(got, q, cache, table, lens)


@pytest.mark.parametrize("B", [4, 64])
@pytest.mark.parametrize("first", [0, 1, 700, 960, 975])
def test_shared_prefix_behind_a_short_first_sequence(fa8, first, B):
    """Whole prefix pages come from row 0 whatever its length, what is behind them from
    each row: the same pages in a small batch and in a large one."""
    D, H, Hkv, ps, prefix = 128, 32, 8, 64, 1000
    lens = [prefix + 1 + (7 * b) % 90 for b in range(B)]
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    same_prefix(cache, table, lens, prefix)
    col = prefix // ps
    lens[0] = first
    seqlens[0] = first
    if first <= col * ps:
        table[0, col] = -1  # the first sequence needs no page there
    else:  # its own page holds its own tokens of the prefix, and then anything
        page = int(table[0, col])
        u8(cache.k)[page, :, first - col * ps:] = 0x7f
        cache.v_exp[page, :, first - col * ps:] = 255
    table[0, col + 1:] = -1
    q = make_q(B, H, 1, D, "bf16")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = fa8.launch_count()
    got = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, return_lse=True,
                                           status=status)
    assert fa8.launch_count() - before == (3 if B == 64 else 2)
    assert int(status) == 0
    assert_near(got, q, cache, table, lens)


def prefix_case(fa8, B, H, Hkv, Sq, D, prefix, ps, dtype, size=0.7):
    """A batch for which the prefix has a launch of its own; one sequence ends inside it,
    one is empty, one ends with it."""
    lens = [prefix + Sq + (11 * b) % 140 for b in range(B)]
    lens[1], lens[5], lens[7] = prefix - 3, 0, prefix
    table, seqlens, pages = shared_table(lens, prefix, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    same_prefix(cache, table, lens, prefix)
    return cache, table, seqlens, lens, make_q(B, H, Sq, D, dtype, size=size)


def prefix_call(fa8, q, cache, table, seqlens, prefix, **kw):
    before = fa8.launch_count()
    got = fa8.flash_attn_fp8_shared_prefix(q, cache, table, seqlens, prefix, return_lse=True, **kw)
    assert fa8.launch_count() - before == 3  # the prefix, what is behind it, the join
    return got


@pytest.mark.parametrize("D,dtype", [(64, "fp16"), (128, "bf16"), (128, "fp16")])
@pytest.mark.parametrize("ps,prefix", [(16, 1009), (32, 1000), (64, 1024), (128, 1300), (256, 1500),
                                       (384, 1600), (1024, 1024)])
def test_prefix_apart_pages(fa8, ps, prefix, D, dtype):
    cache, table, seqlens, lens, q = prefix_case(fa8, 48, 32, 16, 1, D, prefix, ps, dtype)
    got = prefix_call(fa8, q, cache, table, seqlens, prefix)
    assert_near(got, q, cache, table, lens)
    again = prefix_call(fa8, q, cache, table, seqlens, prefix)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


@pytest.mark.parametrize("B,H,Hkv,Sq,D", [(64, 64, 8, 1, 128), (32, 32, 8, 5, 64), (400, 8, 8, 1, 64),
                                          (20, 16, 2, 33, 128)])
def test_prefix_apart_row_shapes(fa8, B, H, Hkv, Sq, D):
    prefix = 1500
    cache, table, seqlens, lens, q = prefix_case(fa8, B, H, Hkv, Sq, D, prefix, 32, "bf16")
    got = prefix_call(fa8, q, cache, table, seqlens, prefix)
    assert_near(got, q, cache, table, lens)


@pytest.mark.parametrize("where", ["k", "v"])
def test_prefix_apart_nan_rows(fa8, where):
    """A NaN token inside the prefix reaches the queries that see it, one behind it its
    own sequence's."""
    prefix, Sq = 1100, 3
    cache, table, seqlens, lens, q = prefix_case(fa8, 48, 32, 8, Sq, 128, prefix, 16, "fp16")
    clean, _ = prefix_call(fa8, q, cache, table, seqlens, prefix)
    exps = cache.k_exp if where == "k" else cache.v_exp
    codes = u8(cache.k if where == "k" else cache.v)
    lens[9] = seqlens[9] = prefix + 40
    for b, pos, head in ((0, 1080, 2), (9, prefix + 38, 5)):  # the second: one of its queries is before it
        page, slot = int(table[b, pos // 16]), pos % 16
        exps[page, head, slot] = 255
        codes[page, head, slot] = 0
    out, lse = prefix_call(fa8, q, cache, table, seqlens, prefix)
    want = torch.zeros(48, 32, Sq, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        for i in range(Sq):
            want[b, 8:12, i] = n - Sq + i >= 1080
    want[9, 20:24, 1:] = True
    bad = out.isnan()
    assert torch.equal(bad.all(-1), want) and torch.equal(bad.any(-1), want)
    keep = ~want
    keep[9] = False  # another length than before
    assert torch.equal(out[keep], clean[keep])
    assert not bool(lse[~want].isnan().any())


def test_prefix_apart_bad_pages(fa8):
    """Page ids outside the cache, inside the prefix and behind it; a refused length."""
    prefix, ps = 1024, 16
    cache, table, seqlens, lens, q = prefix_case(fa8, 48, 32, 8, 1, 128, prefix, ps, "bf16")
    clean, _ = prefix_call(fa8, q, cache, table, seqlens, prefix)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    bad = table.clone()
    bad[3, prefix // ps] = cache.k.shape[0]
    bad[4, prefix // ps] = -(1 << 31)
    out, lse = prefix_call(fa8, q, cache, bad, seqlens, prefix, status=status)
    assert int(status) == 8
    for b in range(48):
        if b in (3, 4):
            assert bool(out[b].isnan().all()) and bool(lse[b].isnan().all())
        else:
            assert torch.equal(out[b], clean[b])
    bad = table.clone()
    bad[0, 30] = 1 << 30  # of the prefix: all sequences but those that end before it
    status.zero_()
    out, _ = prefix_call(fa8, q, cache, bad, seqlens, prefix, status=status)
    assert int(status) == 8
    seen = torch.tensor(lens, device="cuda") > 30 * ps
    assert torch.equal(out.isnan().all(-1).all(-1).all(-1), seen)
    assert bool((out[~seen] == clean[~seen]).all())
    status.zero_()
    seqlens[2], seqlens[6] = -1, table.shape[1] * ps + 1
    out = torch.full_like(q, 5.0)
    prefix_call(fa8, q, cache, table, seqlens, prefix, out=out, status=status)
    assert int(status) == 4 and bool((out[2] == 5).all()) and bool((out[6] == 5).all())
    tol = 2 * torch.finfo(q.dtype).eps * (clean.abs() + 1)  # other shares of the work: other sums
    keep = [b for b in range(48) if b not in (2, 6)]
    assert bool(((out - clean).abs() <= tol)[keep].all())


def test_prefix_apart_captured(fa8):
    """The chain of three launches in a graph: replayed back to back, with other lengths,
    on a side stream beside eager calls."""
    prefix, ps = 1024, 16
    cache, table, seqlens, lens, q = prefix_case(fa8, 48, 32, 8, 1, 128, prefix, ps, "bf16")
    room = table.shape[1] * ps
    table = table.clamp(min=0)  # every row full: the lengths change
    prefix_call(fa8, q, cache, table, seqlens, prefix)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = prefix_call(fa8, q, cache, table, seqlens, prefix)
    side = torch.cuda.Stream()
    for lengths in (lens, [room - 7 * b % 50 for b in range(48)], [prefix] * 48, [0] * 48,
                    [1 + 24 * b for b in range(48)]):
        assert max(lengths) <= room
        seqlens.copy_(torch.tensor(lengths))
        want = prefix_call(fa8, q, cache, table, seqlens, prefix)
        for t in got:
            t.fill_(3.0)
        torch.cuda.synchronize()
        eager = []
        with torch.cuda.stream(side):
            for _ in range(10):
                g.replay()
        for _ in range(10):
            eager.append(prefix_call(fa8, q, cache, table, seqlens, prefix))
        torch.cuda.synchronize()
        for o, l in [got] + eager:
            assert torch.equal(o, want[0]) and torch.equal(l, want[1])


@pytest.mark.parametrize("host", [False, True])
def test_wide_integers_are_not_cut(fa8, host):
    """64-bit page ids and lengths beyond 32 bits are refused like any other."""
    D, Hkv, ps = 64, 2, 16
    cache = make_cache(fa8, 8, Hkv, ps, D)
    table = torch.arange(8, dtype=torch.int64).view(2, 4)
    lens = torch.tensor([50, 20])
    place = (lambda t: t) if host else (lambda t: t.cuda())  # noqa: E731
    q = make_q(2, 4, 1, D, "fp16")
    want = fa8.flash_attn_fp8_decode(q, cache, place(table), place(lens))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for far in (1 << 32, -(1 << 32), 1 << 62):
        bad = table.clone()
        bad[0, 1] += far
        status.zero_()
        out = fa8.flash_attn_fp8_decode(q, cache, place(bad), place(lens), status=status)
        assert int(status) == 8 and bool(out[0].isnan().all()) and torch.equal(out[1], want[1])
        status.zero_()
        out = torch.full_like(q, 5.0)
        fa8.flash_attn_fp8_decode(q, cache, place(table), place(lens + torch.tensor([far, 0])),
                                  out=out, status=status)
        assert int(status) == 4 and bool((out[0] == 5).all())
        assert float((out[1] - want[1]).abs().max()) <= 2 * torch.finfo(q.dtype).eps * (
            1 + float(want[1].abs().max()))
        x = torch.randn(2, Hkv, 1, D, device="cuda").half()
        before = u8(cache.k).clone()
        status.zero_()
        fa8.kv_cache_write(cache, x, x, place(table), place(lens + far), status=status)
        assert int(status) == 4 and torch.equal(u8(cache.k), before)


def c_copy(cache, table, seqlens, k, v, cu=None, status=None):
    """The C ABI's parameters of a copy of packed (with cu) or dense contiguous rows."""
    from ada_cute_fp8_flash_attention_b200 import c_abi
    pages, heads_kv, page_size, D = cache.k.shape
    p = c_abi.kv_copy_params(pages, heads_kv, page_size, D, seqlens.numel(), table.shape[1])
    c = p.cache
    c.k, c.v = cache.k.data_ptr(), cache.v.data_ptr()
    c.k_exp, c.v_exp = cache.k_exp.data_ptr(), cache.v_exp.data_ptr()
    c.page_table, c.seqlens = table.data_ptr(), seqlens.data_ptr()
    c.status = status.data_ptr() if status is not None else None
    p.k, p.v = k.data_ptr(), v.data_ptr()
    p.dtype = c_abi.FA8_DT_BF16 if k.dtype == torch.bfloat16 else c_abi.FA8_DT_F16
    if cu is not None:
        p.cu_seqlens, p.tokens = cu.data_ptr(), k.shape[0]
        p.k_stride_s, p.k_stride_h = k.stride(0), k.stride(1)
        p.v_stride_s, p.v_stride_h = v.stride(0), v.stride(1)
    else:
        p.tokens = k.shape[2]
        p.k_stride_b, p.k_stride_h, p.k_stride_s = k.stride()[:3]
        p.v_stride_b, p.v_stride_h, p.v_stride_s = v.stride()[:3]
    return p


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,heads_kv,n", [(64, 3, 5), (128, 8, 300)])
def test_c_abi_write_read_decode(fa8, D, heads_kv, n, dtype):
    """The C entry points on a side stream give what the torch ones do, packed and dense."""
    from ada_cute_fp8_flash_attention_b200 import c_abi
    B, ps = 3, 32
    lens = [n + 40, n, n + 7]
    pages = pages_for(lens, ps)
    table, seqlens = make_table(lens, ps, pages)
    x = torch.randn(2, B, heads_kv, n, D, device="cuda").to(dtype)
    packed = [t.transpose(1, 2).reshape(B * n, heads_kv, D).contiguous() for t in x]
    cu = torch.arange(B + 1, dtype=torch.int32, device="cuda") * n
    want = make_cache(fa8, pages, heads_kv, ps, D)
    dense, rows = (type(want)(*(u8(t).clone().view(t.dtype) for t in want)) for _ in range(2))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    fa8.kv_cache_write(want, x[0], x[1], table, seqlens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    c_abi.check(c_abi.kv_write(c_copy(dense, table, seqlens, x[0], x[1], status=status),
                               side.cuda_stream))
    c_abi.check(c_abi.kv_write(c_copy(rows, table, seqlens, *packed, cu=cu, status=status),
                               side.cuda_stream))
    back = [torch.zeros_like(t) for t in packed]
    c_abi.check(c_abi.kv_read(c_copy(rows, table, seqlens, *back, cu=cu, status=status),
                              side.cuda_stream))
    back4 = [torch.zeros_like(t) for t in x]
    c_abi.check(c_abi.kv_read(c_copy(dense, table, seqlens, *back4, status=status),
                              side.cuda_stream))
    q = make_q(B, 2 * heads_kv, 1, D, "bf16" if dtype == torch.bfloat16 else "fp16")
    side.wait_stream(torch.cuda.current_stream())
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:3], device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    p, ws = c_decode(dense, table, seqlens, q, out, status, lse=lse)
    c_abi.check(c_abi.decode(p, ws.data_ptr(), ws.numel(), side.cuda_stream))
    side.synchronize()
    assert int(status) == 0
    for a, b, c in zip(want, dense, rows):
        assert torch.equal(u8(a), u8(b)) and torch.equal(u8(a), u8(c))
    name = "bf16" if dtype == torch.bfloat16 else "fp16"
    k, v = fa8.kv_cache_read(want, table, seqlens, None, n, dtype=name)
    assert torch.equal(back4[0], k) and torch.equal(back4[1], v)
    k, v = fa8.kv_cache_read(want, table, seqlens, cu, B * n, dtype=name)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    o, l = fa8.flash_attn_fp8_decode(q, want, table, seqlens, return_lse=True)
    assert torch.equal(out, o) and torch.equal(lse, l)


@pytest.mark.parametrize("size,k_byte", [(1e36, 8), (1e37, 4), (1e-28, 214), (1.0, 127)])
def test_extreme_queries_over_values_of_any_size(fa8, size, k_byte):
    """bf16 queries at both ends of the type over keys at the other end: the scores are
    ordinary, whichever way an item is computed; a query with an infinity is NaN."""
    D, H, Hkv, ps = 128, 8, 2, 32
    lens = [300, 45]
    pages = pages_for(lens, ps)
    g = torch.Generator(device="cuda").manual_seed(3)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.0)
    codes = torch.randint(0x20, 0x39, cache.k.shape, generator=g, device="cuda", dtype=torch.uint8)
    sign = torch.randint(0, 2, cache.k.shape, generator=g, device="cuda", dtype=torch.uint8) * 128
    cache = cache._replace(k=(codes | sign).view(E4M3), k_exp=torch.full_like(cache.k_exp, k_byte))
    table, seqlens = make_table(lens, ps, pages)
    for apart in (False, True):
        if apart:  # exponents of V far apart
            cache.v_exp.copy_(torch.randint(60, 200, cache.v_exp.shape, generator=g, device="cuda",
                                            dtype=torch.uint8))
        q = (size * make_q(2, H, 1, D, "bf16", size=1.0).float()).bfloat16()
        got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
        assert_near(got, q, cache, table, lens)
        q[0, 1, 0, :] = math.inf
        q[1, 2, 0, 7] = -math.inf
        out, lse = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
        want = torch.zeros(2, H, 1, dtype=torch.bool, device="cuda")
        want[0, 1] = want[1, 2] = True
        assert torch.equal(out.isnan().all(-1), want) and torch.equal(lse.isnan(), want)
        assert torch.equal(out[~want], got[0][~want])


@pytest.mark.parametrize("prefix", [0, 1024])
def test_result_over_its_own_queries(fa8, prefix):
    """out=q, and out a view of q's memory, for ordinary values and for such as are
    computed again."""
    cache, table, seqlens, lens, q = prefix_case(fa8, 48, 32, 8, 1, 128, max(prefix, 64), 16, "bf16")
    for far in (False, True):
        if far:
            cache.v_exp[:, :, ::5] += 60
        call = lambda x, **kw: fa8.flash_attn_fp8_shared_prefix(  # noqa: E731
            x, cache, table, seqlens, prefix, **kw)
        want = call(q)
        x = q.clone()
        assert call(x, out=x).data_ptr() == x.data_ptr() and torch.equal(x, want)
        room = torch.zeros(q.numel() + 4096, dtype=q.dtype, device="cuda")
        x = room[:q.numel()].view(q.shape).copy_(q)
        out = room[4096:].view(q.shape)
        call(x, out=out)
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("zeros", [128, 300, 1000])
@pytest.mark.parametrize("keys", ["zeros", "ordinary"])
@pytest.mark.parametrize("H,Hkv,Sq,D", [(8, 2, 1, 128), (16, 4, 3, 64), (40, 1, 1, 128)])
def test_sequences_that_begin_with_zeros(fa8, H, Hkv, Sq, D, keys, zeros, dtype):
    """Tokens whose values are zeros fill the first tiles: their own result is zero, and
    what follows is as precise as without them."""
    lens, ps = [zeros + 200, zeros, zeros + 3, zeros + 1500], 32
    pages = pages_for(lens, ps)
    cache = make_cache(fa8, pages, Hkv, ps, D, spread=0.3)
    table, seqlens = make_table(lens, ps, pages)
    for b in range(4):
        for col in range(-(-zeros // ps)):
            page, n = int(table[b, col]), min(ps, zeros - col * ps)
            u8(cache.v)[page, :, :n] = 0
            cache.v_exp[page, :, :n] = 127
            if keys == "zeros":
                u8(cache.k)[page, :, :n] = 0
                cache.k_exp[page, :, :n] = 127
    q = make_q(4, H, Sq, D, dtype)
    got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
    assert bool((got[0][1] == 0).all()) and bool(torch.isfinite(got[1]).all())
    assert_near(got, q, cache, table, lens)


def test_largest_value_of_bf16(fa8):
    """bf16's largest rounds to 2^128 as a code and a factor, more than fp32 holds: keys
    with such values count by their weights, whatever shares the work is cut into."""
    D, H, Hkv, ps, n = 128, 8, 2, 16, 9000
    top = torch.finfo(torch.bfloat16).max
    pages = pages_for([n], ps)
    cache = fa8.kv_cache_alloc(pages, Hkv, ps, D)
    table, seqlens = make_table([n], ps, pages)
    g = torch.Generator(device="cuda").manual_seed(4)
    k = torch.randn(1, Hkv, n, D, generator=g, device="cuda")
    v = torch.randn(1, Hkv, n, D, generator=g, device="cuda")
    v[:, :, 100:300] = top
    v[:, :, 5000:5010] = -top
    v[:, 0, 8000] = top
    fa8.kv_cache_write(cache, k.bfloat16(), v.bfloat16(), table, seqlens)
    assert bool((cache.v.float()[cache.v_exp == 247].amax(-1) == 256).any())
    for size in (0.1, 2.0):
        q = make_q(1, H, 1, D, "bf16", size=size)
        got = fa8.flash_attn_fp8_decode(q, cache, table, seqlens, return_lse=True)
        assert not bool(got[0].isnan().any()) and not bool(got[0].isinf().any())
        assert_near(got, q, cache, table, [n])
