"""GPU checks of the cache's attention where it can go wrong: calls whose waits run
out beside calls of another stream.

Helpers, oracle and the tolerances of plain cases are those of test_kv_cache_gpu.
"""

import pytest

from tests.test_kv_cache_gpu import (make_cache, make_q, make_table, pages_for)

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa8(cuda):
    import ada_cute_fp8_flash_attention_b200 as m
    return m


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
