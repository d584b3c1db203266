"""CPU checks of the cache and decode entry points: struct mirrors, defaults and
the host's refusals, which come before any device access; and the oracle's
quantiser against torch's own e4m3 cast."""
from __future__ import annotations

import ctypes as C
import math
import subprocess
from pathlib import Path

import pytest
import torch

from oracle import attention_ref, kv_cache_ref as ref

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def abi():
    from ada_cute_fp8_flash_attention_b200 import c_abi
    return c_abi


@pytest.mark.parametrize("name", ["fa8_kv_cache", "fa8_kv_copy_params", "fa8_decode_params"])
def test_struct_layout_matches_c(abi, tmp_path, name):
    cls = {"fa8_kv_cache": abi.Fa8KvCache, "fa8_kv_copy_params": abi.Fa8KvCopyParams,
           "fa8_decode_params": abi.Fa8DecodeParams}[name]
    fields = [f[0] for f in cls._fields_]
    body = "\n".join(f'  printf("{f} %zu\\n", offsetof({name}, {f}));' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "fa8.h"\nint main(void){{\n'
                   f'  printf("size %zu\\n", sizeof({name}));\n{body}\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True).stdout
    lines = dict(line.split() for line in out.splitlines())
    assert int(lines["size"]) == C.sizeof(cls)
    for f in fields:
        assert int(lines[f]) == getattr(cls, f).offset, f


def _copy(abi):
    p = abi.kv_copy_params(10, 4, 16, 128, 2, 5)
    c = p.cache
    c.k = c.v = c.k_exp = c.v_exp = c.page_table = c.seqlens = 0x100000  # never dereferenced
    p.k = p.v = 0x200000
    p.tokens = 3
    p.k_stride_s = p.v_stride_s = 128
    p.k_stride_h = p.v_stride_h = 384
    p.k_stride_b = p.v_stride_b = 4 * 384
    return p


def _decode(abi):
    p = abi.decode_params(10, 4, 16, 128, 2, 5, 8, 1)
    c = p.cache
    c.k = c.v = c.k_exp = c.v_exp = c.page_table = c.seqlens = 0x100000
    p.q = p.o = 0x200000
    return p


def _set(**kw):
    def mutate(p):
        for name, value in kw.items():
            target = p.cache if name.startswith("c_") else p
            setattr(target, name[2:] if name.startswith("c_") else name, value)
    return mutate


CACHE_REFUSALS = [
    (_set(c_head_dim=96), "FA8_ERR_UNSUPPORTED"),
    (_set(c_page_size=48), "FA8_ERR_UNSUPPORTED"),
    (_set(c_page_size=0), "FA8_ERR_UNSUPPORTED"),
    (_set(c_page_size=192), "FA8_ERR_UNSUPPORTED"),
    (_set(c_heads_kv=0), "FA8_ERR_INVALID_ARG"),
    (_set(c_num_pages=-1), "FA8_ERR_INVALID_ARG"),
    (_set(c_num_pages=1 << 31), "FA8_ERR_UNSUPPORTED"),
    (_set(c_max_pages=1 << 27), "FA8_ERR_UNSUPPORTED"),
    (_set(c_batch=-1), "FA8_ERR_INVALID_ARG"),
    (_set(c_batch=65536), "FA8_ERR_UNSUPPORTED"),
    (_set(c_k=None), "FA8_ERR_INVALID_ARG"),
    (_set(c_v_exp=None), "FA8_ERR_INVALID_ARG"),
    (_set(c_seqlens=None), "FA8_ERR_INVALID_ARG"),
    (_set(c_page_table=None), "FA8_ERR_INVALID_ARG"),
    (_set(c_table_stride=-5), "FA8_ERR_INVALID_ARG"),
    (_set(c_v=0x100008), "FA8_ERR_ALIGNMENT"),
    (_set(c_seqlens=0x100002), "FA8_ERR_ALIGNMENT"),
    (_set(c_k_stride_s=136), "FA8_ERR_ALIGNMENT"),
    (_set(c_v_stride_p=0), "FA8_ERR_ALIGNMENT"),
    (_set(c_k_stride_s=64), "FA8_ERR_INVALID_ARG"),
    (_set(c_v_exp_stride_h=0), "FA8_ERR_INVALID_ARG"),
    (_set(c_k_exp=0x100008), "FA8_ERR_ALIGNMENT"),
    (_set(c_v_exp_stride_p=72), "FA8_ERR_ALIGNMENT"),
]


@pytest.mark.parametrize("mutate,status", CACHE_REFUSALS + [
    (_set(tokens=-1), "FA8_ERR_INVALID_ARG"),
    (_set(tokens=(1 << 30) + 1), "FA8_ERR_UNSUPPORTED"),
    (_set(dtype=2), "FA8_ERR_INVALID_ARG"),
    (_set(k=None), "FA8_ERR_INVALID_ARG"),
    (_set(v=0x200008), "FA8_ERR_ALIGNMENT"),
    (_set(cu_seqlens=0x300001), "FA8_ERR_ALIGNMENT"),
    (_set(k_stride_h=388), "FA8_ERR_ALIGNMENT"),
    (_set(v_stride_b=-8), "FA8_ERR_ALIGNMENT"),
])
@pytest.mark.parametrize("call", ["kv_write", "kv_read"])
def test_copy_refusals(abi, call, mutate, status):
    p = _copy(abi)
    mutate(p)
    assert getattr(abi, call)(p) == getattr(abi, status)
    assert abi.lib().fa8_last_error_message()


@pytest.mark.parametrize("mutate,status", CACHE_REFUSALS + [
    (_set(heads=6), "FA8_ERR_UNSUPPORTED"),
    (_set(heads=-4), "FA8_ERR_INVALID_ARG"),
    (_set(heads=65536), "FA8_ERR_UNSUPPORTED"),
    (_set(seqlen_q=-1), "FA8_ERR_INVALID_ARG"),
    (_set(seqlen_q=65536), "FA8_ERR_UNSUPPORTED"),
    (_set(prefix_len=-1), "FA8_ERR_INVALID_ARG"),
    (_set(prefix_len=81), "FA8_ERR_INVALID_ARG"),
    (_set(c_max_pages=1 << 25, c_batch=4096), "FA8_ERR_UNSUPPORTED"),  # 2^31 key tiles
    (_set(softmax_scale=0.0), "FA8_ERR_INVALID_ARG"),
    (_set(softmax_scale=math.inf), "FA8_ERR_INVALID_ARG"),
    (_set(dtype=3), "FA8_ERR_INVALID_ARG"),
    (_set(q=None), "FA8_ERR_INVALID_ARG"),
    (_set(o=0x200004), "FA8_ERR_ALIGNMENT"),
    (_set(lse=0x200002), "FA8_ERR_ALIGNMENT"),
    (_set(q_stride_h=132), "FA8_ERR_ALIGNMENT"),
    (_set(o_stride_b=-1024), "FA8_ERR_ALIGNMENT"),
])
def test_decode_refusals(abi, mutate, status):
    p = _decode(abi)
    mutate(p)
    ws = max(0, abi.decode_workspace_size(p))
    assert abi.decode(p, 0x400000, ws) == getattr(abi, status)
    assert abi.lib().fa8_last_error_message()


@pytest.mark.parametrize("field", ["batch", "tokens"])
def test_empty_copy_is_a_no_op(abi, field):
    p = _copy(abi)
    setattr(p.cache if field == "batch" else p, field, 0)
    assert abi.kv_write(p) == abi.FA8_OK and abi.kv_read(p) == abi.FA8_OK


@pytest.mark.parametrize("field", ["batch", "heads", "seqlen_q"])
def test_empty_decode_is_a_no_op(abi, field):
    p = _decode(abi)
    setattr(p.cache if field == "batch" else p, field, 0)
    assert abi.decode(p, 0, 0) == abi.FA8_OK


def test_defaults(abi):
    p = abi.decode_params(10, 4, 16, 128, 2, 5, 8, 3)
    c = p.cache
    assert (c.k_stride_s, c.k_stride_h, c.k_stride_p) == (128, 16 * 128, 4 * 16 * 128)
    assert (c.v_exp_stride_h, c.v_exp_stride_p, c.table_stride) == (16, 64, 5)
    assert (p.q_stride_s, p.o_stride_h, p.q_stride_b) == (128, 3 * 128, 8 * 3 * 128)
    assert abs(p.softmax_scale - 128 ** -0.5) < 1e-7 and p.prefix_len == 0


def test_torch_layer_refuses_host_tensors():
    import ada_cute_fp8_flash_attention_b200 as fa8
    cache = fa8.kv_cache_alloc(4, 2, 16, 64, device="cpu")
    assert cache.k.shape == (4, 2, 16, 64) and cache.k.dtype == torch.float8_e4m3fn
    assert int(cache.v_exp.min()) == 127
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    x = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError):
        fa8.kv_cache_write(cache, x, x, table, lens)
    with pytest.raises(RuntimeError):
        fa8.kv_cache_read(cache, table, lens, None, 1)
    with pytest.raises(RuntimeError):
        fa8.flash_attn_fp8_decode(x, cache, table, lens)


def test_oracle_quantiser():
    codes = torch.arange(256, dtype=torch.uint8)
    want = torch.from_numpy(attention_ref.e4m3_decode(codes.numpy())).double()
    got = ref.decode_e4m3(codes)
    assert torch.equal(got[~got.isnan()], want[~want.isnan()])
    assert torch.equal(got.isnan(), want.isnan())
    x = torch.randn(200, 64, dtype=torch.float64).to(torch.bfloat16)
    values, byte = ref.quantise(x)
    f = ref.factor(byte).unsqueeze(-1)
    assert float(values.abs().max()) <= 448
    # the least power of two: half of it would leave the largest magnitude above 448
    assert bool((x.double().abs().amax(-1) > 224 * f.squeeze(-1)).all())
    assert torch.equal((x.double() / f).float().to(torch.float8_e4m3fn).double(), values)
    # a rounding is off by at most half a step: 2^-4 of the value, 2^-10 below 2^-6
    bound = torch.maximum(values.abs() * 2.0 ** -4, torch.full_like(values, 2.0 ** -10))
    assert bool(((x.double() / f - values).abs() <= bound).all())
