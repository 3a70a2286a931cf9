"""What the cache and attention entry points refuse before anything is launched (no device needed), and the kernels'
own checks of block tables and row numbers, run on the host."""
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture()
def capi(built_libs):
    from distserve_b200 import capi

    return capi


def shape(capi, **kw):
    return capi.PoolShape.of(**{**dict(num_blocks=8, num_layers=2, num_heads=4, block_size=16, head_dim=64, elem_size=2), **kw})


def rows(capi, data=0x1000, heads=4, row=256, head=64):
    return capi.Rows(data, heads, row, head)


def batch(capi, **kw):
    return capi.Batch(**{**dict(num_seqs=2, num_rows=5, max_rows=3, starts=0x9000, seq_lens=0xA000, block_tables=0xB000,
                                table_stride=7, max_blocks=7), **kw})


def refused(capi, text, call, code=None):
    with pytest.raises(capi.KvmigError, match=text) as e:
        call()
    assert e.value.code == (capi.EINVAL if code is None else code)


def entry_points(capi):
    """Every entry point that takes pools, as a function of what may be wrong."""
    def write(s=None, b=None, r=None, dtype=0, layer=1, k=0x100000, v=0x200000):
        capi.cache_write(r or rows(capi), rows(capi), dtype, k, v, s or shape(capi), layer, b or batch(capi))

    def read(s=None, b=None, r=None, dtype=0, layer=1, k=0x100000, v=0x200000):
        capi.cache_read(k, v, s or shape(capi), layer, b or batch(capi), r or rows(capi), rows(capi), dtype)

    def paged(s=None, b=None, r=None, dtype=0, layer=1, k=0x100000, v=0x200000):
        capi.paged_attention(r or rows(capi), rows(capi), dtype, k, v, s or shape(capi), layer, b or batch(capi), 0.125, 0x4000, 1 << 30)

    return write, read, paged


@pytest.mark.parametrize("which", range(3))
def test_pools_rows_and_batches(capi, which):
    call = entry_points(capi)[which]
    refused(capi, "layer 2 is outside", lambda: call(layer=2))
    refused(capi, "layer -1 is outside", lambda: call(layer=-1))
    refused(capi, "unknown dtype", lambda: call(dtype=2))
    refused(capi, "pool pointer is NULL", lambda: call(v=0))
    refused(capi, "multiple of 16 bytes", lambda: call(k=0x100008))
    refused(capi, "not elements of 4 bytes", lambda: call(s=shape(capi, elem_size=4)))
    refused(capi, "head_dim 24 is not", lambda: call(s=shape(capi, head_dim=24)))
    refused(capi, "head_dim 272 is not", lambda: call(s=shape(capi, head_dim=272)))
    refused(capi, "head_dim 0 is not", lambda: call(s=shape(capi, head_dim=4, elem_size=1)))
    refused(capi, "head_dim 60 is not", lambda: call(s=shape(capi, head_dim=64, elem_size=1)))
    refused(capi, "not a multiple of 4", lambda: call(s=shape(capi, head_dim=68, elem_size=1, block_size=6)))
    refused(capi, "non-positive", lambda: call(s=shape(capi, block_size=0)))
    refused(capi, "more than 65536", lambda: call(s=shape(capi, block_size=1 << 17)), capi.ELIMIT)
    refused(capi, "address is NULL", lambda: call(r=rows(capi, data=0)))
    refused(capi, "multiple of 16 bytes", lambda: call(r=rows(capi, data=0x1002)))
    refused(capi, "multiples of 8", lambda: call(r=rows(capi, row=260)))
    refused(capi, "multiples of 8", lambda: call(r=rows(capi, head=-64)))
    refused(capi, "less than head_dim", lambda: call(r=rows(capi, head=56)))
    refused(capi, "0 heads", lambda: call(r=rows(capi, heads=0)))
    refused(capi, "negative count", lambda: call(b=batch(capi, num_rows=-1)))
    refused(capi, "negative count", lambda: call(b=batch(capi, num_seqs=-1)))
    refused(capi, "2\\^31-1", lambda: call(b=batch(capi, num_rows=1 << 31)), capi.ELIMIT)
    refused(capi, "starts or seq_lens is NULL", lambda: call(b=batch(capi, starts=0)))
    refused(capi, "less than max_blocks", lambda: call(b=batch(capi, table_stride=6)))
    refused(capi, "block_tables is NULL", lambda: call(b=batch(capi, block_tables=0)))


def test_heads_and_scales(capi):
    write, _, _ = entry_points(capi)
    refused(capi, "3 and 4 heads", lambda: write(r=rows(capi, heads=3)))
    q = lambda heads, **kw: rows(capi, heads=heads, **kw)  # noqa: E731

    def paged(qr, out, s=None, scale=0.125, ws=0x4000, n=1 << 30):
        capi.paged_attention(qr, out, 0, 0x100000, 0x200000, s or shape(capi), 0, batch(capi), scale, ws, n)

    refused(capi, "6 query heads do not split over 4", lambda: paged(q(6), q(6)))
    refused(capi, "q has 8 heads, out 4", lambda: paged(q(8), q(4)))
    for bad in (float("nan"), float("inf"), 1e39):
        refused(capi, "scale is not finite", lambda: paged(q(8), q(8), scale=bad))
    refused(capi, "neither 64 nor 128", lambda: paged(q(4, head=256), q(4, head=256), shape(capi, head_dim=256)))
    refused(capi, "neither 64 nor 128", lambda: paged(q(4, head=80), q(4, head=80), shape(capi, head_dim=80)))

    def prompt(qr, k, v, out, dim=64, scale=0.125, dtype=0, b=None):
        capi.prompt_attention(qr, k, v, out, dtype, dim, b or batch(capi), scale)

    refused(capi, "k has 4 heads, v 2", lambda: prompt(q(8), q(4), q(2), q(8)))
    refused(capi, "6 query heads do not split over 4", lambda: prompt(q(6), q(4), q(4), q(6)))
    refused(capi, "neither 64 nor 128", lambda: prompt(q(4), q(4), q(4), q(4), dim=32))
    refused(capi, "unknown dtype", lambda: prompt(q(4), q(4), q(4), q(4), dtype=7))
    refused(capi, "scale is not finite", lambda: prompt(q(4), q(4), q(4), q(4), scale=float("nan")))
    refused(capi, "starts or seq_lens", lambda: prompt(q(4), q(4), q(4), q(4), b=batch(capi, starts=0)))


def test_workspace_is_asked_for_and_checked(capi):
    s, b = shape(capi), batch(capi)
    n = capi.paged_attention_workspace(s, 8, b)
    assert n >= 0 and n == capi.paged_attention_workspace(s, 8, b)
    refused(capi, "do not split", lambda: capi.paged_attention_workspace(s, 6, b))
    refused(capi, "negative count", lambda: capi.paged_attention_workspace(s, 8, batch(capi, num_rows=-4)))


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU failure mode")
def test_without_a_device_every_call_fails_loudly(capi):
    for call in entry_points(capi):
        refused(capi, "cudaGetDevice", call, capi.ECUDA)
    r = rows(capi)
    refused(capi, "cudaGetDevice", lambda: capi.prompt_attention(r, r, r, r, 0, 64, batch(capi), 0.1), capi.ECUDA)


def test_operators_refuse_host_tensors_and_wrong_shapes(built_libs):
    import distserve_b200

    distserve_b200.load_ops()
    k, pool = torch.zeros(3, 2, 64, dtype=torch.float16), torch.zeros(4, 1, 2, 16, 64, dtype=torch.float16)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        torch.ops.kv_cache_ops.write(k, k, pool, pool.clone(), 0, ints(0)[None], ints(3), ints(0, 3))
    with pytest.raises(RuntimeError, match="float16 or bfloat16"):
        torch.ops.kv_cache_ops.read(pool, pool.clone(), 0, ints(0)[None], ints(0, 3), k.float(), k.float())
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.ops.kv_attention_ops.paged(k.clone().requires_grad_(), pool, pool, 0, ints(0)[None], ints(3), ints(0, 3), 3, 0.1, k)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        torch.ops.kv_attention_ops.prompt(k, k, k, ints(0, 3), 3, 0.1, k.clone())


@pytest.mark.gpu
def test_operators_refuse_what_does_not_fit(built_libs):
    import distserve_b200

    distserve_b200.load_ops()
    dev = dict(device="cuda")
    pool = lambda **kw: torch.zeros(4, 1, 2, 16, 64, dtype=kw.get("dtype", torch.float16), **dev)  # noqa: E731
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, **dev)  # noqa: E731
    q, out = torch.zeros(3, 4, 64, dtype=torch.float16, **dev), torch.zeros(3, 4, 64, dtype=torch.float16, **dev)
    good = dict(q=q, k_cache=pool(), v_cache=pool(), layer=0, block_tables=ints(0)[None], seq_lens=ints(3), starts=ints(0, 3), max_rows=3,
                scale=0.1, out=out)
    torch.ops.kv_attention_ops.paged(**good)
    for text, change in {
        "differ in shape": dict(out=out[:2]),
        "differs in dtype": dict(out=out.bfloat16()),
        "must be contiguous": dict(k_cache=torch.zeros(4, 1, 16, 2, 64, dtype=torch.float16, **dev).transpose(2, 3)),
        "do not hold rows": dict(k_cache=pool(dtype=torch.bfloat16), v_cache=pool(dtype=torch.bfloat16)),
        "4 bytes more": dict(k_cache=pool(dtype=torch.uint8), v_cache=pool(dtype=torch.uint8)),
        "must be int32": dict(seq_lens=ints(3).long()),
        "another device": dict(block_tables=torch.zeros(1, 1, dtype=torch.int32)),
        "entries for 1 sequences": dict(seq_lens=ints(3, 3)),
        "rows for 1 sequences": dict(block_tables=ints(0, 0)[:, None]),
        "dimension": dict(starts=ints(0, 3)[None]),
        "overlap|memory": dict(out=q),
        "single memory location": dict(out=q[:1].expand(3, 4, 64)),
        "is outside": dict(layer=1),
        "scale": dict(scale=float("inf")),
        "values of a head": dict(q=torch.zeros(3, 64, 4, dtype=torch.float16, **dev).transpose(1, 2)),
        "multiples of 8": dict(q=torch.zeros(3, 4, 68, dtype=torch.float16, **dev)[:, :, :64]),
        "multiple of 16 bytes": dict(q=torch.zeros(3 * 4 * 64 + 8, dtype=torch.float16, **dev)[4:4 + 768].view(3, 4, 64)),
        "negative count": dict(max_rows=-1),
    }.items():
        with pytest.raises(RuntimeError, match=text):
            torch.ops.kv_attention_ops.paged(**{**good, **change})
    torch.cuda.synchronize()
    # nothing to do is not an error
    empty = q[:0]
    torch.ops.kv_attention_ops.paged(**{**good, "q": empty, "out": out[:0], "starts": ints(0, 0), "max_rows": 0})
    torch.ops.kv_attention_ops.paged(**{**good, "starts": ints(0), "seq_lens": ints(0)[:0], "block_tables": ints(0)[None][:0]})
    torch.cuda.synchronize()
    assert (out == 0).all()


HOST_CHECK = r"""
#include <cassert>
#include <climits>
#include <cstdio>
#include "kvcache_device.cuh"
using namespace kvmig;
int main() {
    const int tables[2][4] = {{5, 9, 10, -1}, {INT_MIN, INT_MAX, 0, 3}}, starts[] = {0, 4, 2, 9, -1, 3};
    CacheView c = {};
    c.num_blocks = 10;
    c.block_size = 16;
    BatchView b = {starts, nullptr, &tables[0][0], 4, 5, 8, 8, 3};
    assert(block_of(b, c, 0, 0) == 5 && block_of(b, c, 0, 15) == 5 && block_of(b, c, 0, 16) == 9 && block_of(b, c, 0, 31) == 9);
    assert(block_of(b, c, 0, 32) == -1);                 // id 10 of 10 blocks
    assert(block_of(b, c, 0, 48) == -1 && block_of(b, c, 0, INT_MAX) == -1);   // past max_blocks: the table is not read
    assert(block_of(b, c, 1, 0) == -1 && block_of(b, c, 1, 17) == -1 && block_of(b, c, 1, 47) == 0);
    assert(sequence_at(b, 0).valid && sequence_at(b, 0).rows == 4);
    assert(!sequence_at(b, 1).valid && sequence_at(b, 1).rows == 0);           // runs backwards
    assert(!sequence_at(b, 2).valid && !sequence_at(b, 3).valid && !sequence_at(b, 4).valid);
    b.max_blocks = 0;
    assert(block_of(b, c, 0, 0) == -1);
    std::puts("ok");
}
"""


def test_the_kernels_own_checks_on_the_host(tmp_path):
    """Block ids and row numbers come from device memory, so the kernels check them; the same functions, on the host."""
    from distserve_b200.build import _nvcc

    src, exe = tmp_path / "check.cu", tmp_path / "check"
    src.write_text(HOST_CHECK)
    subprocess.run([_nvcc(), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", str(ROOT / "distserve_b200" / "csrc"), "-o", str(exe), str(src)],
                   check=True, capture_output=True, timeout=300)
    assert subprocess.run([str(exe)], capture_output=True, text=True, timeout=60).stdout == "ok\n"
