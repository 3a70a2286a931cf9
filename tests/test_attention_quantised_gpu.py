"""Attention over quantised pools whose V rows differ in size: rows of zeros that draw most of the attention, and scales far
apart.  Against a plain computation in 64 bits, within a bound that assumes nothing about the scales."""
import dataclasses
import functools
import math

import pytest
import torch

from tests import attnref as R

pytestmark = pytest.mark.gpu

ZERO_ROW = 2.0 ** -64       # the scale that a V row of zeros counts with where rows are few (stored: 1)


@pytest.fixture(scope="module", autouse=True)
def _ops(built_libs):
    import distserve_b200

    distserve_b200.load_ops()


def put(pool, p, i, position, rows):
    """Rows [heads, dim] at one position of sequence i."""
    block = pool.shape[3]
    codes, scales = R.split_pool(pool)
    values, scale = R.quantise(rows)
    at = p.tables[i, position // block].long()
    codes[at, p.layer, :, position % block] = R.codes_of(values)
    scales[at, p.layer, :, position % block] = scale.float()


def fill(p, i, rows):
    """V rows [tokens, heads, dim] of sequence i from its first token on."""
    block = p.v_cache.shape[3]
    codes, scales = R.split_pool(p.v_cache)
    values, scale = R.quantise(rows)
    at, offset = p.tables[i, torch.arange(len(rows)) // block].long(), torch.arange(len(rows)) % block
    codes[at, p.layer, :, offset] = R.codes_of(values)
    scales[at, p.layer, :, offset] = scale.float()


def expected(p, i, q, scale, dtype, few):
    """`attnref.attend` with the bound's terms for probabilities replaced.  Where rows are few (`few`), with s_j the scale of V's
    row j (2**-64 for a row of zeros) and c_j its codes, P_j = 2**15 s_j p_j / max_k(s_k p_k) is rounded to fp16:
      2**-11 A           to eleven bits where it is normal
      2**-40 sum_j |c_j| max_k s_k
                         by 2**-25 at most where it is not: 2**-40 of what P_j is divided by, and the sum that divides the
                         output, sum_j P_j / s_j, is at least 2**15 / max_k s_k
      the exponents carry log2 s_j: 2 * 2**-24 (3 max|log2 s| + 16) more from rounding them to 32 bits, in numerator and sum.
    Otherwise V is widened with its scale (exactly) and P_j is rounded to the rows' type as over 16-bit pools."""
    k, v = R.rows_of(p, p.k_cache, i), R.rows_of(p, p.v_cache, i)
    base = R.attend(q, k, v, scale, dtype, False)
    if not few:
        return base
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    _, s = R.split_pool(p.v_cache[p.tables[i, :-(-k.shape[0] // p.v_cache.shape[3])].long()])
    s = s[:, p.layer].transpose(1, 2).flatten(0, 1)[:k.shape[0]].double()
    s = torch.where(v.abs().amax(-1) == 0, torch.full_like(s, ZERO_ROW), s)          # [keys, kv heads]
    first = k.shape[0] - rows
    hidden = torch.arange(k.shape[0]) > torch.arange(rows)[:, None] + first
    score = scale * torch.einsum("qhd,shd->hqs", q.double(), k.repeat_interleave(group, 1))
    p_ = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
    vv = v.repeat_interleave(group, 1)
    big = torch.einsum("hqs,shd->qhd", p_, vv.abs())
    visible = (~hidden).double()[None].expand(heads, -1, -1)
    per_scale = torch.einsum("hqs,shd->qhd", visible, (v.abs() / s[..., None]).repeat_interleave(group, 1))
    s_max = s.amax(0).repeat_interleave(group)[None, :, None]
    size = (abs(scale) * torch.einsum("qhd,shd->hqs", q.double().abs(), k.repeat_interleave(group, 1).abs()) * visible).amax(-1).transpose(0, 1)[..., None]
    h = torch.finfo(R.DTYPES[dtype]).eps / 2
    lift = float(s.log2().abs().max())
    tol = 2.0 ** -11 * big + h * base.out.abs() + 2.0 ** -40 * per_scale * s_max \
        + big * 2.0 ** -24 * (2 * (dim + 2) * size + k.shape[0] + 64 + 2 * (3 * lift + 16))
    return R.Expected(base.out, tol * 1.01 + torch.finfo(R.DTYPES[dtype]).tiny * torch.finfo(R.DTYPES[dtype]).eps)


def run(p, q, scale):
    d = p.to("cuda")
    out = torch.full_like(q, 7.0, device="cuda")
    torch.ops.kv_attention_ops.paged(q.cuda(), d.k_cache, d.v_cache, d.layer, d.tables, d.lens, d.starts, max(p.new), scale, out)
    return out.cpu()


def check(p, q, scale, dtype, few, what):
    out, starts = run(p, q, scale), p.starts.tolist()
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        R.assert_close(out[a:b], expected(p, i, q[a:b], scale, dtype, few), f"{what} sequence {i}")


def heavy_key(p, i, position, weight, scale):
    """Sets K at a position so that it draws about `weight` of the attention of queries of ones: small integers, exact in e4m3."""
    k = R.rows_of(p, p.k_cache, i)
    dim = k.shape[2]
    others = scale * k.sum(-1)
    others = torch.cat([others[:position], others[position + 1:]])
    target = torch.logsumexp(others, 0) + math.log(weight / (1 - weight))
    rows = torch.zeros(k.shape[1], dim, dtype=torch.float64)
    for h in range(k.shape[1]):
        total = round(float(target[h]) / scale)
        rows[h] = total // dim
        rows[h, :total % dim] += 1
    put(p.k_cache, p, i, position, rows)
    score = scale * R.rows_of(p, p.k_cache, i).sum(-1)
    got = torch.softmax(score, 0)[position]
    assert ((got / (1 - got) / (weight / (1 - weight))).log().abs() < 0.1).all()


@functools.lru_cache(maxsize=None)
def pools(dim, keys, magnitude):
    """A sequence whose V rows have this size, but for a row of zeros at position 3."""
    p = R.make_paged(31, [1], [keys - 1], 2, dim, 16, "bf16", True)
    v = (torch.randn(keys, 2, dim, generator=torch.Generator().manual_seed(5)) * magnitude).to(torch.bfloat16)
    fill(p, 0, v)
    put(p.v_cache, p, 0, 3, torch.zeros(2, dim))
    return p


@pytest.mark.parametrize("weight", [0.5, 0.98, 0.9996])
@pytest.mark.parametrize("magnitude", [1.0, 0.05, 0.02, 1e-4, 1e-6, 1e-20])
@pytest.mark.parametrize("keys,dim", [(500, 64), (500, 128), (5000, 128)])
def test_a_row_of_zeros_that_draws_the_attention(keys, dim, magnitude, weight):
    """A sink, or padding stored as zeros: few rows and many, keys in one part and in several."""
    base = pools(dim, keys, magnitude)
    for new, heads in ((1, 2), (1, 16), (5, 2), (20, 2), (140, 2)):
        p = dataclasses.replace(base, new=[new], ctx=[keys - new], starts=R.starts_of([new]), k_cache=base.k_cache.clone())
        heavy_key(p, 0, 3, weight, dim ** -0.5)
        check(p, torch.ones(new, heads, dim, dtype=torch.bfloat16), dim ** -0.5, "bf16", new * heads // 2 <= 64, f"{new} rows, {heads} heads")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new", [1, 5, 40])
def test_only_rows_of_zeros_and_rows_of_negative_zeros(new, dtype):
    p = R.make_paged(33, [new, new], [100, 30], 2, 64, 16, dtype, True)
    for i, n in enumerate(p.lens.tolist()):
        for t in range(n):
            if i == 0 or t % 2:
                put(p.v_cache, p, i, t, torch.zeros(2, 64) if t % 3 else -torch.zeros(2, 64))
    g = torch.Generator().manual_seed(4)
    q = torch.randn(2 * new, 4, 64, generator=g).to(R.DTYPES[dtype])
    out = run(p, q, 0.125)
    assert (out[:new] == 0).all()
    R.assert_close(out[new:], expected(p, 1, q[new:], 0.125, dtype, 2 * new <= 64), "every other row zeros")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new,heads", [(1, 2), (1, 8), (7, 4), (100, 2)])
@pytest.mark.parametrize("ratio", [2.0 ** -13, 2.0 ** 13])
def test_scales_far_apart(ratio, new, heads, dtype):
    """One V row in eight is 2**13 smaller, or larger, than the others; the smaller ones draw the attention."""
    dim, keys = 128, 900
    p = R.make_paged(35, [new], [keys - new], 2, dim, 16, dtype, True)
    g = torch.Generator().manual_seed(6)
    size = torch.where(torch.arange(keys) % 8 == 5, ratio, 1.0)[:, None, None] * 2.0 ** -6
    fill(p, 0, (torch.randn(keys, 2, dim, generator=g) * size).to(R.DTYPES[dtype]))
    q = torch.ones(new, heads, dim, dtype=R.DTYPES[dtype])
    heavy_key(p, 0, 13 if ratio < 1 else 12, 0.98, dim ** -0.5)
    check(p, q, dim ** -0.5, dtype, new * heads // 2 <= 64, "")


@pytest.mark.parametrize("magnitudes", [(2.0 ** 40, 2.0 ** -40), (2.0 ** 100, 2.0 ** 20), (2.0 ** -30, 2.0 ** -85)], ids=str)
def test_bf16_rows_of_very_different_sizes(magnitudes):
    p = R.make_paged(36, [1, 5], [300, 700], 2, 64, 16, "bf16", True)
    g = torch.Generator().manual_seed(7)
    for i, n in enumerate(p.lens.tolist()):
        size = torch.where(torch.arange(n) % 2 == 0, *magnitudes).double()[:, None, None]
        fill(p, i, (torch.randn(n, 2, 64, generator=g, dtype=torch.float64) * size).to(torch.bfloat16))
    q = torch.randn(6, 4, 64, generator=g).to(torch.bfloat16)
    check(p, q, 0.125, "bf16", True, "")
