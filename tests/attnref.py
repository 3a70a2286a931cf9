"""Plain restatement, in 64 bits on the host, of the cache and attention operators, and the inputs of their tests.

Pools are filled so that whatever a correct operator must not use is NaN: slots behind a sequence's last token, blocks
that no table names, the other layers."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
SCALE_BYTES = 4


def quantise(x: torch.Tensor):
    """Rows of x -> (code values, scales), both in 64 bits: scale the smallest 2**e, e >= -100, with max|row| <= 448 * 2**e;
    codes to nearest, ties to even, in steps of 2**-3 of their binade and of 2**-9 below 2**-6."""
    x = x.double()
    top = x.abs().amax(-1)
    scale = torch.ones_like(top)
    for i, t in enumerate(top.flatten().tolist()):
        if not math.isfinite(t):
            s = math.nan
        elif t == 0:
            s = 1.0
        else:
            e = math.frexp(t / 448.0)[1]                       # t / 448 in [2**(e-1), 2**e)
            while e > -100 and t <= 448.0 * 2.0 ** (e - 1):
                e -= 1
            s = 2.0 ** max(e, -100)
        scale.view(-1)[i] = s
    y = x / scale[..., None]
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, scale


def codes_of(values: torch.Tensor) -> torch.Tensor:
    """e4m3 code values (exact) as bytes."""
    return values.to(torch.float32).to(torch.float8_e4m3fn).view(torch.uint8)


def split_pool(pool: torch.Tensor):
    """A quantised pool's codes [.., block_size, head_dim] (bytes) and scales [.., block_size] (32-bit), as views."""
    nb, layers, heads, bs, width = pool.shape
    flat = pool.view(nb, layers, heads, bs * width)
    return flat[..., :bs * (width - 4)].unflatten(-1, (bs, width - 4)), flat[..., bs * (width - 4):].view(torch.float32)


def pool_values(pool: torch.Tensor) -> torch.Tensor:
    """What a pool stands for, in 64 bits."""
    if pool.dtype != torch.uint8:
        return pool.double()
    codes, scales = split_pool(pool)
    return codes.contiguous().view(torch.float8_e4m3fn).double() * scales.double()[..., None]


@dataclass
class Paged:
    """A batch over a pool pair, on the host."""

    k_cache: torch.Tensor
    v_cache: torch.Tensor
    tables: torch.Tensor
    lens: torch.Tensor
    starts: torch.Tensor
    layer: int
    new: List[int]
    ctx: List[int]

    def to(self, device) -> "Paged":
        t = lambda x: x.to(device)  # noqa: E731
        return Paged(t(self.k_cache), t(self.v_cache), t(self.tables), t(self.lens), t(self.starts), self.layer, self.new, self.ctx)


def ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32)


def starts_of(new: Sequence[int], first: int = 0) -> torch.Tensor:
    out = [first]
    for n in new:
        out.append(out[-1] + n)
    return ints(out)


def make_paged(seed: int, new: Sequence[int], ctx: Sequence[int], kv_heads: int, dim: int, block: int, dtype: str, e4m3: bool,
               layers: int = 2, layer: int = 1, spare: int = 3, magnitude: float = 1.0, first_row: int = 0) -> Paged:
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(new, ctx)]
    need = [-(-n // block) for n in lens]
    blocks = sum(need) + spare
    ids = torch.randperm(blocks, generator=g).tolist()
    tables = torch.full((len(new), max(need + [1]) + 1), -7, dtype=torch.int32)       # entries behind the last block: no block
    pools = []
    for _ in range(2):
        width = dim + (SCALE_BYTES if e4m3 else 0)
        if e4m3:
            pool = torch.full((blocks, layers, kv_heads, block, width), 0x7F, dtype=torch.uint8)
            split_pool(pool)[1].fill_(math.nan)
        else:
            pool = torch.full((blocks, layers, kv_heads, block, width), math.nan, dtype=DTYPES[dtype])
        at = 0
        for i, n in enumerate(lens):
            rows = (torch.randn(n, kv_heads, dim, generator=g) * magnitude).to(DTYPES[dtype])
            for b in range(need[i]):
                tables[i, b] = ids[at]
                part = rows[b * block:(b + 1) * block].transpose(0, 1)              # [heads, tokens, dim]
                if e4m3:
                    values, scales = quantise(part)
                    codes, sc = split_pool(pool)
                    codes[ids[at], layer, :, :part.shape[1]] = codes_of(values)
                    sc[ids[at], layer, :, :part.shape[1]] = scales.float()
                else:
                    pool[ids[at], layer, :, :part.shape[1]] = part
                at += 1
        pools.append(pool)
    return Paged(pools[0], pools[1], tables, ints(lens), starts_of(new, first_row), layer, list(new), list(ctx))


def rows_of(p: Paged, pool: torch.Tensor, i: int, count: Optional[int] = None) -> torch.Tensor:
    """The first tokens of sequence i, [count, heads, dim], in 64 bits."""
    n = int(p.lens[i]) if count is None else count
    bs = pool.shape[3]
    used = pool[p.tables[i, :-(-n // bs)].long()]
    return pool_values(used)[:, p.layer].transpose(1, 2).flatten(0, 1)[:n]


@dataclass
class Expected:
    out: torch.Tensor
    tol: torch.Tensor       # how far each value may be off


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, dtype: str, quantised: bool = False) -> Expected:
    """q [Q, heads, D] at the last Q positions of k, v [S, kv_heads, D].

    The bound, per output, with h = eps / 2 of the 16-bit type and A = sum_j p_j |v_j|:
      h A                probabilities rounded to 16 bits before the second product
      h |o|              the same roundings where they enter the sum of the probabilities
      h |o|              the result's own rounding (plus half the type's smallest step)
      2**-23 |v| summed  where probabilities are rounded to fp16 (fp16 rows, and few rows over a quantised pool, whose e4m3
                         codes widen to fp16): below 2**-14 they are rounded absolutely, by 2**-25 at most, and the sum
                         that divides them is at least 1/2; over a quantised pool P_j carries V's scale s_j, so that
                         the 2**-25 count 2**-25 |v_j| s_max / s_j, and s_max / s_j is at most 2 for rows drawn from one
                         normal distribution (their largest magnitudes are within a factor of 2, or next to it)
      A 2**-24 (2 E + n + 64)   32-bit sums over n keys, exponentials, and scores that are off by at most
                         E = (D + 2) scale sum |q k| units of 2**-24, numerator and denominator alike
    """
    rows, heads, dim = q.shape
    group, first = heads // k.shape[1], k.shape[0] - rows
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    qd = q.double()
    hidden = torch.arange(k.shape[0]) > torch.arange(rows)[:, None] + first
    score = scale * torch.einsum("qhd,shd->hqs", qd, kk)
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True) if k.shape[0] else torch.zeros(heads, rows, 1, dtype=torch.float64)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    p = torch.where(torch.isfinite(score), p, torch.zeros_like(p))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.einsum("hqs,shd->qhd", p, vv)
    h = torch.finfo(DTYPES[dtype]).eps / 2
    big = torch.einsum("hqs,shd->qhd", p, vv.abs())
    visible = (~hidden).double()[None].expand(heads, -1, -1)
    absolute = 2.0 ** -23 * torch.einsum("hqs,shd->qhd", visible, vv.abs()) if dtype == "fp16" or quantised else 0.0
    size = abs(scale) * torch.einsum("qhd,shd->hqs", qd.abs(), kk.abs())
    size = (size * visible).amax(-1).transpose(0, 1)[..., None] if k.shape[0] else 0.0
    tol = h * (big + 2 * out.abs()) + absolute + big * 2.0 ** -24 * (2 * (dim + 2) * size + k.shape[0] + 64)
    return Expected(out, tol * 1.01 + torch.finfo(DTYPES[dtype]).tiny * torch.finfo(DTYPES[dtype]).eps)


def attend_paged(p: Paged, q: torch.Tensor, scale: float, dtype: str) -> List[Expected]:
    return [attend(q[a:b], rows_of(p, p.k_cache, i), rows_of(p, p.v_cache, i), scale, dtype, p.k_cache.dtype == torch.uint8)
            for i, (a, b) in enumerate(zip(p.starts.tolist(), p.starts.tolist()[1:]))]


def assert_close(got: torch.Tensor, want: Expected, what: str) -> None:
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want.out).abs()
    worst = (off / want.tol).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.2f} times its bound off (largest difference {off.max().item():.3g})"
