"""Writing tokens into the paged pools and reading them back: bit for bit what the definition says, with nothing else
in the pools touched."""
import math

import pytest
import torch

from tests import attnref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _ops(built_libs):
    import distserve_b200

    distserve_b200.load_ops()


def bits(t):
    return t.contiguous().view(torch.uint8)


def write_on_host(p, k, v):
    """The pools after the write, on the host."""
    out = []
    for rows, pool in ((k, p.k_cache), (v, p.v_cache)):
        pool = pool.clone()
        bs, starts = pool.shape[3], p.starts.tolist()
        for i, (a, b) in enumerate(zip(starts, starts[1:])):
            for t in range(a, b):
                pos = int(p.lens[i]) - (b - a) + t - a
                if pos < 0 or pos // bs >= p.tables.shape[1] or not 0 <= int(p.tables[i, pos // bs]) < pool.shape[0]:
                    continue
                blk = int(p.tables[i, pos // bs])
                if pool.dtype == torch.uint8:
                    values, scales = R.quantise(rows[t])
                    codes, sc = R.split_pool(pool)
                    bad = torch.isnan(scales)
                    codes[blk, p.layer, :, pos % bs] = torch.where(bad[:, None], codes[blk, p.layer, :, pos % bs], R.codes_of(torch.nan_to_num(values)))
                    sc[blk, p.layer, :, pos % bs] = scales.float()
                else:
                    pool[blk, p.layer, :, pos % bs] = rows[t]
        out.append(pool)
    return out


def same_pool(got, want):
    """Equal bits, but for the codes of rows whose scale is NaN and NaN scales' own payload."""
    if got.dtype != torch.uint8:
        return torch.equal(bits(got), bits(want))
    (gc, gs), (wc, ws) = R.split_pool(got.cpu()), R.split_pool(want)
    nan = torch.isnan(ws)
    return torch.equal(torch.isnan(gs), nan) and torch.equal(gs[~nan], ws[~nan]) and torch.equal(gc[~nan], wc[~nan])


CASES = [
    # new, ctx, heads, head_dim, block
    ([1], [0], 1, 64, 16),
    ([1, 1, 1], [0, 15, 16], 3, 128, 16),
    ([5, 0, 33, 1], [0, 4, 31, 100], 2, 80, 16),
    ([7, 2], [3, 0], 5, 16, 4),
    ([3] * 40, [2] * 40, 1, 256, 8),                # more than 32 sequences: the search takes two steps
    ([1] * 1100, [0] * 1100, 1, 16, 4),             # and three
    ([300], [77], 12, 64, 64),
]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_write_and_read_back(case, e4m3, dtype):
    new, ctx, heads, dim, block = CASES[case]
    p = R.make_paged(case, new, ctx, heads, dim, block, dtype, e4m3, first_row=2)
    rows = sum(new) + 5                              # two rows before the first sequence, three behind the last
    g = torch.Generator().manual_seed(99)
    wide = (torch.randn(rows, 3 * heads, dim + 8, generator=g) * 3).to(R.DTYPES[dtype])
    k, v = wide[:, :heads, :dim], wide[:, heads:2 * heads, :dim]          # strided views of one buffer
    want_k, want_v = write_on_host(p, k, v)
    d = p.to("cuda")
    dw = wide.cuda()
    torch.ops.kv_cache_ops.write(dw[:, :heads, :dim], dw[:, heads:2 * heads, :dim], d.k_cache, d.v_cache, d.layer, d.tables, d.lens, d.starts)
    torch.cuda.synchronize()
    assert same_pool(d.k_cache.cpu(), want_k) and same_pool(d.v_cache.cpu(), want_v)

    # the whole sequences come back, earlier tokens included, into strided rows; the rows around them stay
    lens = [a + b for a, b in zip(new, ctx)]
    starts = R.starts_of(lens, 1)
    out = torch.full((sum(lens) + 3, 2 * heads, dim), 7.0, dtype=R.DTYPES[dtype], device="cuda")
    torch.ops.kv_cache_ops.read(d.k_cache, d.v_cache, d.layer, d.tables, starts.cuda(), out[:, :heads], out[:, heads:])
    got = out.cpu()
    p.k_cache, p.v_cache = want_k, want_v
    for i, (a, b) in enumerate(zip(starts.tolist(), starts.tolist()[1:])):
        for pool, part in ((want_k, got[a:b, :heads]), (want_v, got[a:b, heads:])):
            assert torch.equal(part, R.rows_of(p, pool, i).to(R.DTYPES[dtype])), f"sequence {i}"
    assert (got[0] == 7).all() and (got[starts[-1]:] == 7).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rows_at_the_borders_of_quantisation(dtype):
    t = R.DTYPES[dtype]
    top = torch.finfo(t).max
    rows = torch.zeros(14, 1, 16, dtype=torch.float64)
    rows[1, 0, 0] = 448.0
    rows[2, 0, :3] = torch.tensor([449.0 if dtype == "fp16" else 450.0, 7.25, -0.01])
    rows[3, 0, :2] = torch.tensor([top, 1.0])
    rows[4, 0, 5] = -top
    rows[5, 0, :2] = torch.tensor([6e-8, -1.2e-7]) if dtype == "fp16" else torch.tensor([1e-40, -3e-39])
    rows[6, 0, 3] = math.inf
    rows[7, 0, 4] = math.nan
    rows[8, 0] = torch.arange(16) * 2.0 ** -9 + 2.0 ** -10          # halfway between codes below the smallest normal one
    rows[8, 0, 15] = 300.0
    rows[9, 0] = torch.arange(16) * 0.0625 + 16.0 + 1.0             # halfway between codes of one binade
    rows[9, 0, 15] = 447.0 if dtype == "fp16" else 446.0
    rows[10, 0, 0] = 1.75
    rows[11, 0, 0] = 1.7509765625 if dtype == "fp16" else 1.7578125
    rows[12, 0, 0] = -math.inf
    rows[13, 0] = torch.linspace(-1, 1, 16)
    k = rows.to(t)
    p = R.make_paged(3, [14], [0], 1, 16, 4, dtype, True)
    want_k, want_v = write_on_host(p, k, -k)
    d = p.to("cuda")
    torch.ops.kv_cache_ops.write(k.cuda(), -k.cuda(), d.k_cache, d.v_cache, d.layer, d.tables, d.lens, d.starts)
    assert same_pool(d.k_cache.cpu(), want_k) and same_pool(d.v_cache.cpu(), want_v)
    out = torch.zeros(2, 14, 1, 16, dtype=t, device="cuda")
    torch.ops.kv_cache_ops.read(d.k_cache, d.v_cache, d.layer, d.tables, d.starts, out[0], out[1])
    p.k_cache, p.v_cache = want_k, want_v
    for got, pool in zip(out.cpu(), (want_k, want_v)):
        want = R.rows_of(p, pool, 0)
        nan = torch.isnan(want).any(-1)
        assert nan.flatten().tolist() == [i in (6, 7, 12) for i in range(14)]
        assert torch.isnan(got[nan]).all()
        assert torch.equal(got[~nan], want[~nan].clamp(-top, top).to(t))


@pytest.mark.parametrize("e4m3", [False, True])
def test_places_that_do_not_exist(e4m3):
    """Blocks outside the pool, tables too short, negative positions, rows out of range: nothing is written there, a read
    gives NaN there, and everything else is as it should be."""
    p = R.make_paged(5, [6, 4, 3, 5], [6, 0, 2, 0], 2, 32, 4, "fp16", e4m3)
    blocks = p.k_cache.shape[0]
    p.tables[0, 2] = blocks                          # positions 8..11 of sequence 0
    p.tables[1, 0] = -1                              # all of sequence 1
    p.lens[2] = 1                                    # rows at positions -2, -1, 0
    p.tables = p.tables[:, :3].contiguous()          # sequence 3 fits; sequence 0 ends at the table's end
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(18, 2, 32, generator=g).half() for _ in range(2))
    want_k, want_v = write_on_host(p, k, v)
    d = p.to("cuda")
    torch.ops.kv_cache_ops.write(k.cuda(), v.cuda(), d.k_cache, d.v_cache, d.layer, d.tables, d.lens, d.starts)
    assert same_pool(d.k_cache.cpu(), want_k) and same_pool(d.v_cache.cpu(), want_v)
    starts = R.starts_of([14, 2, 1, 5])              # sequence 0: two tokens more than its table holds
    out = torch.zeros(2, 22, 2, 32, dtype=torch.float16, device="cuda")
    torch.ops.kv_cache_ops.read(d.k_cache, d.v_cache, d.layer, d.tables, starts.cuda(), out[0], out[1])
    got = out.cpu()
    assert torch.isnan(got[:, 8:16]).all()           # the bad block, past the table's end, and sequence 1
    p.k_cache, p.v_cache = want_k, want_v
    for x, pool in zip(got, (want_k, want_v)):
        assert torch.equal(x[:8], R.rows_of(p, pool, 0, 8).half())
        assert torch.equal(x[16:17], R.rows_of(p, pool, 2, 1).half())
        assert torch.equal(x[17:], R.rows_of(p, pool, 3, 5).half())
    # sequences whose rows are not in the buffer, or run backwards, are skipped
    before = bits(d.k_cache).clone()
    for starts in ([0, 6, 4, 25, 30], [-3, -1, -1, 19, 19], [18, 18, 18, 18, 19]):
        lens = R.ints([0, 0, 0, 0]) if starts[1] == 6 else d.lens
        torch.ops.kv_cache_ops.write(k.cuda(), v.cuda(), d.k_cache, d.v_cache, d.layer, d.tables, lens.cuda(), R.ints(starts).cuda())
    assert torch.equal(before, bits(d.k_cache))


def test_a_pool_of_more_than_two_to_the_31_values():
    """Offsets pass 32 bits: the last block of a pool of 4.5 GB."""
    blocks, layers, heads, block, dim = 1100, 8, 16, 128, 128
    k_cache = torch.zeros(blocks, layers, heads, block, dim, dtype=torch.bfloat16, device="cuda")
    v_cache = torch.zeros_like(k_cache)
    assert k_cache.numel() > 2 ** 31
    k = torch.randn(130, heads, dim, device="cuda").bfloat16()
    tables, starts, lens = R.ints([[blocks - 1, 0]]).cuda(), R.ints([0, 130]).cuda(), R.ints([130]).cuda()
    torch.ops.kv_cache_ops.write(k, -k, k_cache, v_cache, layers - 1, tables, lens, starts)
    assert torch.equal(k_cache[-1, -1].transpose(0, 1), k[:128]) and torch.equal(v_cache[0, -1, :, :2].transpose(0, 1), -k[128:])
    assert int((k_cache != 0).sum()) == int((k != 0).sum())
    out = torch.empty_like(k), torch.empty_like(k)
    torch.ops.kv_cache_ops.read(k_cache, v_cache, layers - 1, tables, starts, *out)
    assert torch.equal(out[0], k) and torch.equal(out[1], -k)
    attended = torch.empty(1, heads, dim, dtype=torch.bfloat16, device="cuda")
    torch.ops.kv_attention_ops.paged(k[-1:], k_cache, v_cache, layers - 1, tables, lens, R.ints([0, 1]).cuda(), 1, dim ** -0.5, attended)
    want = R.attend(k[-1:].cpu(), k.double().cpu(), -k.double().cpu(), dim ** -0.5, "bf16")
    R.assert_close(attended, want, "attention over the pool's end")
