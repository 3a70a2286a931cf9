"""Attention over the paged cache and of packed prompts against a plain computation in 64 bits, within a bound that
``attnref.attend`` derives for each value."""
import math

import pytest
import torch

from tests import attnref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _ops(built_libs):
    import distserve_b200

    distserve_b200.load_ops()


def run_paged(p, q, scale, max_rows=None, out=None):
    d = p.to("cuda")
    out = torch.full_like(q, 7.0, device="cuda") if out is None else out
    torch.ops.kv_attention_ops.paged(q.cuda(), d.k_cache, d.v_cache, d.layer, d.tables, d.lens, d.starts,
                                     max(p.new) if max_rows is None else max_rows, scale, out)
    return out


def check_paged(p, q, scale, dtype, what="", **kw):
    out = run_paged(p, q, scale, **kw).cpu()
    starts = p.starts.tolist()
    for i, want in enumerate(R.attend_paged(p, q, scale, dtype)):
        R.assert_close(out[starts[i]:starts[i + 1]], want, f"{what} sequence {i}")
    assert (out[:starts[0]] == 7).all() and (out[starts[-1]:] == 7).all(), "rows that no sequence names were touched"


def queries(seed, rows, heads, dim, dtype, magnitude=1.0):
    g = torch.Generator().manual_seed(1000 + seed)
    return (torch.randn(rows, heads, dim, generator=g) * magnitude).to(R.DTYPES[dtype])


# (new tokens, earlier tokens) of each sequence
STEPS = ([1, 1, 1, 1, 1], [0, 15, 16, 130, 700])
DRAFTS = ([3, 1, 0, 5, 2], [0, 62, 20, 255, 33])
CHUNKS = ([130, 1, 17, 0, 64, 200], [3, 40, 0, 9, 129, 300])
LONG_STEP = ([1, 1], [5000, 40])
LONG_DRAFT = ([4], [3001])
LONG_CHUNK = ([150, 3], [2500, 0])


@pytest.mark.parametrize("dtype,e4m3", [("fp16", False), ("bf16", False), ("fp16", True), ("bf16", True)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (8, 1), (10, 2), (7, 1), (64, 2)])
@pytest.mark.parametrize("lengths", [STEPS, DRAFTS, CHUNKS], ids=["steps", "drafts", "chunks"])
def test_paged_shapes(lengths, heads, kv_heads, dim, dtype, e4m3):
    new, ctx = lengths
    p = R.make_paged(heads, new, ctx, kv_heads, dim, 16, dtype, e4m3, first_row=1)
    check_paged(p, queries(heads, sum(new) + 4, heads, dim, dtype), dim ** -0.5, dtype)


@pytest.mark.parametrize("dtype,e4m3", [("fp16", False), ("bf16", True)])
@pytest.mark.parametrize("block", [1, 3, 4, 8, 12, 24, 32, 64, 100, 128, 256])
def test_paged_block_sizes(block, dtype, e4m3):
    if e4m3 and block % 4:
        pytest.skip("quantised pools need a multiple of 4")
    for new, ctx in (STEPS, DRAFTS, CHUNKS):
        p = R.make_paged(block, new, ctx, 2, 64, block, dtype, e4m3)
        check_paged(p, queries(block, sum(new), 6, 64, dtype), 0.125, dtype, f"{new}")


@pytest.mark.parametrize("dtype,e4m3", [("bf16", False), ("fp16", True), ("fp16", False)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (16, 2), (40, 1)])
@pytest.mark.parametrize("lengths", [LONG_STEP, LONG_DRAFT, LONG_CHUNK], ids=["step", "draft", "chunk"])
def test_paged_long_contexts(lengths, heads, kv_heads, dim, dtype, e4m3):
    new, ctx = lengths
    p = R.make_paged(heads, new, ctx, kv_heads, dim, 16, dtype, e4m3)
    check_paged(p, queries(heads, sum(new), heads, dim, dtype), dim ** -0.5, dtype)


# who is cut: the long one of three; only the one with a single token; one of more sequences than a warp has lanes; nobody
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths", [([300, 260, 70], [6000, 200, 0]), ([1, 130], [6000, 300]), ([70] * 34, [0] * 20 + [5000] + [30] * 13),
                                     ([70] * 40, [1100] * 40), ([200, 1, 200], [2300, 2300, 2300])], ids=["long", "single", "many", "none", "alike"])
def test_keys_are_cut_unevenly(lengths, e4m3):
    new, ctx = lengths
    p = R.make_paged(21, new, ctx, 2, 64, 16, "bf16", e4m3)
    check_paged(p, queries(21, sum(new), 4, 64, "bf16"), 0.125, "bf16")


@pytest.mark.parametrize("new", [[1, 1], [6, 6], [40, 40]], ids=str)
@pytest.mark.parametrize("scale,magnitude", [(0.0, 1.0), (-0.3, 1.0), (1.0, 8.0), (0.088, 1e-4), (0.088, 40.0)])
def test_paged_scales_and_magnitudes(scale, magnitude, new):
    """Flat, inverted, one-hot and tiny softmaxes."""
    for dtype, e4m3 in (("fp16", False), ("bf16", False), ("bf16", True), ("fp16", True)):
        p = R.make_paged(7, new, [300, 5], 2, 128, 16, dtype, e4m3, magnitude=magnitude)
        check_paged(p, queries(7, sum(new), 4, 128, dtype, max(1.0, magnitude / 8)), scale, dtype, f"{dtype} {e4m3}")


@pytest.mark.parametrize("new", [1, 9, 150])
@pytest.mark.parametrize("e4m3", [False, True])
def test_rising_scores(e4m3, new):
    """Every key scores higher than all before it: the running maximum changes at every step."""
    dim, n = 64, 900
    p = R.make_paged(1, [new], [n - new], 1, dim, 16, "bf16", e4m3)
    ramp = (torch.arange(n).double() * 0.05)[:, None].expand(n, dim).to(torch.bfloat16)
    for b in range(-(-n // 16)):
        part = ramp[b * 16:(b + 1) * 16][None]
        if e4m3:
            values, scales = R.quantise(part)
            codes, sc = R.split_pool(p.k_cache)
            codes[p.tables[0, b], 1, :, :part.shape[1]] = R.codes_of(values)
            sc[p.tables[0, b], 1, :, :part.shape[1]] = scales.float()
        else:
            p.k_cache[p.tables[0, b], 1, :, :part.shape[1]] = part
    q = torch.ones(new, 2, dim, dtype=torch.bfloat16)
    check_paged(p, q, 0.125, "bf16")


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [2, 40, 300])
def test_rows_without_a_position_are_zero(new, e4m3):
    """A sequence with fewer cached tokens than rows (a padded row): the first rows see nothing."""
    p = R.make_paged(2, [new, 3], [0, 20], 2, 64, 16, "fp16", e4m3)
    q = queries(2, new + 3, 4, 64, "fp16")
    have = new // 2
    p.lens[0] = have
    out = run_paged(p, q, 0.125).cpu()
    assert (out[:new - have] == 0).all()
    R.assert_close(out[new - have:new], R.attend(q[new - have:new], R.rows_of(p, p.k_cache, 0, have), R.rows_of(p, p.v_cache, 0, have), 0.125, "fp16"), "rest")
    R.assert_close(out[new:], R.attend_paged(p, q, 0.125, "fp16")[1], "the other sequence")
    p.lens[0] = 0
    assert (run_paged(p, q, 0.125).cpu()[:new] == 0).all()
    p.lens[0] = -5
    assert (run_paged(p, q, 0.125).cpu()[:new] == 0).all()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("new", [1, 5, 140])
def test_blocks_outside_the_pool_make_nan(new, e4m3):
    for bad in (-1, 1 << 20, -(1 << 31), (1 << 31) - 1):
        p = R.make_paged(3, [new, new, new], [400, 60, 200], 2, 64, 16, "bf16", e4m3)
        p.tables[0, 3] = bad
        q = queries(3, 3 * new, 4, 64, "bf16")
        out = run_paged(p, q, 0.125).cpu()
        assert torch.isnan(out[:new]).all()
        p.tables[0, 3] = 0
        for i in (1, 2):
            R.assert_close(out[i * new:(i + 1) * new], R.attend_paged(p, q, 0.125, "bf16")[i], f"sequence {i}")


@pytest.mark.parametrize("new", [1, 5, 140])
def test_lengths_beyond_the_table_and_rows_beyond_max_rows_make_nan(new):
    p = R.make_paged(4, [new, new], [100, 60], 2, 64, 16, "fp16", False)
    q = queries(4, 2 * new, 2, 64, "fp16")
    good = run_paged(p, q, 0.125).cpu()
    p.lens[0] = p.tables.shape[1] * 16 + 1
    out = run_paged(p, q, 0.125).cpu()
    assert torch.isnan(out[new - 1]).all() and torch.equal(out[new:], good[new:])
    p.lens[0] = (1 << 31) - 1
    assert torch.isnan(run_paged(p, q, 0.125).cpu()[:new]).all()
    p.lens[0] = 100 + new
    if new > 1:
        p.starts = R.ints([0, new, new + 1])
        out = run_paged(p, q, 0.125, max_rows=new - 1).cpu()
        assert torch.isnan(out[:new]).all() and torch.isfinite(out[new]).all() and (out[new + 1:] == 7).all()
    p.starts = R.ints([2 * new - 1, 2 * new + 3, 2 * new + 3])      # rows that the buffer does not have: skipped
    assert (run_paged(p, q, 0.125, max_rows=9).cpu() == 7).all()
    p.starts = R.ints([-4, -1, -1])
    assert (run_paged(p, q, 0.125, max_rows=9).cpu() == 7).all()


def test_strides_and_many_sequences():
    new = [1] * 300
    p = R.make_paged(6, new, [i % 50 for i in range(300)], 1, 64, 16, "fp16", False)
    wide = queries(6, 300, 9, 72, "fp16").cuda()
    out = torch.full((300, 5, 80), 7.0, dtype=torch.float16, device="cuda")
    d = p.to("cuda")
    tables = torch.cat([d.tables, d.tables], 1)[:, :d.tables.shape[1]]           # rows further apart than they are long
    torch.ops.kv_attention_ops.paged(wide[:, 2:6, :64], d.k_cache, d.v_cache, 1, tables, d.lens, d.starts, 1, 0.1, out[:, 1:5, 8:72])
    got, q = out.cpu(), wide.cpu()[:, 2:6, :64]
    for i, want in enumerate(R.attend_paged(p, q, 0.1, "fp16")):
        R.assert_close(got[i:i + 1, 1:5, 8:72], want, f"sequence {i}")
    got[:, 1:5, 8:72] = 7
    assert (got == 7).all()


PROMPTS = [[1], [5, 1, 0, 40], [64, 128, 63, 129], [300, 17, 1, 257], [700]]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 3), (8, 2), (5, 1), (12, 4)])
@pytest.mark.parametrize("lengths", PROMPTS, ids=str)
def test_prompts(lengths, heads, kv_heads, dim, dtype):
    rows = sum(lengths) + 3
    g = torch.Generator().manual_seed(rows)
    qkv = torch.randn(rows, heads + 2 * kv_heads, dim, generator=g).to(R.DTYPES[dtype])
    qkv[:1] = qkv[-2:] = math.nan                    # rows of no sequence
    starts = R.starts_of(lengths, 1)
    dev = qkv.cuda()
    out = torch.full((rows, heads, dim), 7.0, dtype=qkv.dtype, device="cuda")
    torch.ops.kv_attention_ops.prompt(dev[:, :heads], dev[:, heads:heads + kv_heads], dev[:, heads + kv_heads:], starts.cuda(),
                                      max(lengths), dim ** -0.5, out)
    out = out.cpu()
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads].double(), qkv[:, heads + kv_heads:].double()
    for i, (a, b) in enumerate(zip(starts.tolist(), starts.tolist()[1:])):
        R.assert_close(out[a:b], R.attend(q[a:b], k[a:b], v[a:b], dim ** -0.5, dtype), f"prompt {i}")
    assert (out[0] == 7).all() and (out[starts[-1]:] == 7).all()


@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (5, 1)])
def test_prompts_with_heads_first_and_with_one_row_for_all(heads, kv_heads):
    lengths, dim = [150, 1, 300], 64
    n = sum(lengths)
    g = torch.Generator().manual_seed(n + heads)
    q, k, v = (torch.randn(h, n, dim, generator=g).to(torch.bfloat16) for h in (heads, kv_heads, kv_heads))
    one = lambda t: t[:, 7:8].transpose(0, 1).expand(n, -1, -1)  # noqa: E731
    first = lambda t: t.transpose(0, 1)  # noqa: E731
    starts = R.starts_of(lengths)
    for views in ((first, first, first), (one, first, first), (first, one, first), (first, first, one), (one, one, one)):
        out = torch.full((heads, n, dim), 7.0, dtype=torch.bfloat16, device="cuda")
        dq, dk, dv = (view(t.cuda()) for view, t in zip(views, (q, k, v)))
        torch.ops.kv_attention_ops.prompt(dq, dk, dv, starts.cuda(), max(lengths), 0.125, first(out))
        hq, hk, hv = (view(t) for view, t in zip(views, (q, k, v)))
        got = first(out).cpu()
        for i, (a, b) in enumerate(zip(starts.tolist(), starts.tolist()[1:])):
            R.assert_close(got[a:b], R.attend(hq[a:b], hk[a:b].double(), hv[a:b].double(), 0.125, "bf16"), f"prompt {i}")


@pytest.mark.parametrize("new", [1, 9, 140])
@pytest.mark.parametrize("e4m3", [False, True])
def test_paged_queries_with_heads_first_and_with_one_row_for_all(new, e4m3):
    p = R.make_paged(12, [new, new, 2], [60, 700, 3], 2, 128, 16, "fp16", e4m3)
    q, d = queries(12, 8, 2 * new + 2, 128, "fp16"), p.to("cuda")
    for view in (lambda t: t.transpose(0, 1), lambda t: t[:, :1].transpose(0, 1).expand(2 * new + 2, -1, -1)):
        out = torch.full((2 * new + 2, 8, 128), 7.0, dtype=torch.float16, device="cuda")
        torch.ops.kv_attention_ops.paged(view(q.cuda()), d.k_cache, d.v_cache, d.layer, d.tables, d.lens, d.starts, max(new, 2), 0.09, out)
        got = out.cpu()
        for i, e in enumerate(R.attend_paged(p, view(q), 0.09, "fp16")):
            R.assert_close(got[p.starts[i]:p.starts[i + 1]], e, f"sequence {i}")


def test_prompts_do_not_see_each_other_and_too_long_ones_are_nan():
    lengths, dim = [70, 33, 90], 64
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(193, 4, dim, generator=g).half().cuda() for _ in range(3))
    starts = R.starts_of(lengths).cuda()
    run = lambda k, v, n, st=starts: (lambda o: (torch.ops.kv_attention_ops.prompt(q, k, v, st, n, 0.125, o), o.cpu())[1])(torch.full_like(q, 7.0))  # noqa: E731
    good = run(k, v, 90)
    k2, v2 = k.clone(), v.clone()
    k2[70:103], v2[70:103] = math.nan, math.inf
    out = run(k2, v2, 90)
    assert torch.equal(out[:70], good[:70]) and torch.equal(out[103:], good[103:])
    out = run(k, v, 80)
    assert torch.isnan(out[103:]).all() and torch.equal(out[:103], good[:103])
    assert (run(k, v, 90, R.ints([190, 194, 195, 195]).cuda()) == 7).all()


@pytest.mark.parametrize("new", [1, 6, 200])
@pytest.mark.parametrize("e4m3", [False, True])
def test_streams_graphs_and_repetition(new, e4m3):
    """Another stream, two captured graphs replayed at once on two streams, new lengths in a captured graph, and the same
    bits on every repetition."""
    p = R.make_paged(9, [new] * 3, [2000, 37, 900], 2, 128, 16, "fp16", e4m3)
    q = queries(9, 3 * new, 16, 128, "fp16")
    d, dq = p.to("cuda"), q.cuda()
    want = run_paged(p, q, 0.09)
    torch.cuda.synchronize()
    call = lambda out: torch.ops.kv_attention_ops.paged(dq, d.k_cache, d.v_cache, d.layer, d.tables, d.lens, d.starts, new, 0.09, out)  # noqa: E731
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], [torch.zeros_like(dq), torch.zeros_like(dq)]
    for s, o in zip(streams, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(o)
        graphs.append(g)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
    p.lens[0], p.lens[2] = 1000 + new, new
    d.lens.copy_(p.lens)
    graphs[0].replay()
    torch.cuda.synchronize()
    out = outs[0].cpu()
    for i, e in enumerate(R.attend_paged(p, q, 0.09, "fp16")):
        R.assert_close(out[i * new:(i + 1) * new], e, f"after a change of lengths, sequence {i}")


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_tensors_on_another_device_than_the_current_one():
    p = R.make_paged(9, [2, 1], [40, 300], 2, 64, 16, "fp16", False)
    q = queries(9, 3, 4, 64, "fp16")
    with torch.cuda.device(1):
        d, dq = p.to("cuda:1"), q.to("cuda:1")
    out = torch.zeros_like(dq)
    torch.ops.kv_attention_ops.paged(dq, d.k_cache, d.v_cache, d.layer, d.tables, d.lens, d.starts, 2, 0.1, out)
    for i, e in enumerate(R.attend_paged(p, q, 0.1, "fp16")):
        R.assert_close(out[d.starts[i]:d.starts[i + 1]], e, f"sequence {i}")
