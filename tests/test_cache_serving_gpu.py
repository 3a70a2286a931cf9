"""The cache's operators as a deployment runs them: prompts attended and written by the context stage's workers, migrated to
decoding workers of another tensor-parallel size, decoded there token by token with a swap in between, and read back; in
16-bit and in quantised pools.  Also their place in a stream beside migrations, and the serving loop that uses them."""
import pytest
import torch

from distserve_b200 import capi, e2e_loop
from distserve_b200.config import CacheConfig, KVModelConfig, ParallelConfig
from distserve_b200.worker import KVWorker
from tests import attnref as R

pytestmark = pytest.mark.gpu


def table(blocks, width):
    return list(blocks) + [0] * (width - len(blocks))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kv_format,dtype", [("model", "float16"), ("e4m3", "float16"), ("e4m3", "bfloat16")])
def test_prefill_migrate_decode(built_libs, kv_format, dtype):
    capi.reset_registry()
    layers, kv_heads, group, dim, block = 2, 4, 2, 64, 16
    heads = kv_heads * group
    model, cache = KVModelConfig(layers, kv_heads, dim, dtype), CacheConfig(block, 64, kv_format=kv_format)
    ctx_pc = ParallelConfig(2, 0, 1, 0)
    short = {"float16": "fp16", "bfloat16": "bf16"}[dtype]
    g = torch.Generator().manual_seed(11)
    rand = lambda n, h: torch.randn(n, h, dim, generator=g).to(R.DTYPES[short])  # noqa: E731
    prompts, steps = [33, 5, 80], 20
    total = sum(prompts)
    q, k, v = [rand(total, heads) for _ in range(layers)], [rand(total, kv_heads) for _ in range(layers)], [rand(total, kv_heads) for _ in range(layers)]
    starts = R.starts_of(prompts)

    # context stage: two workers, two KV heads each
    src, handles = [[7, 2, 9], [4], [1, 0, 12, 5, 8]], []
    ctx = []
    for t in range(2):
        w = KVWorker(t, "context", model, cache, ctx_pc.with_rank(0, t))
        handles.append(w.init_kvcache_and_swap(16, 1))
        for pool in (w.k_cache, w.v_cache):
            pool.view(torch.uint8).fill_(0x7F)
        mine, mine_q = slice(2 * t, 2 * t + 2), slice(2 * t * group, (2 * t + 2) * group)
        tables, lens, st = ints([table(b, 5) for b in src]), ints(prompts), starts.cuda()
        for layer in range(layers):
            dk, dv, dq = k[layer][:, mine].cuda(), v[layer][:, mine].cuda(), q[layer][:, mine_q].cuda()
            out = w.attend_prompts(dq, dk, dv, st, max(prompts)).cpu()
            w.write_kv(layer, dk, dv, tables, lens, st)
            for i, (a, b) in enumerate(zip(starts.tolist(), starts.tolist()[1:])):
                R.assert_close(out[a:b], R.attend(q[layer][a:b, mine_q], k[layer][a:b, mine].double(), v[layer][a:b, mine].double(), dim ** -0.5, short),
                               f"prompt {i} layer {layer} rank {t}")
        ctx.append(w)

    # decoding stage: one worker with all heads
    dec = KVWorker(0, "decoding", model, cache, ParallelConfig())
    dec.init_kvcache_and_swap(24, 8)
    for pool in (dec.k_cache, dec.v_cache):
        pool.view(torch.uint8).fill_(0x7F)
    dec.register_kvcache_mem_handles(ctx_pc, [handles])
    dst = [[0, 3, 20, 11], [23, 5], [6, 7, 19, 10, 2, 13, 14]]
    for a, b in zip(src, dst):
        dec.migrate_blocks(a, ctx_pc, b[:len(a)])
    # what the pool holds of the prompts, in 64 bits: K and V as given, or as e4m3 keeps them
    def kept(x):
        if kv_format == "model":
            return x.double()
        values, scales = R.quantise(x)
        return values * scales[..., None]

    have = [[[kept(x[layer][a:b]) for a, b in zip(starts.tolist(), starts.tolist()[1:])] for layer in range(layers)] for x in (k, v)]
    lens = list(prompts)
    one = R.starts_of([1, 1, 1]).cuda()
    for step in range(steps):
        if step == 8:                                            # request 1 goes to the host and comes back into other blocks
            dec.swap_blocks([1], dst[1], [6, 1], False)
            dst[1] = [16, 22]
            dec.swap_blocks([1], [6, 1], dst[1], True)
            dec.prepare_step([1])
        lens = [n + 1 for n in lens]
        tables, dl = ints([table(b, 7) for b in dst]), ints(lens)
        for layer in range(layers):
            nk, nv, nq = rand(3, kv_heads), rand(3, kv_heads), rand(3, heads)
            dec.write_kv(layer, nk.cuda(), nv.cuda(), tables, dl, one)
            out = dec.attend(layer, nq.cuda(), tables, dl, one, 1).cpu()
            for i in range(3):
                for x, new in ((0, nk), (1, nv)):
                    have[x][layer][i] = torch.cat([have[x][layer][i], kept(new[i:i + 1])])
                want = R.attend(nq[i:i + 1], have[0][layer][i], have[1][layer][i], dim ** -0.5, short, kv_format == "e4m3")
                R.assert_close(out[i:i + 1], want, f"step {step} layer {layer} request {i}")
    for layer in range(layers):
        rk, rv = dec.read_kv(layer, tables, R.starts_of(lens).cuda(), sum(lens))
        for i, (a, b) in enumerate(zip(R.starts_of(lens).tolist(), R.starts_of(lens).tolist()[1:])):
            assert torch.equal(rk[a:b].cpu(), have[0][layer][i].to(R.DTYPES[short])) and torch.equal(rv[a:b].cpu(), have[1][layer][i].to(R.DTYPES[short]))
    assert capi.get_counter("attention_timeouts") == 0
    capi.reset_registry()


def test_migrations_keep_their_place_beside_the_cache_operators(built_libs):
    """On one stream: a migration out of blocks that are being written comes after the write, and one into blocks that an
    attention call still reads comes after that call, although migrations may begin early among themselves."""
    capi.reset_registry()
    layers, heads, dim, block, blocks = 1, 8, 128, 16, 1200
    model, cache, pc = KVModelConfig(layers, heads, dim), CacheConfig(block, 2000), ParallelConfig()
    a, b = KVWorker(0, "context", model, cache, pc), KVWorker(1, "decoding", model, cache, pc)
    handles = a.init_kvcache_and_swap(blocks, 1)
    b.init_kvcache_and_swap(blocks, 1)
    b.register_kvcache_mem_handles(pc, [[handles]])
    n = blocks * block
    k, v = (torch.randn(n, heads, dim, device="cuda").half() for _ in range(2))
    tables, lens, starts = ints([list(range(blocks))]), ints([n]), ints([0, n])
    one = ints([0, 1])
    q = torch.randn(1, 8 * heads, dim, device="cuda").half()
    a.k_cache.zero_()
    a.v_cache.zero_()
    spare = a.k_cache.clone()
    torch.cuda.synchronize()
    for turn in range(3):
        a.k_cache.copy_(spare)
        a.v_cache.copy_(spare)
        first = b.migrate_blocks_async(list(range(4)), pc, list(range(4)))           # something of the library is on the stream
        a.write_kv(0, k, v, tables, lens, starts)
        second = b.migrate_blocks_async(list(range(4, blocks)), pc, list(range(4, blocks)))
        out = b.attend(0, q, tables, lens, one, 1)
        third = b.migrate_blocks_async([5] * 4, pc, list(range(blocks - 4, blocks)))      # overwrites what the attention read
        late = b.attend(0, q, tables, lens, one, 1)
        for t in (first, second, third):
            b.migrate_wait(t)
        torch.cuda.synchronize()
        bk, bv = b.k_cache[:, 0].transpose(1, 2).flatten(0, 1), b.v_cache[:, 0].transpose(1, 2).flatten(0, 1)
        assert torch.equal(bk[64:n - 64], k[64:n - 64]) and torch.equal(bv[64:n - 64], v[64:n - 64])
        assert torch.equal(bk[n - 64:], k[80:96].repeat(4, 1, 1))
        before_k, before_v = torch.cat([bk[:64], k[64:]]), torch.cat([bv[:64], v[64:]])
        R.assert_close(out, R.attend(q.cpu(), before_k.double().cpu(), before_v.double().cpu(), dim ** -0.5, "fp16"), "before the last migration")
        R.assert_close(late, R.attend(q.cpu(), bk.double().cpu(), bv.double().cpu(), dim ** -0.5, "fp16"), "after it")
    capi.reset_registry()


def test_the_serving_loop_attends_over_what_it_migrated(built_libs):
    capi.reset_registry()
    launches = capi.get_counter("attention_launches")
    out = e2e_loop.run(steps=40, rate=4.0, weight_gb=0.5, pool_blocks=512, time_scale=400.0, attention=True)
    assert out["verified"] is True and out["migrations"] >= 2 and out["attended_tokens"] > 0
    assert capi.get_counter("attention_launches") > launches
    capi.reset_registry()


def test_block_bytes_of_quantised_pools():
    model = KVModelConfig(2, 4, 64)
    assert model.block_bytes(ParallelConfig(), 16, "e4m3") == 2 * 4 * 16 * 68 and model.block_bytes(ParallelConfig(), 16) == 2 * 4 * 16 * 128
    with pytest.raises(ValueError, match="kv_format"):
        CacheConfig(16, 8, kv_format="int8")
