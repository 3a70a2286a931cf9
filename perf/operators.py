"""Timing cases of the paged KV cache's operators: writing new tokens into the cache (16-bit, or quantised to e4m3 with
a scale for each token and head), reading sequences back, attention of new tokens over the cache, and attention of whole
packed prompts.

Every case is computed in a plain form (elementary torch operations, 32 bits) and, with ``own`` set, by the operators
that ``distserve_b200`` registers.  The sizes are one worker's share of the layouts in ``distserve_b200/workloads.py``
(12 heads of 64; 40 heads of 128; grouped heads of 128 split over tensor-parallel workers), with block size 16 unless
said otherwise, and generic long contexts.

A quantised pool is a byte tensor [num_blocks, layers, heads, block_size, head_dim + 4].  The bytes of one (block,
layer, head) are block_size rows of head_dim e4m3 codes and then block_size scales in 32-bit floating point: powers of
two, the smallest for which no value of the row exceeds 448 scales.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
DEVICE = "cuda"


# ---- cases ---------------------------------------------------------------------------------------------------------

def _case(name, op, dtype, heads, kv_heads, dim, seqs, new, ctx, lens_seed, e4m3=False, block=16, layers=2):
    return {"name": name, "op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "seqs": seqs,
            "new_lo": new[0], "new_hi": new[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1], "lens_seed": lens_seed, "e4m3": e4m3,
            "block": block, "layers": layers}


def listed():
    return [
        # one decoding step's new tokens of a batch: a launch-bound write
        _case("write_step", "write", "fp16", 16, 16, 128, 32, (1, 1), (64, 2048), 1),
        # the keys and values of a prefill batch, quantised on their way into the cache
        _case("write_prompts_e4m3", "write", "fp16", 40, 40, 128, 10, (200, 2048), (0, 0), 2, e4m3=True),
        # a few short requests read back
        _case("read_requests", "read", "fp16", 12, 12, 64, 4, (64, 512), (0, 0), 3),
        # long requests of grouped heads read back from a quantised cache
        _case("read_long_e4m3", "read", "bf16", 32, 4, 128, 12, (1024, 8192), (0, 0), 4, e4m3=True),
        # a small model's decoding step: the least work there is
        _case("step_small", "paged", "fp16", 12, 12, 64, 4, (1, 1), (64, 512), 5),
        # a 13B-shaped decoding step without grouped heads: reads a GB of cache
        _case("step_batch", "paged", "fp16", 40, 40, 128, 64, (1, 1), (100, 2048), 6),
        # one long request, one token, grouped heads: few rows, a long axis
        _case("step_one_long", "paged", "bf16", 64, 8, 128, 1, (1, 1), (32768, 32768), 7),
        # up to five drafted tokens a request over a quantised cache with long contexts
        _case("drafts_long_e4m3", "paged", "bf16", 32, 4, 128, 8, (2, 5), (4000, 30000), 8, e4m3=True),
        # chunks of long prompts over what the cache has of them, grouped heads
        _case("chunk", "paged", "bf16", 32, 4, 128, 4, (300, 512), (1000, 8000), 9),
        # chunks and single tokens in one batch over a quantised cache
        _case("mixed_e4m3", "paged", "fp16", 16, 16, 128, 8, (1, 512), (300, 4000), 15, e4m3=True),
        # whole prompts of a small model
        _case("prompts_small", "prompt", "fp16", 12, 12, 64, 8, (64, 512), (0, 0), 11),
        # whole prompts, grouped heads, up to 4096 tokens
        _case("prompts", "prompt", "bf16", 32, 4, 128, 6, (500, 4096), (0, 0), 15),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "paged", "paged", "paged", "prompt"])
    dtype, e4m3 = rng.choice(["fp16", "bf16"]), op != "prompt" and rng.random() < 0.5
    dim, group = rng.choice([64, 128, 128]), rng.choice([1, 1, 2, 4, 5, 8])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12, 16])
    block, seed = rng.choice([8, 16, 16, 16, 32, 64]), rng.randrange(1 << 30)
    if op in ("write", "read"):
        longest = _log_int(rng, 1 if op == "write" else 16, 2048)
        seqs, new, ctx, group = _log_int(rng, 1, 24), (max(1, longest // 3), longest), (0, rng.choice([0, 1000]) if op == "write" else 0), 1
    elif op == "prompt":
        kv_heads, group = min(kv_heads, 8), min(group, 4)
        longest = _log_int(rng, 32, 2048)
        seqs, new, ctx = _log_int(rng, 1, 6), (max(1, longest // 5), longest), (0, 0)
    else:
        longest = rng.choice([1, 1, 1, _log_int(rng, 2, 16), _log_int(rng, 17, 512)])
        far = _log_int(rng, 50, 4000 if longest > 16 else 24000)
        seqs = _log_int(rng, 1, 4 if longest > 16 or far > 8000 else 48)
        kv_heads = min(kv_heads, 8) if seqs * far > 30000 else kv_heads
        new, ctx = (max(1, longest // 3), longest), (far // 4, far)
    return {k: v for k, v in _case("", op, dtype, kv_heads * group, kv_heads, dim, seqs, new, ctx, seed, e4m3, block).items() if k != "name"}


def _lengths(case):
    """New tokens and earlier tokens of each sequence, from the case alone; spread over their logarithm."""
    r = random.Random(case["lens_seed"])
    spread = lambda lo, hi: hi if lo == hi else int(min(hi, max(lo, round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1))) - 1))))  # noqa: E731
    return ([spread(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])],
            [spread(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])])


def work(case):
    new, ctx = _lengths(case)
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    row = hk * (d + 4 if case["e4m3"] else 2 * d)               # one token's K (or V) in the cache
    dense = hk * d * 2                                          # and outside it
    total, cached = sum(new), sum(n + c for n, c in zip(new, ctx))
    if case["op"] in ("write", "read"):
        return {"bytes": 2 * total * (row + dense), "flops": 0}
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, ctx))
    q_and_out = 2 * total * hq * d * 2
    kv = 2 * cached * row if case["op"] == "paged" else 2 * total * dense
    return {"bytes": q_and_out + kv, "flops": 4 * pairs * hq * d}


# ---- inputs --------------------------------------------------------------------------------------------------------

def _tiles(pool):
    """A quantised pool's codes [num_blocks, layers, heads, block_size, head_dim] and scales [.., block_size], as views."""
    nb, layers, heads, bs, width = pool.shape
    flat = pool.view(nb, layers, heads, bs * width)
    codes = flat[..., :bs * (width - 4)].unflatten(-1, (bs, width - 4))
    return codes, flat[..., bs * (width - 4):].view(torch.float32)


def _quantise(x):
    """Codes (bytes) and scales of the rows of x: scale 2**e for the smallest e with max|row| <= 448 * 2**e."""
    top = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)                                     # top = m * 2**e, m in [0.5, 1); 448 = 0.875 * 2**9
    e = torch.where(m > 0.875, e - 8, e - 9)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e.clamp(min=-100)), torch.ones_like(top))
    return (x / scale).to(torch.float8_e4m3fn).view(torch.uint8), scale.squeeze(-1)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    rng = np.random.default_rng([seed, case["lens_seed"]])
    dtype, hq, hk, d, bs, layers = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"], case["block"], case["layers"]
    new, ctx = _lengths(case)
    lens, total, n = [a + b for a, b in zip(new, ctx)], sum(new), case["seqs"]
    normal = lambda *shape: torch.randn(shape, generator=g, device=DEVICE).to(dtype)  # noqa: E731
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    starts = ints([0] + list(np.cumsum(new)))
    state = {"op": case["op"], "starts": starts, "max_new": max(new), "max_len": max(lens), "scale": d ** -0.5}
    if case["op"] == "prompt":
        # what a fused projection gives: q, k and v side by side in one row
        qkv = normal(total, hq + 2 * hk, d)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        return {**state, "q": q, "k": k, "v": v, "out": torch.empty(total, hq, d, dtype=dtype, device=DEVICE)}
    need = [-(-x // bs) for x in lens]
    num_blocks = sum(need) + 7
    ids = rng.permutation(num_blocks)
    tables, at = np.zeros((n, max(need)), dtype=np.int32), 0
    for i, c in enumerate(need):
        tables[i, :c] = ids[at:at + c]
        at += c
    layer = layers - 1
    k_cache, v_cache = normal(num_blocks, layers, hk, bs, d), normal(num_blocks, layers, hk, bs, d)
    if case["e4m3"]:
        pools = []
        for x in (k_cache, v_cache):
            pool = torch.empty(num_blocks, layers, hk, bs, d + 4, dtype=torch.uint8, device=DEVICE)
            codes, scales = _tiles(pool)
            for part in range(layers):
                c, s = _quantise(x[:, part].float())
                codes[:, part], scales[:, part] = c, s
            pools.append(pool)
        k_cache, v_cache = pools
    state |= {"k_cache": k_cache, "v_cache": v_cache, "layer": layer, "tables": ints(tables), "lens": ints(lens)}
    if case["op"] == "write":
        state |= {"k": normal(total, hk, d) * 2, "v": normal(total, hk, d)}
    elif case["op"] == "read":
        state |= {"k_out": torch.empty(total, hk, d, dtype=dtype, device=DEVICE), "v_out": torch.empty(total, hk, d, dtype=dtype, device=DEVICE)}
    else:
        state |= {"q": normal(total, hq, d), "out": torch.empty(total, hq, d, dtype=dtype, device=DEVICE)}
    return state


# ---- the operators -------------------------------------------------------------------------------------------------

def _slots(s, rows):
    """Block and offset of each new token (or, with no lengths, of each token from the first), and its sequence."""
    t = torch.arange(rows, device=s["starts"].device)
    seq = torch.searchsorted(s["starts"][1:], t, right=True)
    pos = t - s["starts"][seq]
    if s["op"] == "write":
        pos = pos + s["lens"][seq] - (s["starts"][seq + 1] - s["starts"][seq])
    bs = s["k_cache"].shape[3]
    return s["tables"][seq, pos // bs].long(), pos % bs


def _plain_write(s):
    blocks, offsets = _slots(s, s["k"].shape[0])
    out = []
    for new, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        if cache.dtype != torch.uint8:
            cache[:, s["layer"]][blocks, :, offsets] = new
            out.append(cache)
            continue
        codes, scales = _tiles(cache)
        c, e = _quantise(new.float())
        codes[:, s["layer"]][blocks, :, offsets] = c
        scales[:, s["layer"]][blocks, :, offsets] = e
        out.append((codes.view(torch.float8_e4m3fn), scales))
    return out


def _cached(cache, layer, blocks, offsets):
    """Rows of one layer in 32 bits, [.., heads, head_dim], for index tensors of any shape."""
    if cache.dtype != torch.uint8:
        return cache[:, layer][blocks, :, offsets].float()
    codes, scales = _tiles(cache)
    return codes[:, layer][blocks, :, offsets].view(torch.float8_e4m3fn).float() * scales[:, layer][blocks, :, offsets].unsqueeze(-1)


def _plain_read(s):
    blocks, offsets = _slots(s, s["k_out"].shape[0])
    top = torch.finfo(s["k_out"].dtype).max
    return tuple(_cached(c, s["layer"], blocks, offsets).clamp(-top, top).to(s["k_out"].dtype) for c in (s["k_cache"], s["v_cache"]))


def _softmax_rows(q, k, v, seen, scale):
    """q [n, Q, heads, D], k and v [n, S, kv_heads, D], seen [n, Q, S]: softmax(scale q k) v in 32 bits."""
    n, rows, heads, d = q.shape
    group = heads // k.shape[2]
    q = q.unflatten(2, (k.shape[2], group)).permute(0, 2, 3, 1, 4).reshape(n, k.shape[2], group * rows, d)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(scale).unflatten(2, (group, rows))
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score.sub_(score.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.flatten(2, 3), v.permute(0, 2, 1, 3)).unflatten(2, (group, rows)) / total.clamp(min=1e-38)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)


def _padded(s):
    """Row numbers of the new tokens, [n, max_new], and which of them exist."""
    starts = s["starts"].long()
    step = torch.arange(s["max_new"], device=starts.device)
    count = starts[1:] - starts[:-1]
    there = step < count[:, None]
    return torch.where(there, starts[:-1, None] + step, 0), there, count


def _plain_paged(s):
    rows, there, count = _padded(s)
    key = torch.arange(s["max_len"], device=rows.device)
    bs = s["k_cache"].shape[3]
    lens = s["lens"].long()
    have = key < lens[:, None]
    blocks, offsets = torch.where(have, s["tables"].long()[:, key // bs], 0), (key % bs).expand(len(lens), -1)
    k, v = (_cached(c, s["layer"], blocks, offsets) for c in (s["k_cache"], s["v_cache"]))
    last = (lens - count)[:, None] + torch.arange(s["max_new"], device=rows.device)
    seen = (key <= last[..., None]) & have[:, None]
    return _softmax_rows(s["q"][rows].float(), k, v, seen, s["scale"])[there].to(s["q"].dtype)


def _plain_prompt(s):
    rows, there, _ = _padded(s)
    at = torch.arange(s["max_new"], device=rows.device)
    seen = (at <= at[:, None]) & there[:, None]
    return _softmax_rows(*(s[x][rows].float() for x in "qkv"), seen, s["scale"])[there].to(s["q"].dtype)


def _own(s):
    import distserve_b200

    distserve_b200.load_ops()
    if s["op"] == "prompt":
        torch.ops.kv_attention_ops.prompt(s["q"], s["k"], s["v"], s["starts"], s["max_new"], s["scale"], s["out"])
        return s["out"]
    if s["op"] == "paged":
        torch.ops.kv_attention_ops.paged(s["q"], s["k_cache"], s["v_cache"], s["layer"], s["tables"], s["lens"], s["starts"],
                                         s["max_new"], s["scale"], s["out"])
        return s["out"]
    if s["op"] == "read":
        torch.ops.kv_cache_ops.read(s["k_cache"], s["v_cache"], s["layer"], s["tables"], s["starts"], s["k_out"], s["v_out"])
        return s["k_out"], s["v_out"]
    torch.ops.kv_cache_ops.write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["layer"], s["tables"], s["lens"], s["starts"])
    if s["k_cache"].dtype != torch.uint8:
        return [s["k_cache"], s["v_cache"]]
    return [(c.view(torch.float8_e4m3fn), e) for c, e in (_tiles(s["k_cache"]), _tiles(s["v_cache"]))]


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "read": _plain_read, "paged": _plain_paged, "prompt": _plain_prompt}[state["op"]](state)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------

def _rows64(s, cache, seq, count):
    """The first `count` tokens of a sequence, [count, heads, head_dim], in 64 bits."""
    bs, width = cache.shape[3], cache.shape[4]
    used = cache[s["tables"][seq, :-(-count // bs)].long(), s["layer"]].contiguous()
    if cache.dtype == torch.uint8:
        raw = used.flatten(2)
        codes = raw[..., :bs * (width - 4)].contiguous().view(torch.float8_e4m3fn).double().view(*used.shape[:3], width - 4)
        used = codes * raw[..., bs * (width - 4):].contiguous().view(torch.float32).double()[..., None]
    return used.double().transpose(1, 2).flatten(0, 1)[:count]


def _attend64(q, k, v, scale):
    """q [Q, heads, D] are the last Q positions of k, v [S, kv_heads, D]; one query head at a time."""
    rows, heads, _ = q.shape
    group, first = heads // k.shape[1], k.shape[0] - rows
    hidden = torch.arange(k.shape[0], device=q.device) > torch.arange(rows, device=q.device)[:, None] + first
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    for h in range(heads):
        score = scale * (q[:, h].double() @ k[:, h // group].T)
        out[:, h] = torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v[:, h // group]
    return out


def _codes64(x):
    """The e4m3 codes' values and the scales of rows in 64 bits, from the definition: nearest code, ties to even."""
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, 2.0 ** torch.ceil(torch.log2(top / 448).clamp(min=-100)), 1.0)
    scale = torch.where(top > 448 * scale, 2 * scale, torch.where((top > 0) & (top <= 224 * scale), scale / 2, scale))
    y = x / scale
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, scale.squeeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    starts, lens = s["starts"].tolist(), s["lens"].tolist() if "lens" in s else None
    pieces = list(zip(starts, starts[1:]))
    if case["op"] == "prompt":
        return torch.cat([_attend64(s["q"][a:b], s["k"][a:b].double(), s["v"][a:b].double(), s["scale"]) for a, b in pieces])
    if case["op"] == "paged":
        return torch.cat([_attend64(s["q"][a:b], _rows64(s, s["k_cache"], i, lens[i]), _rows64(s, s["v_cache"], i, lens[i]), s["scale"])
                          for i, (a, b) in enumerate(pieces)])
    if case["op"] == "read":
        return tuple(torch.cat([_rows64(s, c, i, b - a) for i, (a, b) in enumerate(pieces)]) for c in (s["k_cache"], s["v_cache"]))
    out, bs = [], case["block"]
    for new, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        if case["e4m3"]:
            held, scales = (x.clone() for x in _tiles(cache))
            held = held.view(torch.float8_e4m3fn).double()
            scales = scales.double()
        else:
            held, scales = cache.double(), None
        values, factor = _codes64(new.double()) if case["e4m3"] else (new.double(), None)
        for i, (a, b) in enumerate(pieces):
            pos = torch.arange(lens[i] - (b - a), lens[i], device=DEVICE)
            block = s["tables"][i][pos // bs].long()
            held[block, s["layer"], :, pos % bs] = values[a:b]
            if scales is not None:
                scales[block, s["layer"], :, pos % bs] = factor[a:b]
        out.append(held if scales is None else (held, scales))
    return out
