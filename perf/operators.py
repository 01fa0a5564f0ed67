"""Operators around a serving step of many requests: rotary positions in their forms, low-rank adapters beside a projection, decode attention that
accumulates each key's weight, eviction from the paged cache by those weights, and drawing tokens from given random numbers.

Sizes are those of the two dense shapes of nvr.ModelConfig's presets (heads of 128, 8 kv heads, a vocabulary of 151936, hidden sizes 1024 and 4096).
A case is a dict:
  op "rope"    `tokens` new tokens: q and k heads rotated (`form`: half | pairs; the first `rotary` columns of `dim`; `scaling`), k and v stored in the paged cache
     "lora"    y = base + scale (x A^T) B^T, each row with its request's adapter (`order`: runs of rows | mixed)
     "sample"  a token for each of `batch` rows of logits
     "attend"  one query a sequence over `shortest` .. `longest` cached keys, the weights added to the keys' scores
     "evict"   caches of `shortest` .. `longest` keys brought down to `budget`
"""
import math

import numpy as np
import torch

own = False
VOCAB = 151936
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
SCALINGS = ("plain", "linear", "ntk", "yarn", "bands")
THETA, ORIGINAL = 1e6, 4096  # base of the presets; the context that scaled positions stand for


def listed():
    return [
        # the decode step of a full batch: the smallest launch of a layer, latency counts
        dict(name="rope-step", op="rope", dtype="bfloat16", tokens=32, heads=16, kv_heads=8, dim=128, rotary=128, form="half", scaling="plain", factor=1.0, far=8192, block=256),
        # a portion of a long prompt, far out, pairs side by side in half of each head, 32-bit storage
        dict(name="rope-portion", op="rope", dtype="float32", tokens=1531, heads=32, kv_heads=8, dim=128, rotary=64, form="pairs", scaling="bands", factor=8.0, far=120000, block=256),
        # a full token budget of prompts with stretched positions
        dict(name="rope-prompts", op="rope", dtype="float16", tokens=32768, heads=16, kv_heads=8, dim=128, rotary=128, form="half", scaling="yarn", factor=4.0, far=32768, block=256),
        # a decode batch, each request with its own fine-tuned variant, some with none
        dict(name="lora-step", op="lora", dtype="bfloat16", rows=32, inner=1024, outer=2048, rank=16, adapters=32, order="mixed"),
        # a larger batch over a few variants of the larger model
        dict(name="lora-batch", op="lora", dtype="float16", rows=251, inner=4096, outer=4096, rank=64, adapters=7, order="mixed"),
        # prompts of a few requests through the wide projection
        dict(name="lora-prompts", op="lora", dtype="bfloat16", rows=8192, inner=4096, outer=12288, rank=32, adapters=5, order="runs"),
        # one user's next token
        dict(name="sample-one", op="sample", batch=1, vocab=VOCAB),
        # a throughput server's step, each row with settings of its own
        dict(name="sample-batch", op="sample", batch=256, vocab=VOCAB),
        # one long conversation
        dict(name="attend-one", op="attend", dtype="float16", batch=1, heads=16, kv_heads=8, dim=128, shortest=2047, longest=2047, block=256),
        # a server's mixed batch of the larger model
        dict(name="attend-batch", op="attend", dtype="bfloat16", batch=48, heads=32, kv_heads=8, dim=128, shortest=512, longest=8100, block=256),
        # one prompt, cut down to the cache that its answer may use
        dict(name="evict-one", op="evict", dtype="bfloat16", batch=1, kv_heads=8, dim=128, shortest=4099, longest=4099, budget=2048, first=4, last=256, block=256),
        # a batch of long contexts, most over their budget
        dict(name="evict-batch", op="evict", dtype="float16", batch=32, kv_heads=8, dim=128, shortest=1000, longest=8100, budget=2048, first=4, last=512, block=256),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "lora", "lora", "sample", "attend", "attend", "evict"])
    dtype = rng.choice(["float16", "bfloat16", "float16", "bfloat16", "float32"])
    dim = rng.choice([128, 128, 64])
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
    block, wide = rng.choice([16, 64, 256, 256]), 4 if dtype == "float32" else 2
    if op == "rope":
        rotary = rng.choice([dim, dim, dim // 2, dim // 4])
        scaling = rng.choice(SCALINGS)
        tokens = _log(rng, 1, min(32768, 500000000 // (kv_heads * (2 * group + 5) * dim * wide)))
        return dict(op=op, dtype=dtype, tokens=tokens, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rotary=rotary, form=rng.choice(["half", "pairs"]), scaling=scaling,
                    factor=1.0 if scaling == "plain" else rng.choice([2.0, 4.0, 8.0, 32.0]), far=_log(rng, 1000, 1000000), block=block)
    if op == "lora":
        inner, outer = rng.choice([1024, 2048, 4096]), rng.choice([1000, 1024, 2048, 4096, 12288])
        rank = rng.choice([8, 16, 32, 64, rng.randint(1, 96)])
        rows = _log(rng, 1, (8192 if dtype != "float32" else 1000) * 32 // max(rank, 32))
        return dict(op=op, dtype=dtype, rows=rows, inner=inner, outer=outer, rank=rank, adapters=_log(rng, 1, min(64, max(2, rows))), order=rng.choice(["runs", "mixed"]))
    if op == "sample":
        return dict(op=op, batch=_log(rng, 1, 256), vocab=rng.choice([VOCAB, 32768, rng.randint(100, 50000)]))
    if op == "attend":
        batch = _log(rng, 1, 64)
        longest = _log(rng, 1, min(32000, 2000000 // (batch * kv_heads * wide)))
        return dict(op=op, dtype=dtype, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, shortest=_log(rng, 1, longest), longest=longest, block=block)
    batch = _log(rng, 1, 32)
    longest = _log(rng, 64, min(32000, 800000 // (batch * kv_heads * wide)))
    budget = _log(rng, 16, longest)
    return dict(op=op, dtype=dtype, batch=batch, kv_heads=kv_heads, dim=dim, shortest=_log(rng, 1, longest), longest=longest, budget=budget, first=min(4, budget // 4),
                last=rng.randint(0, budget // 2), block=block)


# ---------------------------------------------------------------------------------------------------------------- inputs
class _State:
    pass


def _lengths(case):
    """Lengths spread geometrically from the shortest to the longest (a batch of one: the longest)."""
    n, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [hi] if n == 1 else [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]


def _frequencies(case):
    """Turns a position makes in each pair of columns (64 bits), and what the rotated numbers are multiplied by."""
    n, s = case["rotary"], case["factor"]
    j = np.arange(n // 2, dtype=np.float64)
    f, amplitude = THETA ** (-2.0 * j / n), 1.0
    if case["scaling"] == "linear":
        f = f / s
    elif case["scaling"] == "ntk":
        f = (THETA * s ** (n / (n - 2.0))) ** (-2.0 * j / n)
    elif case["scaling"] == "yarn":
        where = [n * math.log(ORIGINAL / (b * 2 * math.pi)) / (2 * math.log(THETA)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(where[0]), 0), min(math.ceil(where[1]), n - 1)
        ramp = np.clip((j - lo) / max(hi - lo, 1e-3), 0, 1)
        f, amplitude = f / s * ramp + f * (1 - ramp), 0.1 * math.log(s) + 1.0
    elif case["scaling"] == "bands":
        around = ORIGINAL * f / (2 * math.pi)  # turns within the original context
        smooth = np.clip((around - 1.0) / (4.0 - 1.0), 0, 1)
        f = (1 - smooth) * f / s + smooth * f
    return f / (2 * math.pi), amplitude


def _tables(lengths, block, shuffled, first=0):
    """Block tables of these lengths (-1 behind the last block), the blocks spread over the pool, and the number of blocks."""
    need = [-(-n // block) for n in lengths]
    table = np.full((len(need), max(max(need), 1)), -1, np.int32)
    table[np.arange(table.shape[1])[None] < np.array(need)[:, None]] = first + shuffled.permutation(sum(need))
    return table, sum(need)


def prepare(case, seed):
    s = _State()
    s.case, s.args = case, None
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2 + 7)
    r = np.random.default_rng([seed, 33])

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (std * torch.randn(*shape, generator=g, device="cuda")).to(dtype)

    def dev(a):
        return torch.from_numpy(np.ascontiguousarray(a)).cuda()
    dt = TYPES.get(case.get("dtype"))
    if case["op"] == "rope":
        T, H, G, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        s.qkv = normal(T, H + 2 * G, D, dtype=dt)  # a packed projection's output, as the framework's products leave it
        start = int(r.integers(0, max(1, case["far"] - T)))
        s.positions = dev(start + np.arange(T) if T > 256 else r.integers(0, case["far"], T)).to(torch.int64)  # a prompt's run, or a decode batch
        blocks = -(-T // case["block"]) + 1
        s.slots = dev(r.permutation(blocks * case["block"])[:T].astype(np.int32))
        turns, s.amplitude = _frequencies(case)
        s.turns = dev(turns)
        s.k_cache, s.v_cache = (torch.zeros(blocks * case["block"], G, D, dtype=dt, device="cuda") for _ in range(2))
        s.q, s.k = torch.empty(T, H, D, dtype=dt, device="cuda"), torch.empty(T, G, D, dtype=dt, device="cuda")
    elif case["op"] == "lora":
        T, K, N, R, n = case["rows"], case["inner"], case["outer"], case["rank"], case["adapters"]
        s.x, s.base = normal(T, K, dtype=dt), normal(T, N, dtype=dt)
        s.a, s.b = normal(n, R, K, std=K ** -0.5, dtype=dt), normal(n, N, R, std=0.5 * R ** -0.5, dtype=dt)
        s.scales = dev((0.5 + 1.5 * r.random(n)).astype(np.float32))
        ids = r.integers(-1, n, T) if case["order"] == "mixed" else np.minimum(np.arange(T) * n // max(T, 1), n - 1)  # (-1: a row of the base model alone)
        s.ids = dev(ids.astype(np.int32))
        s.y = torch.empty(T, N, dtype=dt, device="cuda")
    elif case["op"] == "sample":
        B, V = case["batch"], case["vocab"]
        s.logits = normal(B, V, std=2.0)
        s.logits.scatter_add_(1, torch.randint(0, V, (B, 40), generator=g, device="cuda"), normal(B, 40, std=3.0).abs() + 6)  # a few likely tokens
        s.temperature = dev(r.choice([0.0, 0.6, 0.8, 1.0, 1.3], B).astype(np.float32))
        if B == 1:
            s.temperature.fill_(0.8)
        s.top_k = dev(r.choice([0, 20, 50, 1000], B).astype(np.int64))
        s.top_p = dev(r.choice([1.0, 0.8, 0.9, 0.95], B).astype(np.float32))
        s.min_p = dev(r.choice([0.0, 0.0, 0.02, 0.1], B).astype(np.float32))
        s.uniform = dev(r.random(B).astype(np.float32).clip(0, 1 - 2.0 ** -24))
        s.ids, s.logprobs = torch.empty(B, dtype=torch.int64, device="cuda"), torch.empty(B, dtype=torch.float32, device="cuda")
    else:
        lengths, G, D, bs = _lengths(case), case["kv_heads"], case["dim"], case["block"]
        table, used = _tables(lengths, bs, r)
        s.table, s.lengths, s.longest = dev(table), dev(np.array(lengths, np.int32)), max(lengths)
        s.blocks = used
        if case["op"] == "evict":
            to, more = _tables([min(n, case["budget"]) for n in lengths], bs, r, used)
            s.to, s.blocks, s.used = dev(to), used + more, used
        s.k_cache, s.v_cache = normal(s.blocks, bs, G, D, dtype=dt), normal(s.blocks, bs, G, D, dtype=dt)
        s.scores = torch.rand(s.blocks, G, bs, generator=g, device="cuda").pow(8) * 4  # a few keys hold most of the weight
        if case["op"] == "attend":
            s.q = normal(len(lengths), case["heads"], D, std=2.0, dtype=dt)
            s.scored = dev(np.array([n - 1 for n in lengths], np.int32))  # the newest key has no score yet
            s.out, s.new_scores = torch.empty_like(s.q), torch.zeros_like(s.scores)
        else:
            for t in (s.k_cache, s.v_cache, s.scores):
                t[used:].zero_()
            s.new_lens = torch.empty(len(lengths), dtype=torch.int32, device="cuda")
            s.kept = torch.empty(len(lengths), G, case["budget"], dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------- a pass
def run(s):
    if own:
        return _own(s)
    return {"rope": _rope, "lora": _lora, "sample": _sample, "attend": _attend, "evict": _evict}[s.case["op"]](s)


DECAY = 0.98


def _own(s):
    import nvr_import
    nvr = nvr_import.load()
    lib, case = nvr.lib(), s.case
    if s.args is None:
        s.args = _arguments(s, nvr)
    if case["op"] != "sample":
        nvr.check(lib.nvr_ops_set_dtype(case["dtype"].encode()))
    call, args, answer = s.args
    nvr.check(call(*args, torch.cuda.current_stream().cuda_stream))
    return answer


def _arguments(s, nvr):
    """The call of a case, its arguments in front of the stream, and where its answer lies.  Workspaces are the program's, made once."""
    import ctypes
    lib, case = nvr.lib(), s.case

    def space(n):
        s.space = torch.empty(max(int(n), 16), dtype=torch.uint8, device="cuda")
        return s.space.data_ptr()
    if case["op"] == "rope":
        T, H, G, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        w = s.qkv.element_size() * D
        at = s.qkv.data_ptr()
        ld = (H + 2 * G) * D
        return lib.nvr_rope_rotate_store_kv, (at, ld, at + H * w, ld, at + (H + G) * w, ld, s.positions.data_ptr(), s.slots.data_ptr(), T, H, G, D, case["rotary"], int(case["form"] == "pairs"),
                                              s.turns.data_ptr(), s.amplitude, s.q.data_ptr(), H * D, s.k.data_ptr(), G * D, s.k_cache.data_ptr(), s.v_cache.data_ptr(),
                                              s.k_cache.shape[0]), {"q": s.q, "k": s.k, "k_cache": s.k_cache, "v_cache": s.v_cache}
    if case["op"] == "lora":
        T, K, N, R, n = case["rows"], case["inner"], case["outer"], case["rank"], case["adapters"]
        return lib.nvr_lora_add, (s.x.data_ptr(), K, s.a.data_ptr(), s.b.data_ptr(), s.scales.data_ptr(), s.ids.data_ptr(), n, T, K, N, R, s.base.data_ptr(), N, s.y.data_ptr(), N,
                                  space(lib.nvr_lora_workspace_bytes(T, K, N, R))), {"y": s.y}
    if case["op"] == "sample":
        B, V = case["batch"], case["vocab"]
        return lib.nvr_sample_uniform, (s.logits.data_ptr(), V, B, V, s.temperature.data_ptr(), s.top_k.data_ptr(), s.top_p.data_ptr(), s.min_p.data_ptr(), s.uniform.data_ptr(),
                                        s.ids.data_ptr(), s.logprobs.data_ptr(), space(lib.nvr_sample_uniform_workspace_bytes(B, V))), {"ids": s.ids, "logprobs": s.logprobs}
    B, G, D, bs = len(s.lengths), case["kv_heads"], case["dim"], case["block"]
    s.meta = nvr.AttnMetaC(is_prefill=0, context_lens=s.lengths.data_ptr(), block_tables=s.table.data_ptr(), max_blocks=s.table.shape[1], batch=B, max_context_len=s.longest)
    meta = ctypes.byref(s.meta)
    if case["op"] == "attend":
        H = case["heads"]
        return lib.nvr_paged_attn_decode_scored, (s.q.data_ptr(), H * D, s.k_cache.data_ptr(), s.v_cache.data_ptr(), meta, H, G, D, bs, s.blocks, D ** -0.5, s.scores.data_ptr(),
                                                  s.scored.data_ptr(), DECAY, s.new_scores.data_ptr(), s.out.data_ptr(),
                                                  space(lib.nvr_paged_attn_scored_workspace_bytes(B, H, G, D, s.longest))), {"out": s.out, "scores": s.new_scores}
    return lib.nvr_kv_evict, (s.k_cache.data_ptr(), s.v_cache.data_ptr(), s.scores.data_ptr(), meta, G, D, bs, s.blocks, case["budget"], case["first"], case["last"], s.to.data_ptr(),
                              s.to.shape[1], s.new_lens.data_ptr(), s.kept.data_ptr(), space(lib.nvr_kv_evict_workspace_bytes(B, G, case["budget"], s.longest))), {
        "k": s.k_cache[s.used:], "v": s.v_cache[s.used:], "scores": s.scores[s.used:], "lens": s.new_lens, "kept": s.kept}


# ---- plain forms
def _rope(s):
    case, n = s.case, s.case["rotary"]
    H, G = case["heads"], case["kv_heads"]
    at = s.positions.double()[:, None] * s.turns[None]
    at = 2 * math.pi * (at - at.round())
    c, sn = (at.cos() * s.amplitude).float()[:, None], (at.sin() * s.amplitude).float()[:, None]
    x = s.qkv[:, :H + G].float()
    y = x.clone()
    one, two = (slice(0, n, 2), slice(1, n, 2)) if case["form"] == "pairs" else (slice(0, n // 2), slice(n // 2, n))
    y[..., one] = x[..., one] * c - x[..., two] * sn
    y[..., two] = x[..., two] * c + x[..., one] * sn
    y = y.to(s.qkv.dtype)
    k_cache, v_cache = s.k_cache, s.v_cache
    k_cache[s.slots.long()] = y[:, H:]
    v_cache[s.slots.long()] = s.qkv[:, H + G:]
    return {"q": y[:, :H].contiguous(), "k": y[:, H:].contiguous(), "k_cache": k_cache, "v_cache": v_cache}


def _lora(s):
    T, n, R = s.x.shape[0], s.a.shape[0], s.a.shape[1]
    mine = (s.ids[:, None] == torch.arange(n, device="cuda")[None]).float() * s.scales[None]
    v = (s.x.float() @ s.a.float().view(n * R, -1).t()).view(T, n, R) * mine[..., None]
    return {"y": (s.base.float() + v.view(T, n * R) @ s.b.float().transpose(1, 2).reshape(n * R, -1)).to(s.y.dtype)}


def _sample(s):
    x = s.logits.double()
    V = x.shape[1]
    greedy = s.temperature == 0
    t = torch.where(greedy, 1.0, s.temperature.double())[:, None]
    z, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = ((z - z[:, :1]) / t).exp()
    at = torch.arange(V, device="cuda")[None]
    k = torch.where(greedy, 1, torch.where(s.top_k > 0, s.top_k, V))[:, None]
    w = torch.where(at < k, w, 0.0)
    total = w.cumsum(1)
    p = s.top_p.double()[:, None]
    w = torch.where((p < 1) & (total - w >= p * total[:, -1:]) & (at > 0), 0.0, w)  # behind the first that brings the sum to top_p
    w = torch.where(w >= s.min_p.double()[:, None], w, 0.0)
    mass = torch.zeros_like(w).scatter_(1, order, w)
    total = mass.cumsum(1)
    goal = s.uniform.double()[:, None] * total[:, -1:]
    ids = (total <= goal).sum(1)
    return {"ids": ids, "logprobs": (mass.gather(1, ids[:, None]) / total[:, -1:]).log()[:, 0].float()}


def _slots(s):
    """Row of the pool of key j of each sequence [B, L], and whether there is such a key."""
    j, bs = torch.arange(s.longest, device="cuda"), s.case["block"]
    there = j[None] < s.lengths[:, None]
    return torch.where(there, s.table.long()[:, j // bs] * bs + j % bs, 0), there


def _per_head(s, pool):
    """Scores of a pool by key: [B, L, G] of [blocks, G, block]."""
    at, there = _slots(s)
    return torch.where(there[..., None], pool.transpose(1, 2).reshape(-1, pool.shape[1])[at], 0.0)


def _attend(s):
    case = s.case
    B, H, G, D = len(s.lengths), case["heads"], case["kv_heads"], case["dim"]
    at, there = _slots(s)
    q = s.q.float().view(B, G, H // G, D)
    k, v = (c.view(-1, G, D)[at].float().permute(0, 2, 1, 3).contiguous() for c in (s.k_cache, s.v_cache))
    x = (q @ k.transpose(2, 3).contiguous()) * D ** -0.5
    x = torch.where(there[:, None, None], x, -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp()
    w = x / x.sum(-1, keepdim=True)
    out = (w @ v).view(B, H, D).to(s.q.dtype)
    j = torch.arange(s.longest, device="cuda")[None]
    new = w.sum(2).transpose(1, 2) + torch.where((j < s.scored[:, None])[..., None], DECAY * _per_head(s, s.scores), 0.0)
    flat = torch.zeros(s.blocks * case["block"], G, device="cuda")
    flat[at[there]] = new[there]
    return {"out": out, "scores": flat.view(s.blocks, -1, G).transpose(1, 2).contiguous()}


def _evict(s):
    case, bs = s.case, s.case["block"]
    B, G, D, n = len(s.lengths), case["kv_heads"], case["dim"], case["budget"]
    at, there = _slots(s)
    score = _per_head(s, s.scores).transpose(1, 2)  # [B, G, L]
    j = torch.arange(s.longest, device="cuda")[None]
    len_ = s.lengths[:, None].long()
    always = (j < case["first"]) | (j >= len_ - case["last"])
    score = torch.where(always[:, None], math.inf, score)
    score = torch.where(there[:, None], score, -math.inf)
    best = torch.sort(score, dim=2, descending=True, stable=True)[1][..., :n]
    mark = torch.zeros(B, G, s.longest, dtype=torch.bool, device="cuda").scatter_(2, best, True) & there[:, None]
    far = torch.where(mark, j[None], s.longest + 1)
    kept = torch.sort(far, dim=2)[0][..., :n]
    kept = torch.nn.functional.pad(kept, (0, n - kept.shape[2]), value=s.longest + 1)
    have = kept < s.longest
    new_lens = s.lengths.clamp(max=n)
    room = s.to.shape[1] * bs  # rows that the tables name
    rows = s.blocks - s.used
    i = torch.arange(min(n, room), device="cuda")
    to = torch.where(i[None] < new_lens[:, None], s.to.long()[:, i // bs] * bs + i % bs, 0)[:, None].expand(B, G, -1) - s.used * bs
    kept_, have_ = kept[..., :len(i)], have[..., :len(i)]
    src = at[:, None].expand(B, G, -1).gather(2, torch.where(have_, kept_, 0))
    head = torch.arange(G, device="cuda")[None, :, None].expand(B, G, len(i))
    to, src, head = to[have_], src[have_], head[have_]
    k, v = (torch.zeros(rows * bs, G, D, dtype=c.dtype, device="cuda") for c in (s.k_cache, s.v_cache))
    k[to, head], v[to, head] = s.k_cache.view(-1, G, D)[src, head], s.v_cache.view(-1, G, D)[src, head]
    sc = torch.zeros(rows * bs, G, device="cuda")
    sc[to, head] = s.scores.transpose(1, 2).reshape(-1, G)[src, head]
    return {"k": k.view(rows, bs, G, D), "v": v.view(rows, bs, G, D), "scores": sc.view(rows, bs, G).transpose(1, 2).contiguous(), "lens": new_lens,
            "kept": torch.where(have, kept, -1).int()}


# ---------------------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    w = 4 if case.get("dtype") == "float32" else 2
    if case["op"] == "rope":
        T, H, G, D = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": T * (w * D * (2 * H + 5 * G) + 12) + 4 * case["rotary"], "flops": 3 * T * (H + G) * case["rotary"]}
    if case["op"] == "lora":
        T, K, N, R = case["rows"], case["inner"], case["outer"], case["rank"]
        n = min(case["adapters"], T)
        return {"bytes": w * (T * K + 2 * T * N + n * R * (K + N)) + 4 * T, "flops": 2 * T * R * (K + N)}
    if case["op"] == "sample":
        return {"bytes": case["batch"] * (4 * case["vocab"] + 40), "flops": 16 * case["batch"] * case["vocab"]}
    lengths, G, D = _lengths(case), case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        H, n = case["heads"], sum(lengths)
        return {"bytes": n * G * (2 * D * w + 8) + 2 * len(lengths) * H * D * w, "flops": 4 * n * H * D}
    kept = sum(min(n, case["budget"]) for n in lengths)
    return {"bytes": 4 * G * sum(lengths) + kept * G * (4 * D * w + 4) + 4 * G * len(lengths) * case["budget"], "flops": G * sum(lengths)}


# ---------------------------------------------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "lora": _exact_lora, "sample": _exact_sample, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s)


def _exact_rope(s):
    case, n = s.case, s.case["rotary"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    turns, amplitude = _frequencies(case)
    angle = torch.from_numpy(2 * math.pi * np.remainder(s.positions.cpu().numpy()[:, None] * turns[None], 1.0)).cuda()
    turn = torch.polar(torch.full_like(angle, amplitude), angle)[:, None]  # complex numbers, a pair each
    x = s.qkv.double()
    part = x[:, :H + G, :n]
    z = torch.view_as_complex(part.reshape(*part.shape[:2], n // 2, 2).contiguous()) if case["form"] == "pairs" else torch.complex(part[..., :n // 2].contiguous(), part[..., n // 2:].contiguous())
    z = z * turn
    y = torch.view_as_real(z).reshape(part.shape) if case["form"] == "pairs" else torch.cat([z.real, z.imag], 2)
    y = torch.cat([y, x[:, :H + G, n:]], 2)
    k_cache, v_cache = (torch.zeros(s.k_cache.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    k_cache.index_copy_(0, s.slots.long(), y[:, H:])
    v_cache.index_copy_(0, s.slots.long(), x[:, H + G:])
    return {"q": y[:, :H], "k": y[:, H:], "k_cache": k_cache, "v_cache": v_cache}


def _exact_lora(s):
    y = s.base.double()
    for a in range(s.a.shape[0]):
        rows = (s.ids == a).nonzero()[:, 0]
        y[rows] += float(s.scales[a]) * (s.x[rows].double() @ s.a[a].double().t()) @ s.b[a].double().t()
    return {"y": y}


def _exact_sample(s):
    x = s.logits.cpu().numpy().astype(np.float64)
    t, k, p, m, u = (v.cpu().numpy().astype(np.float64) for v in (s.temperature, s.top_k, s.top_p, s.min_p, s.uniform))
    ids, logs = [], []
    for r in range(len(x)):
        if t[r] == 0:
            ids.append(int(np.argmax(x[r])))
            logs.append(0.0)
            continue
        order = np.argsort(-x[r], kind="stable")
        order = order[:int(k[r])] if k[r] > 0 else order
        w = np.exp((x[r][order] - x[r][order[0]]) / t[r])
        if p[r] < 1:
            n = int(np.searchsorted(np.cumsum(w), p[r] * w.sum())) + 1
            order, w = order[:n], w[:n]
        order, w = order[w >= m[r]], w[w >= m[r]]
        back = np.argsort(order)
        order, w = order[back], w[back]
        i = min(int(np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right")), len(w) - 1)
        ids.append(int(order[i]))
        logs.append(math.log(w[i] / w.sum()))
    return {"ids": torch.tensor(ids), "logprobs": torch.tensor(logs, dtype=torch.float64)}


def _rows(s, b):
    n, bs = int(s.lengths[b]), s.case["block"]
    j = torch.arange(n, device="cuda")
    return s.table[b].long()[j // bs], j % bs


def _exact_attend(s):
    case = s.case
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    out, scores = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda"), torch.zeros(s.scores.shape, dtype=torch.float64, device="cuda")
    for b in range(len(s.lengths)):
        page, row = _rows(s, b)
        k, v = s.k_cache[page, row].double(), s.v_cache[page, row].double()  # [n, G, D]
        for h in range(G):
            w = torch.softmax(s.q[b, h * (H // G):(h + 1) * (H // G)].double() @ k[:, h].t().contiguous() / math.sqrt(D), 1)
            out[b, h * (H // G):(h + 1) * (H // G)] = w @ v[:, h].contiguous()
            before = s.scores[page, h, row].double() * DECAY
            before[int(s.scored[b]):] = 0
            scores[page, h, row] = before + w.sum(0)
    return {"out": out, "scores": scores}


def _exact_evict(s):
    case, bs = s.case, s.case["block"]
    n, rows = case["budget"], s.blocks - s.used
    k, v = (torch.zeros(rows, bs, *c.shape[2:], dtype=torch.float64, device="cuda") for c in (s.k_cache, s.v_cache))
    scores = torch.zeros(rows, case["kv_heads"], bs, dtype=torch.float64, device="cuda")
    kept = torch.full(s.kept.shape, -1, dtype=torch.int32, device="cuda")
    for b in range(len(s.lengths)):
        page, row = _rows(s, b)
        L = len(page)
        for h in range(case["kv_heads"]):
            c = s.scores[page, h, row].cpu().numpy().astype(np.float64)
            middle = np.arange(min(case["first"], L), max(case["first"], L - case["last"]))
            if L > n:
                best = middle[np.argsort(-c[middle], kind="stable")[:n - case["first"] - case["last"]]]
                mine = np.sort(np.concatenate([np.arange(case["first"]), best, np.arange(L - case["last"], L)]))
            else:
                mine = np.arange(L)
            m = torch.from_numpy(mine).cuda()
            i = torch.arange(len(mine), device="cuda")
            kept[b, h, :len(mine)] = m.int()
            to = s.to[b].long()[i // bs] - s.used
            k[to, i % bs, h], v[to, i % bs, h] = s.k_cache[page[m], row[m], h].double(), s.v_cache[page[m], row[m], h].double()
            scores[to, h, i % bs] = s.scores[page[m], h, row[m]].double()
    return {"k": k, "v": v, "scores": scores, "lens": s.lengths.clamp(max=n), "kept": kept}
