"""GPU tests (-m gpu) of the operators around a serving step against their definitions in 64 bits (serving_util).

Tolerances come from the arithmetic: a value rounded once is off by half a step of its type (HALF_STEP), a sum of n products in 32 bits by at most n 2^-24 of the sum of the products' sizes."""
import ctypes as C
import math

import numpy as np
import pytest

import nvr_import
from serving_util import DTYPES, F32, HALF_STEP, SENTINEL, SMALLEST, Arena, attend, byref, decode, encode, evict, kind, meta, rope, rope_turns, sample, tables, typed

nvr = nvr_import.load()
pytestmark = pytest.mark.gpu
L = nvr.lib()


@pytest.fixture(scope="module", autouse=True)
def _device():
    assert nvr.device_count() >= 1, "no HIP device visible: the GPU tests must run on an MI355X"
    nvr.check(L.nvr_device_set(0))
    yield
    nvr.synchronize()
    typed("float16")


@pytest.fixture
def arena():
    a = Arena()
    yield a
    nvr.synchronize()
    a.kept.clear()


def within(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, worst %g of the %g allowed" % (what, bad.sum(), bad.size, np.abs(got - want)[bad].max(), np.broadcast_to(tol, want.shape)[bad].min())


# ------------------------------------------------------------------------------------------------------------ rotary positions
KINDS = {"plain": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


@pytest.mark.parametrize("rotary", [2, 64, 128])
@pytest.mark.parametrize("name,factor,low,high", [("plain", 1.0, 1.0, 32.0), ("linear", 8.0, 1.0, 32.0), ("ntk", 4.0, 1.0, 32.0), ("yarn", 16.0, 1.0, 32.0), ("yarn", 0.5, 1.0, 32.0), ("bands", 8.0, 1.0, 4.0)])
def test_rope_frequencies(arena, name, factor, low, high, rotary):
    sc = nvr.RopeScalingC(KINDS[name], 500000.0, factor, 8192.0, low, high)
    if name == "ntk" and rotary == 2:
        pytest.skip("refused: NTK needs more than one pair")
    d, amplitude = arena.space(rotary // 2 * 8), C.c_float()
    nvr.check(L.nvr_rope_frequencies(byref(sc), rotary, d.ptr, byref(amplitude)))
    turns, a = rope_turns(name, rotary, 500000.0, factor, 8192.0, low, high)
    assert np.allclose(d.to_numpy((rotary // 2,), np.float64), turns, rtol=1e-13, atol=0)      # (powers and logarithms of 64 bits: a few steps of 2^-53)
    assert abs(amplitude.value - a) <= a * 2 ** -23


ROPE_CASES = [  # T, H, KVH, D, rotary, pairs, far, extra columns between rows
    (1, 4, 2, 128, 128, False, 10, 0), (33, 16, 8, 128, 128, False, 4096, 0), (7, 3, 1, 64, 32, True, 1000000, 0), (5, 2, 2, 80, 32, False, 100, 0), (9, 2, 1, 96, 24, True, 100, 8),
    (3, 1, 1, 2, 2, False, 50, 0), (4, 2, 1, 10, 6, True, 50, 3), (4100, 2, 1, 64, 64, False, 1 << 40, 0), (2050, 1, 1, 128, 64, True, 130000, 0), (6, 0, 2, 64, 64, False, 9, 0), (6, 2, 0, 64, 64, True, 9, 0),
    (13, 4, 2, 256, 256, False, 70000, 0), (2, 1, 1, 1024, 1024, False, 70000, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,H,G,D,rotary,pairs,far,gap", ROPE_CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_rope_rotate_store(arena, dtype, T, H, G, D, rotary, pairs, far, gap, in_place):
    rng = np.random.default_rng(T * 31 + D)
    typed(dtype)
    w, ld = np.dtype(kind(dtype)).itemsize, (H + 2 * G) * D + gap
    x, bits = encode(rng.standard_normal((T, ld)) * 4, dtype)
    positions = rng.integers(-far if far < 1000 else 0, far, T)
    turns, amplitude = rope_turns("yarn", rotary, 10000.0, 4.0)
    slots_n = T + 5
    slots = rng.permutation(slots_n)[:T].astype(np.int32)
    if T > 2:
        slots[1] = -1 if T % 2 else slots_n                        # not stored
    buf = arena.dev(bits)
    kc, vc = arena.space(slots_n * max(G, 1) * D * w), arena.space(slots_n * max(G, 1) * D * w)
    at = buf.ptr
    q_out, k_out = (None, None) if in_place else (arena.space(T * max(H, 1) * D * w), arena.space(T * max(G, 1) * D * w))
    qo, ldqo = (at, ld) if in_place else (q_out.ptr, H * D)
    ko, ldko = (at + H * D * w, ld) if in_place else (k_out.ptr, G * D)
    nvr.check(L.nvr_rope_rotate_store_kv(at, ld, at + H * D * w, ld, at + (H + G) * D * w, ld, arena.dev(positions.astype(np.int64)).ptr, arena.dev(slots).ptr, T, H, G, D, rotary, int(pairs),
                                         arena.dev(turns).ptr, amplitude, qo, ldqo, ko, ldko, kc.ptr, vc.ptr, slots_n, None))
    heads = x[:, :(H + G) * D].reshape(T, H + G, D)
    amplitude = float(np.float32(amplitude))
    want = rope(heads, positions, turns, amplitude, pairs)
    # cos and sin rounded, two products of which one is rounded, one sum: 3 roundings of 32 bits of either term, then the store's
    size = np.abs(rope(np.abs(heads), positions * 0, turns, amplitude, pairs)) + amplitude * np.abs(heads).max(-1, keepdims=True)
    tol = 4 * F32 * size + HALF_STEP[dtype] * np.abs(want) * (1 + 2 ** -10) + SMALLEST[dtype]
    if in_place:
        all_ = decode(buf.to_numpy((T, ld), kind(dtype)), dtype)
        q, k = all_[:, :H * D].reshape(T, H, D), all_[:, H * D:(H + G) * D].reshape(T, G, D)
        assert np.array_equal(all_[:, (H + G) * D:], x[:, (H + G) * D:])
    else:
        q, k = decode(q_out.to_numpy((T, H, D), kind(dtype)), dtype), decode(k_out.to_numpy((T, G, D), kind(dtype)), dtype)
    within(np.concatenate([q, k], 1), want, tol, "rotated")
    assert np.array_equal(np.concatenate([q, k], 1)[..., rotary:], heads[..., rotary:])
    if G:
        K, V = kc.to_numpy((slots_n, G, D), kind(dtype)), vc.to_numpy((slots_n, G, D), kind(dtype))
        stored = np.zeros(slots_n, bool)
        for t in range(T):
            if 0 <= slots[t] < slots_n:
                stored[slots[t]] = True
                assert np.array_equal(decode(K[slots[t]], dtype), k[t])
                assert np.array_equal(decode(V[slots[t]], dtype), x[t, (H + G) * D:(H + 2 * G) * D].reshape(G, D))
        untouched = np.frombuffer(bytes([SENTINEL]) * w, kind(dtype))[0]
        assert (K[~stored] == untouched).all() and (V[~stored] == untouched).all()


def test_rope_without_caches_and_unaligned_rows(arena):
    """Rotation alone; rows that begin 2 bytes off a piece of 16 take the form that reads numbers one by one, with the same values."""
    rng = np.random.default_rng(5)
    typed("bfloat16")
    T, H, G, D = 11, 4, 2, 64
    turns, _ = rope_turns("plain", 64)
    x, bits = encode(rng.standard_normal((T, (H + G) * D)), "bfloat16")
    pos = arena.dev(rng.integers(0, 5000, T))
    answers = []
    for off in (0, 1):
        src = np.zeros(T * (H + G) * D + 8, np.uint16)
        src[off:off + bits.size] = bits.ravel()
        buf, q, k = arena.dev(src), arena.space(T * H * D * 2 + 16), arena.space(T * G * D * 2 + 16)
        at, ld = buf.ptr + 2 * off, (H + G) * D
        nvr.check(L.nvr_rope_rotate_store_kv(at, ld, at + H * D * 2, ld, None, 0, pos.ptr, None, T, H, G, D, 64, 0, arena.dev(turns).ptr, 1.0, q.ptr + 2 * off, H * D, k.ptr + 2 * off, G * D,
                                             None, None, 0, None))
        answers.append((q.to_numpy((T * H * D + 8,), np.uint16)[off:off + T * H * D], k.to_numpy((T * G * D + 8,), np.uint16)[off:off + T * G * D]))
    assert np.array_equal(answers[0][0], answers[1][0]) and np.array_equal(answers[0][1], answers[1][1])


# ------------------------------------------------------------------------------------------------------------ low-rank adapters
def lora_case(arena, dtype, T, K, N, R, n, ids, in_place=False, gap=0, scales=True, seed=0, amplify=1.0, off=0):
    rng = np.random.default_rng(seed + T + K + N + R)
    typed(dtype)
    w = np.dtype(kind(dtype)).itemsize
    x, xb = encode(rng.standard_normal((T, K + gap)) * amplify, dtype)
    A, Ab = encode(rng.standard_normal((max(n, 1), R, K)) * K ** -0.5 * amplify, dtype)
    B, Bb = encode(rng.standard_normal((max(n, 1), N, R)) * R ** -0.5 / amplify ** 2, dtype)
    base, bb = encode(rng.standard_normal((T, N + gap)), dtype)
    sc = (0.5 + rng.random(max(n, 1))).astype(np.float32)
    ids = np.asarray(ids, np.int32)
    pad = np.zeros(off, kind(dtype))
    dx, da, db = (arena.dev(np.concatenate([pad, b.ravel()])).ptr + off * w for b in (xb, Ab, Bb))
    dbase = arena.dev(bb)
    dy = dbase if in_place else arena.space(T * (N + gap) * w)
    ws = arena.space(L.nvr_lora_workspace_bytes(T, K, N, R), 0xFF)       # (NaN wherever something stale would be read)
    nvr.check(L.nvr_lora_add(dx, K + gap, da, db, arena.dev(sc).ptr if scales else None, arena.dev(ids).ptr, n, T, K, N, R, dbase.ptr, N + gap, dy.ptr, N + gap, ws.ptr, None))
    bits = dy.to_numpy((T, N + gap), kind(dtype))
    got = decode(bits, dtype)[:, :N]
    want, tol = base[:, :N].copy(), np.zeros((T, N))
    two = {"float16": 2.0 ** -21, "bfloat16": 2.0 ** -15, "float32": 0.0}[dtype]        # v in two numbers: half a step of half a step, relative to the row's largest (float16), to itself (bfloat16)
    for a in range(n):
        rows = ids == a
        if not rows.any():
            continue
        s = float(sc[a]) if scales else 1.0
        v = s * x[rows, :K] @ A[a].T
        dv = s * (K + 8) * F32 * (np.abs(x[rows, :K]) @ np.abs(A[a]).T) + two * np.abs(v).max(1, keepdims=True)
        want[rows] += v @ B[a].T
        tol[rows] = dv @ np.abs(B[a]).T + (R + 8) * F32 * (np.abs(v) @ np.abs(B[a]).T) + F32 * np.abs(base[rows, :N])
    touched = (ids >= 0) & (ids < n)
    tol += HALF_STEP[dtype] * (np.abs(want) + tol) + SMALLEST[dtype]
    within(got[touched], want[touched], tol[touched], "adapters")
    assert np.array_equal(got[~touched], base[~touched, :N])
    if gap:
        assert np.array_equal(bits[:, N:], bb[:, N:] if in_place else np.full((T, gap), np.frombuffer(bytes([SENTINEL]) * w, kind(dtype))[0]))
    return bits


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,N,R,n", [(1, 64, 64, 8, 1), (1, 1024, 2048, 16, 3), (5, 256, 100, 1, 2), (17, 96, 72, 5, 4), (32, 1024, 512, 16, 32), (64, 200, 1000, 33, 7), (251, 512, 264, 64, 7),
                                       (256, 128, 64, 96, 300), (3, 40, 17, 256, 2), (16, 2048, 33, 128, 1), (7, 33, 31, 3, 2)])
def test_lora_few_rows(arena, dtype, T, K, N, R, n):
    rng = np.random.default_rng(T)
    lora_case(arena, dtype, T, K, N, R, n, rng.integers(-1, n + 1, T))          # n: not an adapter either


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K,N,R,n,order", [(257, 64, 96, 16, 3, "mixed"), (1000, 128, 200, 32, 5, "runs"), (1001, 72, 64, 7, 300, "mixed"), (2049, 256, 128, 64, 2, "mixed"), (700, 64, 64, 200, 1, "runs"),
                                             (513, 64, 40, 128, 1, "runs"), (4097, 32, 32, 8, 64, "mixed")])
def test_lora_many_rows(arena, dtype, T, K, N, R, n, order):
    rng = np.random.default_rng(T)
    ids = rng.integers(-1, n, T) if order == "mixed" else np.minimum(np.arange(T) * (n + 1) // T - 1, n - 1)
    lora_case(arena, dtype, T, K, N, R, n, ids)


@pytest.mark.parametrize("T", [40, 600])
@pytest.mark.parametrize("dtype", DTYPES)
def test_lora_in_place_with_strides_and_unaligned_tensors(arena, dtype, T):
    rng = np.random.default_rng(1)
    ids = rng.integers(-1, 3, T)
    lora_case(arena, dtype, T, 96, 56, 16, 3, ids, in_place=True, gap=8)
    lora_case(arena, dtype, T, 96, 56, 16, 3, ids, in_place=True, gap=3, off=1)
    lora_case(arena, dtype, T, 96, 56, 16, 3, ids, scales=False, gap=5, off=3)


@pytest.mark.parametrize("T", [30, 500])
def test_lora_rows_without_adapters_and_no_adapters(arena, T):
    lora_case(arena, "bfloat16", T, 64, 48, 8, 2, np.full(T, -1))
    lora_case(arena, "bfloat16", T, 64, 48, 8, 2, np.full(T, -1), in_place=True)
    lora_case(arena, "float16", T, 64, 48, 8, 0, np.zeros(T))


@pytest.mark.parametrize("amplify", [2.0 ** 6, 2.0 ** -8])
def test_lora_inner_products_beyond_float16(arena, amplify):
    """x A^T of 10^5 (beyond float16) and of 10^-5 (among its subnormals) against B that undoes it."""
    lora_case(arena, "float16", 20, 512, 40, 16, 2, np.arange(20) % 2, amplify=amplify)


def test_lora_bits_repeat(arena):
    """No atomics decide an order of sums: a call gives the same bits again."""
    typed("bfloat16")
    ids = np.array([0, 1, 0, 2, 1, 0])
    a = lora_case(arena, "bfloat16", 6, 64, 64, 16, 3, ids, seed=3)
    b = lora_case(arena, "bfloat16", 6, 64, 64, 16, 3, ids, seed=3)
    assert np.array_equal(a, b)


def test_lora_of_infinite_rows_stays_in_its_rows(arena):
    typed("float16")
    T, K, N, R = 20, 64, 32, 8
    rng = np.random.default_rng(2)
    x = rng.standard_normal((T, K)).astype(np.float16)
    x[3, 5], x[4, 6] = np.inf, np.nan
    A, B, base = rng.standard_normal((1, R, K)).astype(np.float16), rng.standard_normal((1, N, R)).astype(np.float16), rng.standard_normal((T, N)).astype(np.float16)
    y, ws = arena.space(T * N * 2), arena.space(L.nvr_lora_workspace_bytes(T, K, N, R))
    nvr.check(L.nvr_lora_add(arena.dev(x).ptr, K, arena.dev(A).ptr, arena.dev(B).ptr, None, arena.dev(np.zeros(T, np.int32)).ptr, 1, T, K, N, R, arena.dev(base).ptr, N, y.ptr, N, ws.ptr, None))
    got = y.to_numpy((T, N), np.float16)
    fine = np.isfinite(got).all(1)
    assert not np.isfinite(got[[3, 4]]).any() and fine[[t for t in range(T) if t not in (3, 4)]].all()


# ------------------------------------------------------------------------------------------------------------ tokens from given numbers
def sample_rows(arena, x, T, k, p, m, u, ld=None, logprobs=True, off=0):
    B, V = x.shape
    ld = ld or V
    buf = np.full(B * ld + off, np.nan, np.float32)
    for r in range(B):
        buf[off + r * ld:off + r * ld + V] = x[r]
    ids, lp = arena.space(B * 8), arena.space(B * 4)
    ws = arena.space(L.nvr_sample_uniform_workspace_bytes(B, V), 0xFF)

    def opt(a, t):
        return None if a is None else arena.dev(np.asarray(a, t)).ptr
    nvr.check(L.nvr_sample_uniform(arena.dev(buf).ptr + 4 * off, ld, B, V, opt(T, np.float32), opt(k, np.int64), opt(p, np.float32), opt(m, np.float32), opt(u, np.float32), ids.ptr,
                                   lp.ptr if logprobs else None, ws.ptr, None))
    return ids.to_numpy((B,), np.int64), lp.to_numpy((B,), np.float32)


def check_sample(arena, x, T, k, p, m, u, **kw):
    x = np.asarray(x, np.float32)
    B = len(x)
    T, k, p, m, u = (np.broadcast_to(np.asarray(a, t), (B,)) for a, t in ((T, np.float32), (k, np.int64), (p, np.float32), (m, np.float32), (u, np.float32)))
    ids, lp = sample_rows(arena, x, T, k, p, m, u, **kw)
    want = [sample(x[r], float(T[r]), int(k[r]), float(p[r]), float(m[r]), float(u[r])) for r in range(B)]
    assert ids.tolist() == [w[0] for w in want]
    for got, (_, w) in zip(lp.tolist(), want):
        assert got == w if math.isinf(w) else abs(got - w) <= 1e-7 * max(1.0, abs(w)), (got, w)       # (64 bits inside: one rounding to 32, 6e-8)


@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 100), (4, 4096), (3, 4097), (2, 16385), (7, 50001), (2, 151936), (70, 40000)])
def test_sample_settings(arena, B, V):
    rng = np.random.default_rng(V)
    for std in (0.3, 2.0, 8.0):
        x = rng.standard_normal((B, V)) * std
        for T, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.02), (0.0, 5, 0.5, 0.1), (2.5, 1000, 0.99, 0.0), (0.05, 3, 0.2, 0.9)):
            check_sample(arena, x, T, k, p, m, rng.random(B).astype(np.float32))


def test_sample_rows_of_their_own_settings(arena):
    rng = np.random.default_rng(9)
    B, V = 40, 30000
    x = rng.standard_normal((B, V)) * 3
    check_sample(arena, x, rng.choice([0.0, 0.5, 1.0, 1.7], B), rng.choice([0, 1, 20, 29999, 30000, 10 ** 12, -3], B), rng.choice([0.0, 0.3, 0.9, 1.0, -1.0, 2.0], B), rng.choice([0.0, 0.01, 0.3, 1.0, 5.0], B),
                 rng.random(B).astype(np.float32), ld=V + 7)
    check_sample(arena, x, 1.0, 0, 0.9, 0.0, rng.random(B).astype(np.float32), ld=V + 4, off=1)


def test_sample_ends_of_the_unit_interval(arena):
    rng = np.random.default_rng(10)
    x = rng.standard_normal((4, 9000))
    for u in (0.0, 1 - 2.0 ** -24):
        check_sample(arena, x, 1.0, 0, 1.0, 0.0, u)
        check_sample(arena, x, 1.0, 7, 1.0, 0.0, u)
    ids, _ = sample_rows(arena, x.astype(np.float32), None, None, None, None, np.full(4, 1.5))     # beyond it: the last token with weight
    assert ids.tolist() == [8999] * 4


def test_sample_ties(arena):
    """Equal logits: prefixes end inside them, lowest indices first; more of them than the candidate list holds."""
    for V in (8, 5000, 20000):
        x = np.zeros((3, V), np.float32)
        x[1, ::2] = 1.0
        x[2] = np.arange(V) % 3
        rng = np.random.default_rng(V)
        for k, p in ((0, 0.5), (V // 2 + 1, 1.0), (5, 0.5), (V // 4 * 3, 0.25), (0, 1.0)):
            for u in rng.random(4).astype(np.float32):
                check_sample(arena, x, 1.0, k, p, 0.0, u)
        check_sample(arena, x, 1.0, 0, 1.0, 1.0, 0.999)
        check_sample(arena, x, 0.0, 0, 1.0, 0.0, 0.5)


def test_sample_zeros_of_either_sign_are_alike(arena):
    x = np.zeros((2, 300), np.float32)
    x[:, ::3] = -0.0
    x[1, 5] = -1.0
    for k, p in ((0, 0.4), (100, 1.0), (7, 1.0)):
        check_sample(arena, x, 1.0, k, p, 0.0, [0.3, 0.95])


def test_sample_flat_bins(arena):
    """Distinct logits so close together that tens of thousands fall into the bin that the prefix ends in."""
    rng = np.random.default_rng(11)
    V = 60000
    x = (5.0 + rng.random((3, V)) * 0.01).astype(np.float32)
    for k, p, m in ((0, 0.5, 0.0), (30001, 1.0, 0.0), (40000, 0.3, 0.0), (0, 1.0, 0.999), (20000, 0.9, 0.995)):
        check_sample(arena, x, 1.0, k, p, m, rng.random(3).astype(np.float32))


def test_sample_masked_logits(arena):
    rng = np.random.default_rng(12)
    V = 20000
    x = rng.standard_normal((8, V)).astype(np.float32)
    low = np.finfo(np.float32).min
    x[0, 100:] = -np.inf
    x[1, :] = -np.inf
    x[2, :] = np.nan
    x[3, ::2] = np.nan
    x[4, :] = low
    x[5, 1:] = low
    x[6, [5, 17000]] = np.inf
    x[7, :] = -np.inf
    x[7, 12345] = -300.0
    u = rng.random(8).astype(np.float32)
    for k, p, m in ((0, 1.0, 0.0), (50, 0.9, 0.0), (0, 0.9, 0.1), (300, 1.0, 0.0)):
        for T in (1.0, 0.0, 0.3):
            check_sample(arena, x, T, k, p, m, u)


def test_sample_large_and_small_scales(arena):
    rng = np.random.default_rng(13)
    for std, T in ((1e4, 1e3), (1e-3, 1e-3), (1e30, 1e30), (100.0, 1e-3), (1.0, 1e6), (1e-6, 1e-4)):
        x = (rng.standard_normal((3, 6000)) * std).astype(np.float32)
        for k, p, m in ((0, 1.0, 0.0), (20, 0.9, 0.0), (0, 1.0, 0.1)):
            check_sample(arena, x, T, k, p, m, rng.random(3).astype(np.float32))


def test_sample_optional_arguments_and_streams(arena):
    rng = np.random.default_rng(14)
    x = rng.standard_normal((2, 3000)).astype(np.float32)
    u = np.array([0.2, 0.7], np.float32)
    ids, _ = sample_rows(arena, x, None, None, None, None, u, logprobs=False)
    assert ids.tolist() == [sample(x[r], 1.0, 0, 1.0, 0.0, float(u[r]))[0] for r in range(2)]


# ------------------------------------------------------------------------------------------------------------ scored attention
def scored_case(arena, dtype, lengths, H, G, D, block, seed=0, scored=None, decay=0.9, bad=(), in_place=False, max_context=None, q_gap=0, qs=1.0, poison=False, mutate=None):
    rng = np.random.default_rng(seed + sum(lengths) + H + D)
    typed(dtype)
    w = np.dtype(kind(dtype)).itemsize
    table, blocks = tables(rng, lengths, block, extra=1)
    B = len(lengths)
    q, qb = encode(rng.standard_normal((B, H * D + q_gap)) * qs, dtype)
    k, kb = encode(rng.standard_normal((blocks, block, G, D)), dtype)
    v, vb = encode(rng.standard_normal((blocks, block, G, D)), dtype)
    named = table.copy()
    for b, i, page in bad:
        table[b, i] = page
    if poison:                                                     # every row that no key of a sequence has: not a number
        free = np.ones((blocks, block), bool)
        for b, n in enumerate(lengths):
            for j in range(n):
                free[named[b, j // block], j % block] = False
        nan = {"float16": 0x7E00, "bfloat16": 0x7FC0, "float32": 0x7FC00000}[dtype]
        kb[free], vb[free] = nan, nan
    scores = rng.random((blocks, G, block)).astype(np.float32)
    scale = D ** -0.5
    ds = arena.dev(scores)
    dn = ds if in_place else arena.space(scores.nbytes)
    before = dn.to_numpy(scores.shape, np.float32)
    top = max(max(lengths), 0) if max_context is None else max_context
    m = meta(arena, lengths, table, top)
    out = arena.space(B * H * D * w)
    ws = arena.space(L.nvr_paged_attn_scored_workspace_bytes(B, H, G, D, top), 0xFF)
    nvr.check(L.nvr_paged_attn_decode_scored(arena.dev(qb).ptr, H * D + q_gap, arena.dev(kb).ptr, arena.dev(vb).ptr, byref(m), H, G, D, block, blocks, scale, ds.ptr,
                                             arena.dev(np.array(scored, np.int32)).ptr if scored is not None else None, decay, dn.ptr, out.ptr, ws.ptr, None))
    got = decode(out.to_numpy((B, H, D), kind(dtype)), dtype)
    new = dn.to_numpy(scores.shape, np.float32)
    two = {"float16": 2.0 ** -21, "bfloat16": 2.0 ** -15, "float32": 0.0}[dtype]
    touched = np.zeros(scores.shape, bool)
    for b, n in enumerate(lengths):
        n = min(n, top, table.shape[1] * block)
        j = np.arange(n)
        page = table[b, j // block]
        j = j[(page >= 0) & (page < blocks)]
        if len(j) == 0:
            assert (got[b] == 0).all()
            continue
        page, row = table[b, j // block], j % block
        qq, kk, vv = q[b, :H * D].reshape(H, D), k[page, row], v[page, row]
        want, weights = attend(qq, kk, vv, scale)
        # a score is off by (D + 4) roundings of its products' sizes, a weight by twice the largest such (numerator and sum) and the exponential's, and so on
        size = max(float((np.abs(kk[:, g]) @ np.abs(qq[h])).max()) for h in range(H) for g in [h * G // H]) * scale
        dw = 2 * (D + 4) * F32 * size + (n / 4 + 64) * F32
        for h in range(H):
            s = scale * (kk[:, h * G // H] @ qq[h])
            e = np.exp(s - s.max())
            tol = (2 * dw + two) * ((e / e.sum()) @ np.abs(vv[:, h * G // H]))
            within(got[b, h], want[h], tol + HALF_STEP[dtype] * (np.abs(want[h]) + tol) + SMALLEST[dtype], "out")
        first = (n - 1 if scored is None else scored[b])
        for g in range(G):
            old = np.where(j < first, np.float64(np.float32(decay)) * scores[page, g, row], 0.0)
            within(new[page, g, row].astype(np.float64), old + weights[:, g], 2 * dw * weights[:, g] + 4 * F32 * (old + weights[:, g]) + 1e-37, "scores")
            touched[page, g, row] = True
    assert np.array_equal(new[~touched].view(np.uint32), before[~touched].view(np.uint32))
    return got, new


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G,D", [(2, 1, 64), (16, 8, 128), (8, 8, 128), (32, 8, 128), (16, 1, 64), (3, 1, 128), (4, 2, 256)])
def test_scored_attention(arena, dtype, H, G, D):
    scored_case(arena, dtype, [1, 33, 130], H, G, D, 16)
    scored_case(arena, dtype, [517], H, G, D, 256)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("block", [1, 7, 16, 48, 64, 256, 300])
def test_scored_attention_blocks(arena, dtype, block):
    """Pages that end inside a tile, and rows of the pool that no sequence has (not a number: their weight of 0 must not meet them)."""
    scored_case(arena, dtype, [5, 31, 32, 33, 64, 100], 4, 2, 64, block, poison=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scored_attention_lengths(arena, dtype):
    scored_case(arena, dtype, [0, 1, 0, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 511, 513, 1025], 4, 2, 128, 64, poison=True)
    scored_case(arena, dtype, [3000, 1, 2200], 4, 1, 64, 32)
    scored_case(arena, dtype, [0, 0], 4, 2, 128, 64)


def test_scored_attention_of_many_sequences(arena):
    rng = np.random.default_rng(3)
    scored_case(arena, "bfloat16", rng.integers(0, 700, 90).tolist(), 4, 2, 64, 64)


def test_scored_attention_new_keys_and_in_place(arena):
    scored_case(arena, "float16", [40, 90, 130], 4, 2, 64, 16, scored=[0, 50, 130], decay=1.0)
    scored_case(arena, "bfloat16", [40, 90, 130], 4, 2, 64, 16, scored=[0, 50, 999], decay=0.5, in_place=True)
    scored_case(arena, "bfloat16", [40, 90, 130], 4, 2, 64, 16, in_place=True, q_gap=3)
    scored_case(arena, "float32", [40, 90, 130], 4, 2, 64, 16, scored=[-5, 1, 3], in_place=True, q_gap=1)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scored_attention_pages_outside_the_pool(arena, dtype):
    """Keys whose page is not in the pool are not there: a whole tile, a part of one, a whole sequence."""
    scored_case(arena, dtype, [200, 200, 10], 4, 2, 64, 16, bad=[(0, 2, -1), (0, 5, 1 << 20), (1, 8, -7), (1, 9, -7), (2, 0, -1)])
    scored_case(arena, dtype, [200, 200], 4, 2, 64, 64, bad=[(0, 0, -1), (1, 3, 1 << 30)])


def test_scored_attention_cuts_contexts_at_their_bound(arena):
    scored_case(arena, "float16", [50, 500, 300], 4, 2, 64, 16, max_context=256, scored=[49, 499, 299])


def test_scored_attention_peaked(arena):
    """Weights of one key and of none: scores of +-hundreds."""
    scored_case(arena, "float32", [300, 65], 4, 2, 64, 16, qs=60.0)
    scored_case(arena, "float16", [300, 65], 4, 2, 128, 16, qs=30.0)


def test_scored_attention_agrees_with_the_plain_one(arena):
    rng = np.random.default_rng(4)
    typed("float16")
    H, G, D, block, lengths = 16, 8, 128, 256, [700, 1300]
    table, blocks = tables(rng, lengths, block)
    q, k, v = (rng.standard_normal(s).astype(np.float16) for s in ((2, H, D), (blocks, block, G, D), (blocks, block, G, D)))
    dq, dk, dv, m = arena.dev(q), arena.dev(k), arena.dev(v), meta(arena, lengths, table)
    a, b = arena.space(q.nbytes), arena.space(q.nbytes)
    sc = arena.space(blocks * G * block * 4, 0)
    nvr.check(L.nvr_paged_attn_decode(dq.ptr, H * D, dk.ptr, dv.ptr, byref(m), H, G, D, block, D ** -0.5, a.ptr, arena.space(L.nvr_paged_attn_workspace_bytes(2, H, D, 1300)).ptr, None))
    nvr.check(L.nvr_paged_attn_decode_scored(dq.ptr, H * D, dk.ptr, dv.ptr, byref(m), H, G, D, block, blocks, D ** -0.5, sc.ptr, None, 1.0, sc.ptr, b.ptr,
                                             arena.space(L.nvr_paged_attn_scored_workspace_bytes(2, H, G, D, 1300)).ptr, None))
    x, y = a.to_numpy(q.shape, np.float16).astype(np.float64), b.to_numpy(q.shape, np.float16).astype(np.float64)
    within(x, y, 2 * HALF_STEP["float16"] * np.abs(y) + 1e-5, "the two attentions")             # (each rounded once; 32-bit sums of 1300 keys below that)
    total = sc.to_numpy((blocks, G, block), np.float32).sum(dtype=np.float64)
    assert abs(total - 2 * H) < 2 * H * 1e-5                                                   # a head's weights sum to 1


# ------------------------------------------------------------------------------------------------------------ eviction
def evict_case(arena, dtype, lengths, G, D, block, budget, first, last, out_of_place, seed=0, scores=None, bad=(), kept_out=True, max_context=None):
    rng = np.random.default_rng(seed + sum(lengths) + budget)
    typed(dtype)
    u = kind(dtype)
    B = len(lengths)
    cut = [min(n, budget) for n in lengths]
    table, blocks = tables(rng, lengths, block)
    to, more = tables(rng, cut, block)
    to = np.where(to >= 0, to + blocks, -1).astype(np.int32)
    total = blocks + (more if out_of_place else 0)
    for b, i, page in bad:
        table[b, i] = page
    top = np.iinfo(u).max
    k, v = (rng.integers(0, top, (total, block, G, D), dtype=u) for _ in range(2))
    if scores is None:
        s = (rng.integers(0, 50, (total, G, block)) / 8).astype(np.float32)                     # many ties
    else:
        s = scores((total, G, block), rng)
    dk, dv, ds = arena.dev(k), arena.dev(v), arena.dev(s)
    new, kept, ws = arena.space(B * 4), arena.space(B * G * budget * 4), arena.space(L.nvr_kv_evict_workspace_bytes(B, G, budget, max(lengths)))
    m = meta(arena, lengths, table, max_context)
    nvr.check(L.nvr_kv_evict(dk.ptr, dv.ptr, ds.ptr, byref(m), G, D, block, total, budget, first, last, arena.dev(to).ptr if out_of_place else None, to.shape[1] if out_of_place else 0, new.ptr,
                             kept.ptr if kept_out else None, ws.ptr, None))
    K, V, S = k.copy(), v.copy(), s.copy()
    want_kept, want_len = np.full((B, G, budget), -1, np.int32), np.zeros(B, np.int32)
    for b, n in enumerate(lengths):
        n = min(n, max_context) if max_context is not None else n
        j = np.arange(n)
        if n and ((table[b, j // block] < 0) | (table[b, j // block] >= total)).any():
            want_len[b] = -1
            continue
        want_len[b] = min(n, budget)
        dest = to if out_of_place else table
        for g in range(G):
            mine = evict(s[table[b, j // block], g, j % block], budget, first, last)
            want_kept[b, g, :len(mine)] = mine
            i = np.arange(len(mine))
            src, dst = (table[b, mine // block], mine % block), (dest[b, i // block], i % block)
            K[dst[0], dst[1], g], V[dst[0], dst[1], g], S[dst[0], g, dst[1]] = k[src[0], src[1], g], v[src[0], src[1], g], s[src[0], g, src[1]]
    assert np.array_equal(new.to_numpy((B,), np.int32), want_len)
    got = (kept if kept_out else ws).to_numpy((B, G, budget), np.int32)
    assert np.array_equal(got, want_kept)
    assert np.array_equal(ds.to_numpy(s.shape, np.uint32), S.view(np.uint32))
    assert np.array_equal(dk.to_numpy(k.shape, u), K) and np.array_equal(dv.to_numpy(v.shape, u), V)


@pytest.mark.parametrize("out_of_place", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,G,D,block,budget,first,last", [
    ([10, 1, 0, 64, 63], 2, 64, 16, 16, 2, 4), ([300, 40, 299], 8, 128, 256, 100, 4, 32), ([1000], 1, 128, 16, 999, 0, 0), ([1000], 3, 64, 7, 1, 0, 0), ([1000, 2], 2, 64, 32, 1, 0, 1),
    ([500, 77], 2, 8, 64, 64, 64, 0), ([500, 77], 2, 8, 64, 64, 0, 64), ([257], 1, 256, 1, 256, 0, 255), ([2000, 1999], 2, 40, 48, 1500, 4, 100), ([5, 6], 2, 64, 16, 10, 1, 1)])
def test_evict(arena, dtype, lengths, G, D, block, budget, first, last, out_of_place):
    evict_case(arena, dtype, lengths, G, D, block, budget, first, last, out_of_place)


@pytest.mark.parametrize("out_of_place", [False, True])
def test_evict_long_contexts(arena, out_of_place):
    """More competing keys than LDS holds, and several steps of rows to close up."""
    evict_case(arena, "float16", [12000, 10260, 9000], 2, 64, 256, 3000, 4, 500, out_of_place)
    evict_case(arena, "float16", [30000], 1, 64, 64, 20001, 4, 0, out_of_place, scores=lambda s, r: r.random(s).astype(np.float32))


@pytest.mark.parametrize("out_of_place", [False, True])
def test_evict_scores_that_are_alike_or_no_numbers(arena, out_of_place):
    def odd(shape, rng):
        s = rng.choice(np.array([0.0, -0.0, 1.0, -1.0, np.inf, -np.inf, np.nan, 1e-40, -1e-40], np.float32), shape)
        return s
    evict_case(arena, "bfloat16", [700, 90], 2, 64, 16, 80, 3, 5, out_of_place, scores=odd)
    evict_case(arena, "bfloat16", [700, 90], 2, 64, 16, 80, 0, 0, out_of_place, scores=lambda s, r: np.zeros(s, np.float32))
    evict_case(arena, "bfloat16", [700, 90], 2, 64, 16, 80, 0, 0, out_of_place, scores=lambda s, r: np.full(s, np.nan, np.float32))


@pytest.mark.parametrize("out_of_place", [False, True])
def test_evict_leaves_sequences_with_bad_pages(arena, out_of_place):
    evict_case(arena, "float16", [100, 100, 20, 100], 2, 64, 16, 40, 2, 8, out_of_place, bad=[(1, 3, -1), (2, 0, 1 << 20)], kept_out=False)


def test_evict_cuts_contexts_at_their_bound(arena):
    evict_case(arena, "float16", [100, 300], 2, 64, 16, 40, 2, 8, False, max_context=200)
    evict_case(arena, "float16", [100, 300], 2, 64, 16, 40, 2, 8, False, max_context=40)


def test_evict_refuses_tables_that_are_too_short_on_the_device(arena):
    """to_tables rows of one block for a budget of three: every sequence that needs more stays as it is."""
    typed("float16")
    lengths, block = [60, 10], 16
    table = np.arange(5, dtype=np.int32)
    t = np.array([[0, 1, 2, 3], [4, -1, -1, -1]], np.int32)
    k = np.random.default_rng(0).integers(0, 60000, (8, block, 1, 8), dtype=np.uint16)
    s = np.random.default_rng(1).random((8, 1, block)).astype(np.float32)
    dk, dv, ds, new, kept = arena.dev(k), arena.dev(k), arena.dev(s), arena.space(8), arena.space(2 * 48 * 4)
    m = meta(arena, lengths, t)
    nvr.check(L.nvr_kv_evict(dk.ptr, dv.ptr, ds.ptr, byref(m), 1, 8, block, 8, 48, 0, 0, arena.dev(np.array([[5], [6]], np.int32)).ptr, 1, new.ptr, kept.ptr, None, None))
    assert new.to_numpy((2,), np.int32).tolist() == [-1, 10]
    got = dk.to_numpy(k.shape, np.uint16)
    assert np.array_equal(got[:6], k[:6]) and np.array_equal(got[6, :10], k[4, :10]) and np.array_equal(got[6, 10:], k[6, 10:]) and np.array_equal(got[7], k[7])


# ------------------------------------------------------------------------------------------------------------ together, captured, on streams of their own, far into a pool
class Step:
    """One layer's decode step of a batch whose requests have adapters of their own and whose caches are held to a budget, then a token each: the framework's product, nvr_lora_add beside it,
    nvr_rope_rotate_store_kv, nvr_paged_attn_decode_scored, nvr_kv_evict, nvr_linear + nvr_lora_add for the output, logits, nvr_sample_uniform."""

    def __init__(self, arena, dtype, stream=None, seed=0, bound=128):
        rng = np.random.default_rng(seed)
        self.arena, self.dtype, self.stream, self.rng, self.bound = arena, dtype, stream, rng, bound
        typed(dtype)
        self.W, self.H, self.G, self.D, self.R, self.n, self.V, self.block, self.budget, self.first, self.last = 256, 4, 2, 64, 8, 3, 1024, 16, 48, 2, 8
        self.lengths = [60, 47, 30, 52, 48]
        B, self.w = len(self.lengths), np.dtype(kind(dtype)).itemsize
        N = (self.H + 2 * self.G) * self.D
        self.B, self.N = B, N

        def weights(*shape, std):
            return encode(rng.standard_normal(shape) * std, dtype)
        self.host = {"x": weights(B, self.W, std=1.0), "wqkv": weights(N, self.W, std=self.W ** -0.5), "wo": weights(self.W, self.H * self.D, std=(self.H * self.D) ** -0.5),
                     "head": weights(self.V, self.W, std=1.5 * self.W ** -0.5), "a1": weights(self.n, self.R, self.W, std=self.W ** -0.5), "b1": weights(self.n, N, self.R, std=0.5),
                     "a2": weights(self.n, self.R, self.H * self.D, std=(self.H * self.D) ** -0.5), "b2": weights(self.n, self.W, self.R, std=0.5)}
        self.dev = {k: arena.dev(v[1]) for k, v in self.host.items()}
        self.ids, self.scales = np.array([0, 2, -1, 1, 0], np.int32), np.array([0.5, 1.0, 2.0], np.float32)
        self.table, self.blocks = tables(rng, [n + 32 for n in self.lengths], self.block)
        k, v = (encode(rng.standard_normal((self.blocks, self.block, self.G, self.D)), dtype) for _ in range(2))
        self.k0, self.v0 = k[1], v[1]
        self.s0 = rng.random((self.blocks, self.G, self.block)).astype(np.float32)
        self.turns, self.amplitude = rope_turns("bands", self.D, factor=8.0, low=1.0, high=4.0)
        self.d = {"ids": arena.dev(self.ids), "scales": arena.dev(self.scales), "turns": arena.dev(self.turns), "table": arena.dev(self.table), "k": arena.dev(self.k0), "v": arena.dev(self.v0),
                  "scores": arena.dev(self.s0), "qkv": arena.space(B * N * self.w), "q": arena.space(B * self.H * self.D * self.w), "out": arena.space(B * self.H * self.D * self.w),
                  "o": arena.space(B * self.W * self.w), "logits": arena.space(B * self.V * 4), "new_lens": arena.space(B * 4), "kept": arena.space(B * self.G * self.budget * 4),
                  "token": arena.space(B * 8), "logprob": arena.space(B * 4), "ws_lora": arena.space(L.nvr_lora_workspace_bytes(B, self.H * self.D, N, self.R)),
                  "ws_attn": arena.space(L.nvr_paged_attn_scored_workspace_bytes(B, self.H, self.G, self.D, bound)), "ws_sample": arena.space(L.nvr_sample_uniform_workspace_bytes(B, self.V)),
                  "T": arena.dev(np.array([0.0, 0.7, 1.0, 1.3, 0.9], np.float32)), "tk": arena.dev(np.array([0, 20, 0, 50, 0], np.int64)), "tp": arena.dev(np.array([1, 1, 0.9, 0.95, 1], np.float32)),
                  "mp": arena.dev(np.array([0, 0, 0, 0.02, 0.05], np.float32)), "u": arena.space(B * 4), "pos": arena.space(B * 8), "slots": arena.space(B * 4), "lens": arena.space(B * 4), "scored": arena.space(B * 4)}
        self.positions = np.array([5000, 47, 123456, 52, 300], np.int64)

    def feed(self, lengths):
        """The step's small inputs: every sequence gets a key behind its `lengths`."""
        n = np.array(lengths, np.int32)
        slots = (self.table[np.arange(self.B), n // self.block] * self.block + n % self.block).astype(np.int32)
        self.uniform = self.rng.random(self.B).astype(np.float32)
        for name, a in (("lens", n + 1), ("scored", n), ("slots", slots), ("pos", self.positions), ("u", self.uniform)):
            a = np.ascontiguousarray(a)
            nvr.check(L.nvr_memcpy_h2d(self.d[name].ptr, a.ctypes.data, a.nbytes))
        self.slots = slots

    def launch(self):
        d, w, s = self.d, self.dev, self.stream
        B, N, W, H, G, D, R = self.B, self.N, self.W, self.H, self.G, self.D, self.R
        m = nvr.AttnMetaC(is_prefill=0, context_lens=d["lens"].ptr, block_tables=d["table"].ptr, max_blocks=self.table.shape[1], batch=B, max_context_len=self.bound)
        ws, q = self.w, d["qkv"].ptr
        nvr.check(L.nvr_linear(w["x"].ptr, W, w["wqkv"].ptr, B, W, N, q, 0, s))
        nvr.check(L.nvr_lora_add(w["x"].ptr, W, w["a1"].ptr, w["b1"].ptr, d["scales"].ptr, d["ids"].ptr, self.n, B, W, N, R, q, N, q, N, d["ws_lora"].ptr, s))
        nvr.check(L.nvr_rope_rotate_store_kv(q, N, q + H * D * ws, N, q + (H + G) * D * ws, N, d["pos"].ptr, d["slots"].ptr, B, H, G, D, D, 0, d["turns"].ptr, self.amplitude, d["q"].ptr, H * D, None, 0,
                                             d["k"].ptr, d["v"].ptr, self.blocks * self.block, s))
        nvr.check(L.nvr_paged_attn_decode_scored(d["q"].ptr, H * D, d["k"].ptr, d["v"].ptr, byref(m), H, G, D, self.block, self.blocks, D ** -0.5, d["scores"].ptr, d["scored"].ptr, 0.9, d["scores"].ptr,
                                                 d["out"].ptr, d["ws_attn"].ptr, s))
        nvr.check(L.nvr_kv_evict(d["k"].ptr, d["v"].ptr, d["scores"].ptr, byref(m), G, D, self.block, self.blocks, self.budget, self.first, self.last, None, 0, d["new_lens"].ptr, d["kept"].ptr, None, s))
        nvr.check(L.nvr_linear(d["out"].ptr, H * D, w["wo"].ptr, B, H * D, W, d["o"].ptr, 0, s))
        nvr.check(L.nvr_lora_add(d["out"].ptr, H * D, w["a2"].ptr, w["b2"].ptr, d["scales"].ptr, d["ids"].ptr, self.n, B, H * D, W, R, d["o"].ptr, W, d["o"].ptr, W, d["ws_lora"].ptr, s))
        nvr.check(L.nvr_linear(d["o"].ptr, W, w["head"].ptr, B, W, self.V, d["logits"].ptr, 1, s))
        nvr.check(L.nvr_sample_uniform(d["logits"].ptr, self.V, B, self.V, d["T"].ptr, d["tk"].ptr, d["tp"].ptr, d["mp"].ptr, d["u"].ptr, d["token"].ptr, d["logprob"].ptr, d["ws_sample"].ptr, s))

    NAMES = (("qkv", None), ("q", None), ("out", None), ("o", None), ("k", None), ("v", None), ("scores", np.uint32), ("logits", np.uint32), ("new_lens", np.int32), ("kept", np.int32),
             ("token", np.int64), ("logprob", np.uint32))

    def answers(self):
        return {n: self.d[n].to_numpy((self.d[n].nbytes // np.dtype(t or kind(self.dtype)).itemsize,), t or kind(self.dtype)) for n, t in self.NAMES}

    def restore(self):
        for name, a in (("k", self.k0), ("v", self.v0), ("scores", self.s0)):
            nvr.check(L.nvr_memcpy_h2d(self.d[name].ptr, a.ctypes.data, a.nbytes))


@pytest.mark.parametrize("dtype,bound", [("float16", 128), ("bfloat16", 128), ("float32", 128), ("float16", 2000), ("float32", 2000)])
def test_a_step_of_all_of_them(arena, dtype, bound):
    """Three steps; each stage against its definition on what the stage in front of it left."""
    st = Step(arena, dtype, bound=bound)
    lengths = list(st.lengths)
    B, N, W, H, G, D = st.B, st.N, st.W, st.H, st.G, st.D
    cache_k, cache_v = st.k0.copy(), st.v0.copy()
    scores = st.s0.astype(np.float64)
    up = HALF_STEP[dtype]
    for _ in range(3):
        st.feed(lengths)
        st.launch()
        nvr.synchronize()
        a = st.answers()
        val = {k: decode(v, dtype) for k, v in a.items() if k in ("qkv", "q", "out", "o")}
        x, h = st.host["x"][0], {k: v[0] for k, v in st.host.items()}

        def adapted(inp, base_w, A, Bm):
            base = inp @ base_w.T
            add = np.zeros_like(base)
            for b in range(B):
                if st.ids[b] >= 0:
                    add[b] = st.scales[st.ids[b]] * (inp[b] @ A[st.ids[b]].T) @ Bm[st.ids[b]].T
            return base, add
        # projection: rounded once behind the product and once behind the adapters; sums of W products in 32 bits
        base, add = adapted(x, h["wqkv"], h["a1"], h["b1"])
        size = np.abs(x) @ np.abs(h["wqkv"]).T
        within(val["qkv"].reshape(B, N), base + add, up * (np.abs(base) + np.abs(base + add)) * 1.01 + (W + 32) * F32 * size * 3 + SMALLEST[dtype] * 2 + 2.0 ** -15 * np.abs(add).max() * (dtype == "bfloat16"), "projection")
        qkv = val["qkv"].reshape(B, H + 2 * G, D)
        want = rope(qkv[:, :H + G], st.positions, st.turns, st.amplitude, False)
        near = up * np.abs(want) * 1.01 + 8 * F32 * np.abs(qkv).max() + SMALLEST[dtype]
        within(val["q"].reshape(B, H, D), want[:, :H], near[:, :H], "rotated queries")
        shape = (st.blocks, st.block, G, D)
        got_k, got_v, got_s = a["k"].reshape(shape), a["v"].reshape(shape), a["scores"].view(np.float32).reshape(st.s0.shape)
        for b in range(B):
            page, row = divmod(int(st.slots[b]), st.block)
            cache_v[page, row] = a["qkv"].reshape(B, H + 2 * G, D)[b, H + G:]
            cache_k[page, row] = encode(want[b, H:], dtype)[1]
        new = []
        for b in range(B):
            n = lengths[b] + 1
            j = np.arange(n)
            page, row = st.table[b, j // st.block], j % st.block
            kk, vv = decode(cache_k[page, row], dtype), decode(cache_v[page, row], dtype)
            out, weight = attend(val["q"].reshape(B, H, D)[b], kk, vv, D ** -0.5)
            # a key that was rounded the other way moves its score by a step: 2^-10 of |q||k| at most in 16 bits
            within(val["out"].reshape(B, H, D)[b], out, up * np.abs(out) * 1.01 + (4 * up + 200 * F32) * np.abs(vv).max() + SMALLEST[dtype], "attention")
            scores[page, :, row] = np.where(j[:, None] < lengths[b], 0.9 * scores[page, :, row], 0.0) + weight
            m = min(n, st.budget)
            for g in range(G):
                kept = a["kept"].reshape(B, G, st.budget)[b, g]
                assert (kept[m:] == -1).all() and (np.diff(kept[:m]) > 0).all()
                if n > st.budget:
                    assert np.array_equal(kept[:st.first], np.arange(st.first)) and np.array_equal(kept[m - st.last:m], np.arange(n - st.last, n))
                    # what was left out scores no more than what was kept, but for the tolerance of the scores
                    out_of = np.setdiff1d(np.arange(st.first, n - st.last), kept)
                    inside = kept[st.first:m - st.last]
                    assert scores[page[out_of], g, row[out_of]].max() <= scores[page[inside], g, row[inside]].min() + 16 * up
                i = np.arange(m)
                dst, src = (st.table[b, i // st.block], i % st.block), (page[kept[:m]], row[kept[:m]])
                assert np.array_equal(got_v[dst[0], dst[1], g], cache_v[src[0], src[1], g])
                within(decode(got_k[dst[0], dst[1], g], dtype), decode(cache_k[src[0], src[1], g], dtype), 2.02 * up * np.abs(decode(cache_k[src[0], src[1], g], dtype)) + 16 * F32 * np.abs(qkv).max(), "keys")
                within(got_s[dst[0], g, dst[1]].astype(np.float64), scores[src[0], g, src[1]], np.full(m, 16 * up), "scores")
            new.append(m)
        assert a["new_lens"].tolist() == new
        base, add = adapted(val["out"].reshape(B, -1), h["wo"], h["a2"], h["b2"])
        within(val["o"].reshape(B, W), base + add, up * (np.abs(base) + np.abs(base + add)) * 1.01 + 600 * F32 * (np.abs(val["out"]).max() * 20) + SMALLEST[dtype] * 2 + 2.0 ** -15 * np.abs(add).max() * (dtype == "bfloat16"), "output")
        logits = a["logits"].view(np.float32).reshape(B, st.V)
        T, k, p, m = ([0.0, 0.7, 1.0, 1.3, 0.9], [0, 20, 0, 50, 0], [1, 1, 0.9, 0.95, 1], [0, 0, 0, 0.02, 0.05])
        assert a["token"].tolist() == [sample(logits[b], float(np.float32(T[b])), k[b], float(np.float32(p[b])), float(np.float32(m[b])), float(st.uniform[b]))[0] for b in range(B)]
        # the next step goes on from what is there
        cache_k, cache_v, scores = got_k.copy(), got_v.copy(), got_s.astype(np.float64)
        lengths = new
        st.positions = st.positions + 1


@pytest.mark.parametrize("dtype,bound", [("bfloat16", 128), ("float32", 128), ("bfloat16", 2000), ("float16", 2000)])
def test_a_captured_step_replays(arena, dtype, bound):
    """The step in a graph, replayed with other inputs and eager work between: the bits of the eager step each time."""
    stream = C.c_void_p()
    nvr.check(L.nvr_stream_create(byref(stream)))
    st = Step(arena, dtype, stream, bound=bound)
    st.feed(st.lengths)
    st.launch()
    nvr.check(L.nvr_stream_synchronize(stream))
    graph = C.c_void_p()
    nvr.check(L.nvr_graph_capture_begin(stream))
    st.launch()
    nvr.check(L.nvr_graph_capture_end(stream, byref(graph)))
    for turn in range(4):
        lengths = [min(n + 3 * turn, 75) for n in st.lengths]
        st.positions = st.positions + 17
        st.restore()
        st.feed(lengths)
        st.launch()
        nvr.check(L.nvr_stream_synchronize(stream))
        eager = st.answers()
        st.restore()
        for name in ("qkv", "q", "out", "o", "logits", "token", "kept", "new_lens"):
            nvr.check(L.nvr_device_memset(st.d[name].ptr, SENTINEL, st.d[name].nbytes))
        nvr.synchronize()
        nvr.check(L.nvr_graph_launch(graph, stream))
        nvr.check(L.nvr_stream_synchronize(stream))
        again = st.answers()
        for name in eager:
            assert np.array_equal(eager[name], again[name]), (turn, name)
    nvr.check(L.nvr_graph_destroy(graph))
    nvr.check(L.nvr_stream_destroy(stream))


def test_two_streams_at_once(arena):
    """Two steps on streams of their own, with workspaces of their own, in flight together: the bits of each alone."""
    streams = [C.c_void_p(), C.c_void_p()]
    for s in streams:
        nvr.check(L.nvr_stream_create(byref(s)))
    steps = [Step(arena, "float16", s, seed=i) for i, s in enumerate(streams)]
    alone = []
    for st in steps:
        st.feed(st.lengths)
        st.launch()
        nvr.synchronize()
        alone.append(st.answers())
        st.restore()
    nvr.synchronize()
    for st in steps:
        st.launch()
    nvr.synchronize()
    for st, want in zip(steps, alone):
        got = st.answers()
        for name in want:
            assert np.array_equal(want[name], got[name]), name
    for s in streams:
        nvr.check(L.nvr_stream_destroy(s))


def test_pool_beyond_32_bits_of_numbers(arena):
    """Blocks 2^31 numbers and more into caches of 4.9 GB: stored, attended to, evicted in place and into other blocks."""
    typed("float16")
    G, D, block, blocks, H = 8, 128, 256, 9400, 8
    row = G * D
    assert blocks * block * row > 1 << 31
    k, v, s = (nvr.DeviceBuffer(n) for n in (blocks * block * row * 2, blocks * block * row * 2, blocks * G * block * 4))
    rng = np.random.default_rng(0)
    table = np.array([[9399, 3, 9300, 8800]], np.int32)
    to = np.array([[9350, 9399 - 1]], np.int32)
    n = 900
    hk, hv, hs = rng.standard_normal((4, block, G, D)).astype(np.float16), rng.standard_normal((4, block, G, D)).astype(np.float16), rng.random((4, G, block)).astype(np.float32)

    def put():
        for i, p in enumerate(table[0]):
            for buf, a, size in ((k, hk, block * row * 2), (v, hv, block * row * 2), (s, hs, G * block * 4)):
                c = np.ascontiguousarray(a[i])
                nvr.check(L.nvr_memcpy_h2d(buf.ptr + int(p) * size, c.ctypes.data, size))

    def block_of(buf, p, shape, t):
        a = np.empty(shape, t)
        nvr.check(L.nvr_memcpy_d2h(a.ctypes.data, buf.ptr + int(p) * a.nbytes, a.nbytes))
        return a
    put()
    # the newest key by the rotation, in the far block
    x = rng.standard_normal((1, H + 2 * G, D)).astype(np.float16)
    turns, _ = rope_turns("plain", D)
    page, at = table[0, (n - 1) // block], (n - 1) % block
    dx, q = arena.dev(x), arena.space(H * D * 2)
    nvr.check(L.nvr_rope_rotate_store_kv(dx.ptr, (H + 2 * G) * D, dx.ptr + H * D * 2, (H + 2 * G) * D, dx.ptr + (H + G) * D * 2, (H + 2 * G) * D, arena.dev(np.array([n - 1])).ptr,
                                         arena.dev(np.array([page * block + at], np.int32)).ptr, 1, H, G, D, D, 0, arena.dev(turns).ptr, 1.0, q.ptr, H * D, None, 0, k.ptr, v.ptr, blocks * block, None))
    want = rope(x[:, H:H + G].astype(np.float64), np.array([n - 1]), turns, 1.0, False)[0]
    stored = block_of(k, page, (block, G, D), np.float16)
    within(stored[at].astype(np.float64), want, HALF_STEP["float16"] * np.abs(want) + 1e-5, "stored key")
    assert np.array_equal(block_of(v, page, (block, G, D), np.float16)[at], x[0, H + G:])
    hk[(n - 1) // block, at], hv[(n - 1) // block, at] = stored[at], x[0, H + G:]
    m = nvr.AttnMetaC(is_prefill=0, context_lens=arena.dev(np.array([n], np.int32)).ptr, block_tables=arena.dev(table).ptr, max_blocks=4, batch=1, max_context_len=n)
    out = arena.space(H * D * 2)
    nvr.check(L.nvr_paged_attn_decode_scored(q.ptr, H * D, k.ptr, v.ptr, byref(m), H, G, D, block, blocks, D ** -0.5, s.ptr, None, 1.0, s.ptr, out.ptr,
                                             arena.space(L.nvr_paged_attn_scored_workspace_bytes(1, H, G, D, n)).ptr, None))
    j = np.arange(n)
    wout, weight = attend(q.to_numpy((H, D), np.float16).astype(np.float64), hk[j // block, j % block].astype(np.float64), hv[j // block, j % block].astype(np.float64), D ** -0.5)
    within(out.to_numpy((H, D), np.float16).astype(np.float64), wout, 2 * HALF_STEP["float16"] * np.abs(wout) + 2e-5, "far attention")
    for i in range(4):
        hs[i] = block_of(s, table[0, i], (G, block), np.float32)
    new, kept = arena.space(4), arena.space(G * 400 * 4)
    for dest in (to, None):
        put()
        nvr.check(L.nvr_kv_evict(k.ptr, v.ptr, s.ptr, byref(m), G, D, block, blocks, 400, 4, 64, arena.dev(dest).ptr if dest is not None else None, 2 if dest is not None else 0, new.ptr, kept.ptr, None, None))
        names = (dest if dest is not None else table)[0]
        got_k, got_s = [block_of(k, p, (block, G, D), np.float16) for p in names[:2]], [block_of(s, p, (G, block), np.float32) for p in names[:2]]
        for g in range(G):
            mine = evict(hs[j // block, g, j % block], 400, 4, 64)
            assert np.array_equal(kept.to_numpy((G, 400), np.int32)[g], mine)
            i = np.arange(400)
            assert np.array_equal(np.array(got_k)[i // block, i % block, g], hk[mine // block, mine % block, g])
            assert np.array_equal(np.array(got_s)[i // block, g, i % block], hs[mine // block, g, mine % block])
    nvr.synchronize()


def test_lora_of_thousands_of_adapters(arena):
    rng = np.random.default_rng(7)
    lora_case(arena, "float16", 3000, 16, 24, 4, 8191, rng.integers(-1, 8191, 3000))
    lora_case(arena, "bfloat16", 60, 16, 24, 4, 8191, rng.integers(-1, 8191, 60))


def test_sample_of_many_short_rows(arena):
    rng = np.random.default_rng(8)
    check_sample(arena, rng.standard_normal((700, 33)) * 2, 1.0, 5, 0.9, 0.01, rng.random(700).astype(np.float32))
    check_sample(arena, rng.standard_normal((300, 17000)) * 2, 1.0, 0, 0.9, 0.0, rng.random(300).astype(np.float32))


@pytest.mark.parametrize("B", [1, 256])
def test_sample_long_prefixes(arena, B):
    """Prefixes of hundreds to tens of thousands of tokens, alone and where chunks are large; twice, for the same bits."""
    rng = np.random.default_rng(9)
    V = 50257
    x = rng.standard_normal((B, V)) * 2
    x[:, rng.integers(0, V, 30)] += 7
    for k, p, m in ((300, 1.0, 0.0), (1500, 0.9, 0.0), (5000, 1.0, 0.0), (20000, 0.97, 0.0), (0, 0.5, 0.0), (0, 0.99, 0.0), (0, 0.9, 0.0005), (0, 1.0, 0.0002), (2500, 0.999, 0.001)):
        u = rng.random(B).astype(np.float32)
        u[0] = 0 if B == 1 and k else u[0]
        n = min(B, 24)
        args = [np.broadcast_to(np.asarray(a, t), (B,)) for a, t in ((0.9, np.float32), (k, np.int64), (p, np.float32), (m, np.float32), (u, np.float32))]
        ids, lp = sample_rows(arena, x.astype(np.float32), *args)
        again = sample_rows(arena, x.astype(np.float32), *args)
        assert np.array_equal(ids, again[0]) and np.array_equal(lp.view(np.uint32), again[1].view(np.uint32))
        for r in range(n):
            want = sample(x[r].astype(np.float32), float(np.float32(0.9)), k, float(np.float32(p)), float(np.float32(m)), float(u[r]))
            assert ids[r] == want[0], (k, p, m, r)
            assert abs(lp[r] - want[1]) <= 2.0 ** -23 * max(1, abs(want[1])), (k, p, m, r)


def test_sample_whole_rows_of_equal_logits(arena):
    """Every logit the same, and two values in turn: ends of prefixes are told by the index alone, in one bin of more tokens than LDS holds."""
    rng = np.random.default_rng(10)
    for V in (2049, 20000, 70001):
        same = np.zeros((2, V), np.float32)
        two = np.where(np.arange(V) % 2 == 0, 0.5, 0.5 + 1e-6).astype(np.float32)[None].repeat(2, 0)
        for x in (same, two):
            for k, p, m in ((0, 1.0, 0.0), (1, 1.0, 0.0), (1777, 1.0, 0.0), (0, 0.25, 0.0), (1999, 0.5, 0.0), (0, 1.0, 1.0), (V - 1, 1.0, 0.0)):
                check_sample(arena, x, 1.0, k, p, m, rng.random(2).astype(np.float32))


@pytest.mark.parametrize("T,K,N,R,n", [(200000, 16, 16, 4, 5), (200000, 8, 16, 130, 3), (70000, 8, 40, 4, 5000)])
def test_lora_of_many_rows(arena, T, K, N, R, n):
    """More rows than one pass of the grouping takes, in tiles of 64 rows and of 16."""
    lora_case(arena, "float16", T, K, N, R, n, np.random.default_rng(T + R).integers(-1, n, T))


@pytest.mark.parametrize("dtype,T,K,N,R,n", [("float32", 5, 4096, 64, 16, 2), ("float32", 5, 2048, 64, 16, 2), ("bfloat16", 64, 4096, 4104, 32, 64), ("float16", 64, 4096, 4104, 17, 2), ("bfloat16", 64, 72, 8, 32, 64),
                                             ("float16", 1, 4097, 31, 32, 1), ("float16", 1, 4096, 31, 32, 1)])
def test_lora_one_launch_and_two(arena, dtype, T, K, N, R, n):
    """Sizes on either side of what one launch takes."""
    lora_case(arena, dtype, T, K, N, R, n, np.random.default_rng(T + K).integers(-1, n, T))


def test_lora_into_its_own_input(arena):
    """y may be x: all of x is read before any of y is written."""
    typed("float32")
    rng = np.random.default_rng(3)
    T, K, R = 24, 1024, 8
    x, base = rng.standard_normal((2, T, K)).astype(np.float32)
    A, B = rng.standard_normal((1, R, K)).astype(np.float32) / 32, rng.standard_normal((1, K, R)).astype(np.float32)
    y = arena.dev(x)
    nvr.check(L.nvr_lora_add(y.ptr, K, arena.dev(A).ptr, arena.dev(B).ptr, None, arena.dev(np.zeros(T, np.int32)).ptr, 1, T, K, K, R, arena.dev(base).ptr, K, y.ptr, K,
                             arena.space(L.nvr_lora_workspace_bytes(T, K, K, R)).ptr, None))
    v = x.astype(np.float64) @ A[0].T.astype(np.float64)
    want = base + v @ B[0].T.astype(np.float64)
    # sums of K and R products in 32 bits
    within(y.to_numpy((T, K), np.float32).astype(np.float64), want, F32 * ((K + R) * (np.abs(x) @ np.abs(A[0]).T) @ np.abs(B[0]).T + np.abs(want)) + 1e-30, "into x")


@pytest.mark.parametrize("out_of_place", [False, True])
def test_evict_of_more_keys_than_lds_holds(arena, out_of_place):
    evict_case(arena, "bfloat16", [40000, 32769, 32768, 100], 1, 64, 256, 20000, 4, 700, out_of_place)


@pytest.mark.parametrize("dtype,T,K,N,R,n", [("float16", 65, 64, 40, 16, 1), ("bfloat16", 512, 1024, 264, 32, 7), ("float16", 513, 72, 33, 20, 1022), ("float16", 513, 72, 33, 20, 1023), ("float32", 1024, 64, 128, 8, 3),
                                             ("bfloat16", 1024, 64, 128, 96, 40), ("bfloat16", 1025, 64, 128, 8, 3), ("float32", 1000, 16, 16, 90, 1000), ("bfloat16", 40, 1024, 72, 96, 3), ("float16", 64, 200, 1000, 49, 64)])
def test_lora_rows_found_by_each_workgroup(arena, dtype, T, K, N, R, n):
    rng = np.random.default_rng(T + n)
    a = lora_case(arena, dtype, T, K, N, R, n, rng.integers(-1, n, T), seed=1)
    rng = np.random.default_rng(T + n)
    assert np.array_equal(a, lora_case(arena, dtype, T, K, N, R, n, rng.integers(-1, n, T), seed=1))
    lora_case(arena, dtype, T, K, N, R, n, np.full(T, n - 1))
    lora_case(arena, dtype, T, K, N, R, n, np.full(T, -1))


def test_copies_to_the_host_wait_for_every_stream(arena):
    """What a stream still has to write is in a copy to the host that follows its launches: products for some milliseconds, then a token a row."""
    typed("float16")
    stream = C.c_void_p()
    nvr.check(L.nvr_stream_create(byref(stream)))
    T, K = 4096, 4096
    x, w, y = arena.space(T * K * 2, 0), arena.space(K * K * 2, 0), arena.space(T * K * 2, 0)
    B, V = 4, 1000
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((B, V)).astype(np.float32)
    d, u, ids, ws = arena.dev(logits), arena.dev(np.zeros(B, np.float32)), arena.space(B * 8), arena.space(L.nvr_sample_uniform_workspace_bytes(B, V))
    t = arena.dev(np.zeros(B, np.float32))
    nvr.synchronize()
    for _ in range(30):
        nvr.check(L.nvr_linear(x.ptr, K, w.ptr, T, K, K, y.ptr, 0, stream))
    nvr.check(L.nvr_sample_uniform(d.ptr, V, B, V, t.ptr, None, None, None, u.ptr, ids.ptr, None, ws.ptr, stream))
    got = np.empty(B, np.int64)
    nvr.check(L.nvr_memcpy_d2h(got.ctypes.data, ids.ptr, got.nbytes))
    assert got.tolist() == logits.argmax(1).tolist()
    nvr.check(L.nvr_stream_destroy(stream))


@pytest.mark.parametrize("out_of_place", [False, True])
def test_evict_without_a_bound_on_contexts(arena, out_of_place):
    evict_case(arena, "float16", [300, 40, 299], 2, 64, 16, 100, 4, 32, out_of_place, max_context=2 ** 31 - 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G,D,block", [(16, 1, 64, 16), (4, 2, 128, 256), (3, 1, 256, 7), (32, 8, 128, 64), (5, 5, 64, 1)])
def test_scored_attention_of_short_contexts(arena, dtype, H, G, D, block):
    """Contexts of up to 128 keys, which one launch answers: the same bits as where the bound on contexts asks for two."""
    lengths = [0, 1, 128, 2, 15, 16, 17, 0, 31, 32, 33, 63, 64, 65, 100, 127, 128]
    one = scored_case(arena, dtype, lengths, H, G, D, block, poison=True)
    two = scored_case(arena, dtype, lengths, H, G, D, block, poison=True, max_context=257)
    used = [i for i, n in enumerate(lengths) if n]
    assert np.array_equal(one[0][used], two[0][used]) and np.array_equal(one[1].view(np.uint32), two[1].view(np.uint32))
    scored_case(arena, dtype, [60, 128, 9], H, G, D, block, scored=[0, 999, -3], decay=0.25, in_place=True, q_gap=8)
    if block < 128:
        scored_case(arena, dtype, [128, 100, 5], H, G, D, block, bad=[(0, 0, -1), (0, 1, 1 << 30), (2, 0, -7)])
    scored_case(arena, dtype, [100, 7], H, G, D, block, max_context=50)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,G,D,B,longest", [(8, 4, 64, 70, 511), (8, 8, 128, 40, 512), (8, 4, 64, 70, 513), (4, 1, 128, 20, 400), (16, 1, 256, 9, 256)])
def test_scored_attention_of_contexts_around_one_launch(arena, dtype, H, G, D, B, longest):
    """Sequences enough for the chip and not, contexts on either side of what one launch takes."""
    rng = np.random.default_rng(longest + B)
    lengths = rng.integers(0, longest, B).tolist()
    lengths[3], lengths[5] = longest, 0
    scored_case(arena, dtype, lengths, H, G, D, 64, poison=True)


@pytest.mark.parametrize("out_of_place", [False, True])
@pytest.mark.parametrize("dtype,lengths,G,D,block,budget,first,last", [("float16", [300, 64, 0, 65, 1000], 3, 128, 16, 64, 4, 20), ("float32", [300, 128, 129], 2, 256, 256, 64, 0, 0), ("float32", [300, 70], 2, 256, 256, 65, 0, 64),
                                                                      ("bfloat16", [4000, 5000], 1, 8, 7, 4096, 4, 100), ("bfloat16", [5000, 20], 1, 8, 1, 4097, 4, 100), ("float16", [700, 3], 2, 40, 64, 256, 1, 1),
                                                                      ("float16", [33000, 40], 1, 64, 256, 40, 4, 4), ("bfloat16", [1000, 257], 2, 128, 256, 257, 4, 4)])
def test_evict_of_few_rows(arena, dtype, lengths, G, D, block, budget, first, last, out_of_place):
    """Rows on either side of what the first launch moves itself."""
    evict_case(arena, dtype, lengths, G, D, block, budget, first, last, out_of_place)


@pytest.mark.parametrize("V", [2049, 20000, 151936])
@pytest.mark.parametrize("T", [0.7, 1.3, 100.0])
def test_sample_min_p_of_one_keeps_the_largest(arena, V, T):
    """The largest logits weigh exactly 1, wherever they lie in their cell: rows with more of them than a chunk's list holds, and rows so flat that every token is near the largest."""
    rng = np.random.default_rng(V)
    x = np.stack([np.full(V, 2.3), np.full(V, 5.1), np.full(V, -0.9), rng.standard_normal(V), np.where(rng.random(V) < 0.5, 5.1, 5.0)])
    for k, p, m in ((0, 1.0, 1.0), (0, 1.0, 5.0), (0, 0.7, 1.0), (V // 2, 1.0, 1.0), (V - 1, 0.9, 1.0)):
        check_sample(arena, x, T, k, p, m, rng.random(5).astype(np.float32))


@pytest.mark.parametrize("most,B,V", [((256, 10000), 127, 10000), ((256, 16384), 100, 16384), ((200, 20000), 100, 9000), ((4, 151936), 4, 98304)])
def test_sample_in_the_workspace_of_a_larger_step(arena, most, B, V):
    """A step of fewer rows, or of a smaller vocabulary, in the space that the largest asked for: nothing behind it is written."""
    rng = np.random.default_rng(B + V)
    x = (rng.standard_normal((B, V)) * 2).astype(np.float32)
    u = rng.random(B).astype(np.float32)
    size, guard = L.nvr_sample_uniform_workspace_bytes(*most), 1 << 16
    assert size >= L.nvr_sample_uniform_workspace_bytes(B, V)
    ws, ids = arena.space(size + guard), arena.space(B * 8)
    T, k, p, m = (np.resize(np.array(a, t), B) for a, t in (([0.8, 1.0], np.float32), ([0, 50, 0], np.int64), ([0.9, 1.0], np.float32), ([0.0, 0.02, 0.0], np.float32)))
    nvr.check(L.nvr_sample_uniform(arena.dev(x).ptr, V, B, V, *(arena.dev(a).ptr for a in (T, k, p, m, u)), ids.ptr, None, ws.ptr, None))
    assert ids.to_numpy((B,), np.int64).tolist() == [sample(x[r], float(T[r]), int(k[r]), float(p[r]), float(m[r]), float(u[r]))[0] for r in range(B)]
    assert (ws.to_numpy((size + guard,), np.uint8)[size:] == SENTINEL).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_scored_attention_pages_outside_the_pool_in_two_launches(arena, dtype):
    """As above with a bound of more than 512 keys, where a second launch turns scores into weights: pages missing at a tile's begin and end, a whole tile, whole units, all of a sequence, the newest key's."""
    lengths = [600, 600, 600, 140, 20, 600]
    bad = [(0, 0, -1), (0, 2, -1), (0, 3, 1 << 20), (0, 37, -1)] + [(1, i, -7) for i in range(8, 24)] + [(2, i, -1) for i in range(2, 38)] + [(3, i, 1 << 30) for i in range(9)] + [(4, 1, -1)]
    for in_place in (False, True):
        scored_case(arena, dtype, lengths, 4, 2, 64, 16, bad=bad, in_place=in_place, poison=True)
    scored_case(arena, dtype, [600, 1300], 8, 1, 128, 64, bad=[(0, 9, -1), (1, 0, -1), (1, 3, 1 << 30), (1, 20, -1)], poison=True)
    scored_case(arena, dtype, [600, 530], 4, 2, 64, 7, bad=[(0, i, -1) for i in range(0, 86, 3)] + [(1, 75, -1), (1, 40, -2)], poison=True)      # (keys of a request of four in different pages)
    rng = np.random.default_rng(6)
    lengths = rng.integers(1, 700, 80).tolist()                    # more than 64 sequences: the shares are counted another way
    scored_case(arena, dtype, lengths, 4, 2, 64, 64, bad=[(b, int(rng.integers(0, -(-n // 64))), -1) for b, n in enumerate(lengths) if b % 3 == 0])


def test_scored_attention_cuts_contexts_at_their_bound_in_two_launches(arena):
    scored_case(arena, "float16", [50, 2000, 700, 701], 4, 2, 64, 16, max_context=701, scored=[49, 1999, 699, 700])
    scored_case(arena, "float32", [2000, 3, 5000], 4, 2, 64, 16, max_context=1025)
    scored_case(arena, "bfloat16", [900, 40], 4, 2, 64, 16, max_context=1 << 16)


def test_scored_attention_where_no_sequence_can_have_keys(arena):
    """A bound of 0 keys: outputs of 0, scores as they were, and no workspace (its size is 0)."""
    for dtype in DTYPES:
        typed(dtype)
        w = np.dtype(kind(dtype)).itemsize
        B, H, G, D, block = 3, 4, 2, 64, 16
        assert L.nvr_paged_attn_scored_workspace_bytes(B, H, G, D, 0) == 0
        m = meta(arena, [5, 0, 300], np.zeros((B, 4), np.int32), 0)
        q, kv, out = arena.space(B * H * D * w, 0), arena.space(block * G * D * w, 0), arena.space(B * H * D * w)
        old, new = arena.space(G * block * 4, 0), arena.space(G * block * 4)
        nvr.check(L.nvr_paged_attn_decode_scored(q.ptr, H * D, kv.ptr, kv.ptr, byref(m), H, G, D, block, 1, 0.125, old.ptr, None, 0.5, new.ptr, out.ptr, None, None))
        assert (out.to_numpy((B * H * D * w,), np.uint8) == 0).all() and (new.to_numpy((G * block * 4,), np.uint8) == SENTINEL).all()


FIRST = """
import sys
sys.path[:0] = [%r, %r]
import ctypes as C
import numpy as np
from serving_util import Arena, byref
import test_serving_gpu as t
nvr, L = t.nvr, t.L
nvr.check(L.nvr_device_set(0))
arena, stream, graph = Arena(), C.c_void_p(), C.c_void_p()
nvr.check(L.nvr_stream_create(byref(stream)))
st = t.Step(arena, %r, stream, bound=%d)
st.feed(st.lengths)
nvr.synchronize()
nvr.check(L.nvr_graph_capture_begin(stream))
st.launch()
nvr.check(L.nvr_graph_capture_end(stream, byref(graph)))
answers = []
for turn in range(3):
    st.restore()
    nvr.check(L.nvr_graph_launch(graph, stream))
    nvr.check(L.nvr_stream_synchronize(stream))
    answers.append(st.answers())
    st.restore()
    st.launch()
    nvr.check(L.nvr_stream_synchronize(stream))
    answers.append(st.answers())
for a in answers:
    for name in a:
        assert np.array_equal(a[name], answers[-1][name]), name
nvr.check(L.nvr_graph_destroy(graph))
print("captured first: ok")
"""


@pytest.mark.parametrize("dtype,bound", [("float16", 128), ("bfloat16", 2000), ("float32", 128), ("float32", 2000)])
def test_a_first_call_may_be_captured(dtype, bound):
    """A process whose very first calls of these operators are captured: nothing is left to an eager call before."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    r = subprocess.run([sys.executable, "-c", FIRST % (os.path.dirname(here), here, dtype, bound)], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=100)
    assert r.returncode == 0 and "captured first: ok" in r.stdout, r.stderr[-3000:]


# ------------------------------------------------------------------------------------------------------------ the largest sizes that are accepted
def test_rope_of_as_many_tokens_as_are_accepted(arena):
    rng = np.random.default_rng(20)
    typed("float16")
    T = 1 << 23
    bits = rng.integers(0, 0x7000, (T, 3, 2), dtype=np.uint16)     # q, k and v of one head of 2
    positions = rng.integers(0, 1 << 40, T)
    turns = np.array([0.1591549430918953])
    slots = (np.arange(T)[::-1] + 3).astype(np.int32)
    d, out, cache = arena.dev(bits), arena.space(T * 4), [arena.space((T + 3) * 4) for _ in range(2)]
    nvr.check(L.nvr_rope_rotate_store_kv(d.ptr, 6, d.ptr + 4, 6, d.ptr + 8, 6, arena.dev(positions).ptr, arena.dev(slots).ptr, T, 1, 1, 2, 2, 0, arena.dev(turns).ptr, 1.0, out.ptr, 2, None, 0,
                                         cache[0].ptr, cache[1].ptr, T + 3, None))
    x = bits[:, :2].view(np.float16).astype(np.float64)
    want = rope(x, positions, turns, 1.0, False)
    tol = 4 * F32 * 2 * np.abs(x).max(-1, keepdims=True) + HALF_STEP["float16"] * np.abs(want) * (1 + 2 ** -10) + SMALLEST["float16"]
    fits = np.abs(want) < 65000                                    # (float16 ends at 65504)
    k = cache[0].to_numpy((T + 3, 2), np.float16)[3:][::-1].astype(np.float64)
    for i, got in enumerate((out.to_numpy((T, 2), np.float16).astype(np.float64), k)):
        ok = np.abs(got - want[:, i]) <= tol[:, i]
        assert (ok | ~fits[:, i]).all()
    v = cache[1].to_numpy((T + 3, 2), np.uint16)
    assert np.array_equal(v[3:][::-1], bits[:, 2]) and (v[:3] == 0x7B7B).all()


@pytest.mark.parametrize("dtype,T,K,N,R,n", [("bfloat16", 3, 1 << 22, 40, 4, 2), ("float32", 70, 1 << 20, 8, 3, 2), ("float16", 3, 40, 1 << 22, 4, 2), ("bfloat16", 2, 256, 1 << 22, 16, 1), ("float16", 1 << 19, 8, 16, 4, 5),
                                             ("float16", 1 << 19, 8, 8, 130, 1)])
def test_lora_of_the_largest_sizes(arena, dtype, T, K, N, R, n):
    lora_case(arena, dtype, T, K, N, R, n, np.arange(T) % (n + 1) - 1)


def test_sample_of_as_many_logits_as_are_accepted(arena):
    """2^22 logits: 256 chunks of a row, indices of 22 bits; prefixes that end among equal logits far out, and in the lists and the row."""
    rng = np.random.default_rng(21)
    V = 1 << 22
    x = np.stack([rng.standard_normal(V) * 2, np.full(V, 1.7), (rng.integers(0, 40, V) * 0.05)]).astype(np.float32)
    x[0, rng.integers(0, V, 30)] += 9
    for k, p, m, u in ((0, 1.0, 0.0, 1 - 2.0 ** -24), (0, 0.75, 0.0, 0.99), (3000001, 1.0, 0.0, 0.9999), (50, 0.9, 0.0, 0.5), (1500, 1.0, 0.0, 0.8), (0, 1.0, 1.0, 0.999), (0, 0.999, 0.3, 0.7)):
        check_sample(arena, x, [0.9, 0.7, 1.1], k, p, m, np.full(3, u, np.float32))


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_scored_attention_of_as_many_keys_as_are_accepted(arena, dtype):
    """A context of 2^23 keys of which a few pages are in the pool, the first and the last among them."""
    rng = np.random.default_rng(22)
    typed(dtype)
    H, G, D, block, n = 4, 2, 64, 256, 1 << 23
    w = np.dtype(kind(dtype)).itemsize
    blocks = 9
    table = np.full((1, n // block), -1, np.int32)
    at = np.array([0, 1, 777, 16383, 16384, 20000, n // block - 2, n // block - 1])
    table[0, at] = rng.permutation(blocks)[:len(at)]
    q, qb = encode(rng.standard_normal((1, H * D)), dtype)
    k, kb = encode(rng.standard_normal((blocks, block, G, D)), dtype)
    v, vb = encode(rng.standard_normal((blocks, block, G, D)), dtype)
    scores = rng.random((blocks, G, block)).astype(np.float32)
    m = meta(arena, [n], table)
    out, ws = arena.space(H * D * w), arena.space(L.nvr_paged_attn_scored_workspace_bytes(1, H, G, D, n), 0xFF)
    ds = arena.dev(scores)
    nvr.check(L.nvr_paged_attn_decode_scored(arena.dev(qb).ptr, H * D, arena.dev(kb).ptr, arena.dev(vb).ptr, byref(m), H, G, D, block, blocks, 0.125, ds.ptr, None, 0.5, ds.ptr, out.ptr, ws.ptr, None))
    page = np.repeat(table[0, at], block)
    row, j = np.tile(np.arange(block), len(at)), np.repeat(at * block, block) + np.tile(np.arange(block), len(at))
    kk, vv = k[page, row], v[page, row]
    want, weights = attend(q.reshape(H, D), kk, vv, 0.125)
    size = max(float((np.abs(kk[:, h // 2]) @ np.abs(q.reshape(H, D)[h])).max()) for h in range(H)) * 0.125
    dw = 2 * (D + 4) * F32 * size + (len(j) / 4 + 64) * F32        # (as in scored_case: absent keys add exact zeros)
    two = {"float16": 2.0 ** -21, "float32": 0.0}[dtype]
    got = decode(out.to_numpy((H, D), kind(dtype)), dtype)
    tol = (2 * dw + two) * np.abs(vv).max()
    within(got, want, tol + HALF_STEP[dtype] * (np.abs(want) + tol) + SMALLEST[dtype], "out")
    new = ds.to_numpy(scores.shape, np.float32)
    for g in range(G):
        old = np.where(j < n - 1, 0.5 * scores[page, g, row].astype(np.float64), 0.0)
        within(new[page, g, row].astype(np.float64), old + weights[:, g], 2 * dw * weights[:, g] + 4 * F32 * (old + weights[:, g]) + 1e-37, "scores")
    free = [b for b in range(blocks) if b not in table[0, at]]
    assert np.array_equal(new[free].view(np.uint32), scores[free].view(np.uint32))


@pytest.mark.parametrize("budget,out_of_place", [(1000, False), ((1 << 24) + 3, False), ((1 << 24) + 3, True)])
def test_evict_of_as_many_keys_as_are_accepted(arena, budget, out_of_place):
    """A context of 2^25 keys, each row holding its key's number."""
    rng = np.random.default_rng(23)
    typed("float16")
    n, block, first, last = 1 << 25, 256, 5, 700
    blocks = n // block
    more = -(-budget // block) if out_of_place else 0
    table = rng.permutation(blocks).astype(np.int32)[None]
    to = (blocks + rng.permutation(more)).astype(np.int32)[None] if out_of_place else table
    rows = np.zeros(((blocks + more) * block, 4), np.uint32)       # 16 bytes a key
    where = (table[0].astype(np.int64)[:, None] * block + np.arange(block)).ravel()
    rows[where, 0] = np.arange(n)
    rows[where, 3] = np.arange(n)[::-1]
    scores = np.zeros((blocks + more) * block, np.float32)
    s = rng.integers(0, 1 << 20, n).astype(np.float32)
    scores[where] = s
    dk, ds = arena.dev(rows), arena.dev(scores)
    dv = arena.dev(rows[:, ::-1])
    new, kept, m = arena.space(4), arena.space(budget * 4), meta(arena, [n], table)
    nvr.check(L.nvr_kv_evict(dk.ptr, dv.ptr, ds.ptr, byref(m), 1, 8, block, blocks + more, budget, first, last, arena.dev(to).ptr if out_of_place else None, more, new.ptr, kept.ptr, None, None))
    best = np.argsort(-s[first:n - last], kind="stable")[:budget - first - last] + first
    want = np.sort(np.concatenate([np.arange(first), best, np.arange(n - last, n)]))
    assert new.to_numpy((1,), np.int32)[0] == budget and np.array_equal(kept.to_numpy((budget,), np.int32), want)
    at = (to[0].astype(np.int64)[:, None] * block + np.arange(block)).ravel()[:budget]
    got = dk.to_numpy(rows.shape, np.uint32)
    assert np.array_equal(got[at, 0], want) and np.array_equal(got[at, 3], n - 1 - want)
    assert np.array_equal(dv.to_numpy(rows.shape, np.uint32)[at, 3], want) and np.array_equal(ds.to_numpy(scores.shape, np.float32)[at], s[want])


def test_as_many_sequences_as_are_accepted(arena):
    rng = np.random.default_rng(24)
    B = 65535
    lengths = np.zeros(B, int)
    some = rng.choice(B, 300, replace=False)
    lengths[some] = rng.integers(1, 60, 300)
    lengths[[0, B - 1]] = [33, 17]
    scored_case(arena, "float16", lengths.tolist(), 2, 1, 64, 16)
    lengths[some[:3]] = [700, 515, 130]
    scored_case(arena, "bfloat16", lengths.tolist(), 2, 1, 64, 16, max_context=701)
    for out_of_place in (False, True):
        evict_case(arena, "float16", lengths.tolist(), 1, 8, 16, 20, 2, 5, out_of_place)
    x = rng.standard_normal((B, 5)).astype(np.float32)
    u = rng.random(B).astype(np.float32)
    ids, lp = sample_rows(arena, x, None, None, np.full(B, 0.8), None, u)
    for r in rng.choice(B, 400, replace=False).tolist() + [0, B - 1]:
        assert ids[r] == sample(x[r], 1.0, 0, float(np.float32(0.8)), 0.0, float(u[r]))[0]


@pytest.mark.parametrize("V", [2, 20, 300, 2050, 20000, 151936, 400000])
def test_sample_goals_that_equal_a_sum(arena, V):
    """Equal logits away from a cell's middle, and halves, quarters and eighths of their number: a nucleus ends with the token that brings the sum to exactly top_p, a token is drawn only where the sum is more than
    the uniform number's."""
    rng = np.random.default_rng(V)
    some = rng.choice(V, min(V, 16), replace=False)
    few = np.full(V, -3.0)
    few[some] = 5.1                                                # up to 16 equal ones above others that T leaves next to nothing
    x = np.stack([np.full(V, 2.3), np.full(V, 1000.1), few, few - 22.8])
    for T in ((0.7, 1.3, 0.01, 0.003), (100.0, 0.05, 0.02, 0.01)):
        for k, p, m in ((0, 1.0, 0.0), (0, 0.5, 0.0), (0, 0.25, 0.0), (0, 0.75, 0.5), (min(V, 16), 0.5, 0.0), (8, 1.0, 0.0), (V // 2, 0.5, 1.0), (0, 1.0, 0.9)):
            for u in (0.5, 0.25, 0.875, 2.0 ** -24, 1 - 2.0 ** -24):
                check_sample(arena, x, T, k, p, m, u)


@pytest.mark.parametrize("V", [200, 2000, 20000, 151936])
def test_sample_goals_a_hair_from_a_sum(arena, V):
    """Two halves whose weights differ by 2.4e-13 of themselves, so that the middle of the sum lies 1.2e-13 behind the first half's end, or in front of it; by 4e-12 where filters have the weights in steps of
    2^-40 (of a weight of 1, 9e-13)."""
    a, b = np.float32(2.3), np.nextafter(np.float32(2.3), np.float32(3))
    assert 2e-7 < float(b) - float(a) < 3e-7
    x = np.stack([np.where(np.arange(V) < V // 2, a, b), np.where(np.arange(V) < V // 2, b, a)])
    for T, k, p, m in ((1e6, 0, 1.0, 0.0), (6e4, 0, 1 - 2.0 ** -24, 0.0), (6e4, 0, 1.0, 0.5), (6e4, V + 1, 1 - 2.0 ** -24, 0.9)):
        ids, _ = sample_rows(arena, x, np.full(2, T), np.full(2, k), np.full(2, p), np.full(2, m), np.full(2, 0.5))
        assert ids.tolist() == [V // 2, V // 2 - 1], (T, k, p, m)


@pytest.mark.parametrize("V", [8192, 114688])
def test_sample_chunks_of_hardly_any_weight(arena, V):
    """A first chunk whose tokens weigh about e^-42, where they may be left out, and a number of 0: the first of them, or the first behind them, never none."""
    edge = np.arange(41.0, 44.0, 0.02)
    x = np.zeros((len(edge), V), np.float32)
    x[:, :V // 2] = -edge[:, None]
    for k, p, m in ((0, 1.0, 0.0), (V - 1, 1.0, 0.0), (0, 1 - 2.0 ** -24, 0.0), (0, 1.0, 1e-30)):
        ids, _ = sample_rows(arena, x + np.float32(2.3), None, np.full(len(edge), k), np.full(len(edge), p), np.full(len(edge), m), np.zeros(len(edge)))
        assert np.isin(ids, [0, V // 2]).all(), (k, p, m, ids)
        if p == 1.0:
            assert (ids[edge < 41.9] == 0).all()                   # (above e^-42: none is left out)
