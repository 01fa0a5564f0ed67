"""Storage types, device buffers and 64-bit definitions of the operators around a serving step (rotary positions in their forms, low-rank adapters, tokens from given
numbers, scored decode attention, eviction), for their tests."""
import ctypes as C
import math

import numpy as np

import nvr_import

nvr = nvr_import.load()
DTYPES = ("float16", "bfloat16", "float32")
HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}   # a rounding to nearest is off by at most that share of the value
SMALLEST = {"float16": 2.0 ** -25, "bfloat16": 0.0, "float32": 0.0}                 # ... and by that much among float16's subnormals
F32 = 2.0 ** -24
SENTINEL = 0x7B


def encode(a, dtype):
    """The values rounded to `dtype` (as float64) and their bits."""
    a = np.asarray(a, np.float32)
    if dtype == "float16":
        b = a.astype(np.float16)
        return b.astype(np.float64), b.view(np.uint16)
    if dtype == "bfloat16":
        u = a.view(np.uint32).astype(np.uint64)
        r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
        r = np.where(np.isnan(a), np.uint16(0x7FC0), r)
        return decode(r, dtype), r
    return a.astype(np.float64), a.view(np.uint32)


def decode(bits, dtype):
    if dtype == "float16":
        return bits.view(np.float16).astype(np.float64)
    if dtype == "bfloat16":
        return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return bits.view(np.float32).astype(np.float64)


def kind(dtype):
    return np.uint32 if dtype == "float32" else np.uint16


class Arena:
    """Device buffers that live until the test is over."""

    def __init__(self):
        self.kept = []

    def dev(self, a):
        b = nvr.DeviceBuffer.from_numpy(np.ascontiguousarray(a))
        self.kept.append(b)
        return b

    def space(self, nbytes, fill=SENTINEL):
        b = nvr.DeviceBuffer(max(int(nbytes), 16))
        nvr.check(nvr.lib().nvr_device_memset(b.ptr, fill, b.nbytes))
        self.kept.append(b)
        return b


def typed(dtype):
    nvr.check(nvr.lib().nvr_ops_set_dtype(dtype.encode()))


# ---- definitions in 64 bits
def rope_turns(kind_, rotary, theta=10000.0, factor=1.0, original=2048.0, low=1.0, high=32.0):
    j = np.arange(rotary // 2, dtype=np.float64)
    if kind_ == "ntk":
        theta = theta * factor ** (rotary / (rotary - 2))
    f = 1.0 / theta ** (2 * j / rotary)
    amplitude = 1.0
    if kind_ == "linear":
        f = f / factor
    if kind_ == "yarn":
        def pair(turns):
            return rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
        a, b = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rotary - 1)
        r = np.clip((j - a) / max(b - a, 1e-3), 0, 1)
        f = f / factor * r + f * (1 - r)
        amplitude = 0.1 * math.log(factor) + 1 if factor > 1 else 1.0
    if kind_ == "bands":
        turns = original * f / (2 * math.pi)
        f = np.where(turns >= high, f, np.where(turns <= low, f / factor, 0.0)) + np.where((turns < high) & (turns > low), 1, 0) * (
            (1 - (turns - low) / (high - low)) * f / factor + (turns - low) / (high - low) * f)
    return f / (2 * math.pi), amplitude


def rope(x, positions, turns, amplitude, pairs):
    """x [T, heads, D], the first 2 len(turns) columns turned."""
    n = 2 * len(turns)
    t = positions[:, None].astype(np.longdouble) * turns[None].astype(np.longdouble)      # (64 bits alone lose a far position's part of a turn)
    a = 2 * math.pi * (t - np.rint(t)).astype(np.float64)
    c, s = amplitude * np.cos(a)[:, None], amplitude * np.sin(a)[:, None]
    y = x.copy()
    one, two = (slice(0, n, 2), slice(1, n, 2)) if pairs else (slice(0, n // 2), slice(n // 2, n))
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., one] * s + x[..., two] * c
    return y


def sample(x, T, k, p, m, u):
    """(token, ln of its share) of one row, in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    if not (x > -np.inf).any():
        return -1, -np.inf
    if not T > 0:
        return int(np.argmax(x)), 0.0
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    order = order[:k] if k > 0 else order
    top = x[order[0]]
    d = np.where(x[order] == top, 0.0, x[order] - top) / T
    w = np.exp(d)
    if 0 <= p < 1:
        n = int((np.cumsum(w) < p * w.sum()).sum()) + 1
        order, w = order[:n], w[:n]
    if m > 0:
        keep = w >= min(m, 1.0)
        order, w = order[keep], w[keep]
    back = np.argsort(order)
    order, w = order[back], w[back]
    i = min(int((np.cumsum(w) <= u * w.sum()).sum()), len(w) - 1)
    return int(order[i]), math.log(w[i] / w.sum())


def attend(q, k, v, scale):
    """q [H, D], k and v [n, G, D]: outputs [H, D] and weights summed over the heads of a kv head [n, G]."""
    H, G = q.shape[0], k.shape[1]
    out, weights = np.zeros(q.shape), np.zeros(k.shape[:2])
    for h in range(H):
        g = h * G // H
        s = scale * (k[:, g] @ q[h])
        w = np.exp(s - s.max())
        w = w / w.sum()
        out[h] = w @ v[:, g]
        weights[:, g] += w
    return out, weights


def evict(scores, n, first, last):
    """Places of the kept keys of one kv head, in order."""
    L = len(scores)
    if L <= n:
        return np.arange(L)
    s = np.where(np.isnan(scores), -np.inf, scores)
    nan_below = np.isnan(scores)
    middle = np.arange(first, L - last)
    best = sorted(middle, key=lambda j: (nan_below[j], -s[j], j))[:n - first - last]
    return np.sort(np.concatenate([np.arange(first), np.array(best, np.int64), np.arange(L - last, L)])).astype(np.int64)


def tables(rng, lengths, block, extra=0):
    """Shuffled block tables (-1 behind a sequence's last block) and the pool's number of blocks (one more than named, at least)."""
    need = [-(-n // block) for n in lengths]
    total = sum(need) + 1 + extra
    order = rng.permutation(total)
    width = max(max(need), 1)
    t = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for b, k in enumerate(need):
        t[b, :k] = order[at:at + k]
        at += k
    return t, total


def meta(arena, lengths, table, max_context=None):
    m = nvr.AttnMetaC(is_prefill=0, context_lens=arena.dev(np.array(lengths, np.int32)).ptr, block_tables=arena.dev(table).ptr, max_blocks=table.shape[1], batch=len(lengths),
                      max_context_len=max(lengths) if max_context is None else max_context)
    return m


byref = C.byref
