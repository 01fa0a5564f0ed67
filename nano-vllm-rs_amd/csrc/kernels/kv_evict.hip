// kv_evict.hip — a sequence's cache brought down to `budget` keys a kv head: its first and last keys, and the best of the others by their scores (ties: the earlier key), close up in their order.
//
// First launch, a workgroup a (sequence, kv head): the score that the last of the kept keys has, by a radix select over the scores (held in LDS up to kHeld of them), then the kept keys in
// order (each thread owns a run of keys; one scan tells where its kept ones go) and the scores at their new places.  Second launch: the rows of K and V (a few of them the first moves itself).
// Into other blocks, every row is on its own: a copy, bound by memory.  In place, row i comes from row kept[i] >= i, which is overwritten by a later row: a workgroup takes a (sequence, kv head)'s
// strip of 128 bytes of the rows, from the front in steps of kMoves requests: all of a step are read before any is written, and no later step reads what it writes.
// 32 sequences of 1000 .. 8100 keys of 8 heads of 128 to 2048, float16, other blocks: 111 us (15 and 94), 4.4 TB/s over both, 5.2 in the copy (a large copy: 5.1); one of 4099 keys: 15 us (11 and 4).
// In place, scores drawn anew before each call: 32 of 8000 keys 150 us (15 and 135; 536 MB read and written), of 2304 137, of 2049 80 (9 and 72; 340 MB: one key too many moves every row behind the one that goes);
// one of 4099 keys 28 (10 and 19: 128 workgroups, each with a chain of steps).
// The select's life is a chain of some twenty LDS round trips and barriers; ballots in place of a thread's run of keys, and a count of a digit's few keys in place of its last two passes, took as long.
#include <algorithm>
#include <type_traits>
#include "serving.h"
#include "elem.h"
#include "scan.h"
#include "../common.h"

namespace nvr { namespace kx {

namespace {
constexpr int kPick = 1024, kHeld = 32768, kRadix = 2048, kTable = 512, kHere = 4, kLongest = 1 << 25;       // kHere: rows that a thread moves 16 bytes of; kHeld: scores in LDS, at most (128 of 160 KB)
struct EvictParams {
    EvictArgs a;
    int32_t *kept;                                                        // [B][KVH][budget]
    int32_t row_bytes, strip;                                             // of a key's row of a head; bytes of it that a workgroup moves
    int32_t held;                                                         // scores that LDS has room for
    uint32_t per_block;                                                   // 2^32 / block_size, rounded down
};
// j / block_size and what is left, without a division: the product's upper half is at most one short
struct Slot { int block, row; };
__device__ __forceinline__ Slot slot_of(const EvictParams &p, int j) {
    Slot s;
    s.block = (int)__umulhi((unsigned)j, p.per_block); s.row = j - s.block * p.a.block_size;
    if (s.row >= p.a.block_size) { ++s.block; s.row -= p.a.block_size; }
    return s;
}
__device__ __forceinline__ int length_of(const EvictArgs &a, int b) {
    const long long most = (long long)a.max_blocks * a.block_size;
    return (int)max(0ll, min((long long)min(a.ctx_lens[b], a.max_ctx), most));
}
__device__ __forceinline__ int row_in(const EvictParams &p, const int32_t *table, int j) {
    const Slot s = slot_of(p, j);
    return table[s.block] * p.a.block_size + s.row;
}
// larger score, larger number; not a number: below all
__device__ __forceinline__ unsigned int rank_of(float f) {
    if (!(f == f)) return 0u;
    const unsigned int u = __float_as_uint(f + 0.f);                      // (-0 is 0)
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
}  // namespace

// MOVE: the rows are few, and are moved here: all are read before any is written.  us so and with a second launch, scores drawn anew before each call, 8 heads of 256 bytes a row, other blocks (in place): one
// sequence of 1000 keys to 64 5.7 8.0 (5.6 8.5), to 256 7.2 8.1 (7.1 9.8); 16 to 128 8.4 10.3 (7.9 11.6), to 256 11.2 12.6 (10.6 13.7); 32 of 2000 to 500 rows of 128 bytes 17.9 19.5 (17.4 21.1)
template <bool MOVE>
__global__ __launch_bounds__(kPick) void kv_evict_select_kernel(EvictParams p) {
    extern __shared__ __attribute__((aligned(16))) float held[];          // scores of keys 0 .. p.held - 1
    __shared__ unsigned int hist[2 * kRadix + kRadix / 2];                // 11, 11 and 10 bits
    __shared__ int32_t from_table[kTable], to_table[kTable];              // (the first kTable blocks of each)
    __shared__ unsigned int waves[16], above[3];
    __shared__ unsigned long long waves2[16];
    __shared__ int found[3];
    const EvictArgs &a = p.a;
    const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int len = length_of(a, b), n = min(len, a.budget);
    const int32_t *table = a.block_tables + (int64_t)b * a.max_blocks, *to = a.to_tables ? a.to_tables + (int64_t)b * a.to_max_blocks : table;
    int32_t *kept = p.kept + ((int64_t)b * a.KVH + g) * a.budget;
    // a sequence whose tables name a block outside the pool, or too few, stays as it is
    int bad = a.to_tables && (long long)a.to_max_blocks * a.block_size < n;
    auto look = [&](const int32_t *t, int32_t *lds, int keys) {
        for (int i = tid, n = keys > 0 ? slot_of(p, keys - 1).block + 1 : 0; i < n; i += kPick) {
            const int block = t[i];
            bad |= block < 0 || block >= a.num_blocks;
            if (i < kTable) lds[i] = block;
        }
    };
    look(table, from_table, len);
    if (!bad) look(to, to_table, n);
    for (int i = tid; i < 2 * kRadix + kRadix / 2; i += kPick) hist[i] = 0;
    if (__syncthreads_or(bad)) {
        if (g == 0 && tid == 0) a.new_lens[b] = -1;
        for (unsigned int i = tid; i < (unsigned int)a.budget; i += kPick) kept[i] = -1;
        return;
    }
    if (g == 0 && tid == 0) a.new_lens[b] = n;
    for (unsigned int i = n + tid; i < (unsigned int)a.budget; i += kPick) kept[i] = -1;      // (a budget may be any)
    const bool all = len <= a.budget;
    if (all && !a.to_tables) {                                            // (nothing moves)
        for (int i = tid; i < n; i += kPick) kept[i] = i;
        return;
    }
    auto place = [&](const int32_t *t, const int32_t *lds, int j) {
        const Slot s = slot_of(p, j);
        return ((int64_t)(s.block < kTable ? lds[s.block] : t[s.block]) * a.KVH + g) * a.block_size + s.row;
    };
    auto from_at = [&](int j) { return place(table, from_table, j); };
    auto to_at = [&](int j) { return place(to, to_table, j); };
    // ---- the scores into LDS, 4 neighbours a thread where blocks are multiples of 4
    const int here = min(len, p.held);
    if (a.block_size % 4 == 0 && ((uintptr_t)a.scores & 15) == 0) {
        for (int i0 = tid * 4; i0 < here; i0 += kPick * 8) {
            float4_t v[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) { const int i = i0 + u * kPick * 4; if (i < here) v[u] = *reinterpret_cast<const float4_t *>(a.scores + from_at(i)); }
#pragma unroll
            for (int u = 0; u < 2; ++u) { const int i = i0 + u * kPick * 4; if (i < here) *reinterpret_cast<float4_t *>(held + i) = v[u]; }
        }
    } else
        for (int i = tid; i < here; i += kPick) held[i] = a.scores[from_at(i)];
    __syncthreads();
    const bool together = len <= p.held;
    // everything: LDS has all scores, and no other place is looked at (a loop of half the instructions: 8 x 48 .. 21715 keys 32.3 -> 25.8 us)
    auto choose = [&](auto everything) {
        constexpr bool ALL = decltype(everything)::value;
        auto score = [&](int i) { return ALL || i < p.held ? held[i] : a.scores[from_at(i)]; };
        // ---- the rank of the last of the best: the `need` best of keys first .. end - 1, of equal ones the earliest `want`
        const int first = a.first, end = len - a.last;
        const unsigned int need = all ? 0 : a.budget - a.first - a.last;      // (fewer than compete)
        unsigned int prefix = 0xffffffffu, want = 0;
        if (need) {
            unsigned int mask = 0;
            prefix = 0; want = need;
            for (int pass = 0; pass < 3; ++pass) {
                const int at = pass == 0 ? 21 : pass == 1 ? 10 : 0, wide = pass == 2 ? 1024 : 2048;
#pragma unroll 4
                for (int i = first + tid; i < end; i += kPick) { const unsigned int k = rank_of(score(i)); if ((k & mask) == prefix) atomicAdd(&hist[pass * kRadix + wide - 1 - ((k >> at) & (wide - 1))], 1u); }
                __syncthreads();
                const unsigned int c0 = 2 * tid < wide ? hist[pass * kRadix + 2 * tid] : 0, c1 = 2 * tid < wide ? hist[pass * kRadix + 2 * tid + 1] : 0;
                const unsigned int v = scan<unsigned int>(c0 + c1, waves) - c0 - c1;      // in front of this thread's two digits
                if (v < want && v + c0 + c1 >= want) {                        // (one thread)
                    const bool odd = v + c0 < want;
                    found[pass] = 2 * tid + odd; above[pass] = odd ? v + c0 : v;
                }
                __syncthreads();
                prefix |= (unsigned int)(wide - 1 - found[pass]) << at; mask |= (unsigned int)(wide - 1) << at;
                want -= above[pass];
            }
        }
        // ---- a thread's run of keys: how many of them are kept, and where they begin
        const int per = (len + kPick - 1) / kPick, i0 = min(len, tid * per), i1 = min(len, i0 + per);
        unsigned int more = 0, same = 0;
        for (int i = i0; i < i1; ++i) {
            const bool always = all || i < first || i >= end;
            const unsigned int k = always ? 0 : rank_of(score(i));
            more += always || (need && k > prefix); same += !always && need && k == prefix;
        }
        const unsigned long long own = ((unsigned long long)more << 32) | same, v = scan<unsigned long long>(own, waves2) - own;
        // the scores at their new places: at once where LDS has them all
        unsigned int seen = (unsigned int)v, at = (unsigned int)(v >> 32) + min(seen, want);
        for (int i = i0; i < i1; ++i) {
            const bool always = all || i < first || i >= end;
            const float f = score(i);
            const unsigned int k = always ? 0 : rank_of(f);
            const bool tie = !always && need && k == prefix;
            if (always || (need && k > prefix) || (tie && seen < want)) {
                kept[at] = i;
                if (MOVE) hist[at] = (unsigned int)i;                 // (the counts have been looked at)
                if (ALL) a.scores[to_at((int)at)] = f;
                ++at;
            }
            seen += tie;
        }
    };
    if constexpr (MOVE) {                                                 // (no more keys than LDS holds)
        choose(std::true_type());
        __syncthreads();
        const int lanes = p.row_bytes / 16, rows = kPick / lanes, lead = tid / lanes;
        const int64_t row = (int64_t)a.KVH * p.row_bytes, off = (int64_t)g * p.row_bytes + tid % lanes * 16;
        auto row_at = [&](const int32_t *t, const int32_t *lds, int j) {
            const Slot q = slot_of(p, j);
            return ((int64_t)(q.block < kTable ? lds[q.block] : t[q.block]) * a.block_size + q.row) * row + off;
        };
        float4_t k[kHere], v[kHere];
#pragma unroll
        for (int u = 0; u < kHere; ++u) {
            const int i = u * rows + lead;
            const int64_t at = lead < rows && i < n ? row_at(table, from_table, (int)hist[i]) : -1;
            k[u] = v[u] = (float4_t){0.f, 0.f, 0.f, 0.f};
            if (at >= 0) { k[u] = *reinterpret_cast<const float4_t *>((const char *)a.k + at); v[u] = *reinterpret_cast<const float4_t *>((const char *)a.v + at); }
        }
#pragma unroll
        for (int u = 0; u < kHere; ++u) asm volatile("" : "+v"(k[u]), "+v"(v[u]));      // (here: all of them have arrived)
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kHere; ++u) {
            const int i = u * rows + lead;
            if (lead >= rows || i >= n) continue;
            const int64_t at = row_at(to, to_table, i);
            *reinterpret_cast<float4_t *>((char *)a.k + at) = k[u];
            *reinterpret_cast<float4_t *>((char *)a.v + at) = v[u];
        }
        return;
    }
    if (together) return choose(std::true_type());
    choose(std::false_type());
    __threadfence_block();
    __syncthreads();
    for (int j0 = 0; j0 < n; j0 += kPick) {                               // from the front: of a step all are read before any is written
        const int i = j0 + tid;
        float f = 0.f;
        if (i < n) f = a.scores[from_at(kept[i])];
        asm volatile("" : "+v"(f));
        __syncthreads();
        if (i < n) a.scores[to_at(i)] = f;
    }
}

// 16 bytes a lane, `strip` bytes of a row; the step in front of the next one's writes is on its way
constexpr int kMoves = 4;                                                 // requests on their way (8 heads of 128, float16, scores drawn anew: 32 x 8000 keys to 2048 2 147 us, 4 150, 8 178; 32 x 2049 81 80 98)
__global__ __launch_bounds__(kPick) void kv_evict_close_kernel(EvictParams p) {
    const EvictArgs &a = p.a;
    const int g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int len = length_of(a, b);
    if (len <= a.budget || a.new_lens[b] < 0) return;
    const int n = a.budget, strips = p.row_bytes / p.strip, which = blockIdx.x;
    char *pool = (char *)(which < strips ? a.k : a.v);
    const int32_t *table = a.block_tables + (int64_t)b * a.max_blocks, *kept = p.kept + ((int64_t)b * a.KVH + g) * a.budget;
    const int lanes = p.strip / 16, piece = tid % lanes, lead = tid / lanes, rows = kPick / lanes;    // rows of a request
    const int64_t row = (int64_t)a.KVH * p.row_bytes, off = (int64_t)g * p.row_bytes + (which % strips) * p.strip + piece * 16;
    float4_t v[kMoves];
    auto request = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kMoves; ++u) {
            const int i = i0 + u * rows + lead;
            if (lead < rows && i < n) { const int j = kept[i]; if (j != i) v[u] = *reinterpret_cast<const float4_t *>(pool + row_in(p, table, j) * row + off); }
        }
    };
    request(0);
    for (int i0 = 0; i0 < n; i0 += kMoves * rows) {
        float4_t w[kMoves];
#pragma unroll
        for (int u = 0; u < kMoves; ++u) { w[u] = v[u]; asm volatile("" : "+v"(w[u])); }      // (here: what this step reads has arrived)
        __syncthreads();
        if (i0 + kMoves * rows < n) request(i0 + kMoves * rows);
#pragma unroll
        for (int u = 0; u < kMoves; ++u) {
            const int i = i0 + u * rows + lead;
            if (lead < rows && i < n && kept[i] != i) *reinterpret_cast<float4_t *>(pool + row_in(p, table, i) * row + off) = w[u];
        }
    }
}

// Into other blocks: a lane 16 bytes of K and of V (of two rows 124 us where this takes 123, of four 126, of eight 131)
__global__ __launch_bounds__(256) void kv_evict_copy_kernel(EvictParams p) {
    const EvictArgs &a = p.a;
    const int g = blockIdx.y, b = blockIdx.z;
    const int n = a.new_lens[b];
    const int lanes = p.row_bytes / 16, rows = 256 / lanes, lead = threadIdx.x / lanes, piece = threadIdx.x % lanes, i = blockIdx.x * rows + lead;
    if (i >= n || lead >= rows) return;
    const int32_t *table = a.block_tables + (int64_t)b * a.max_blocks, *to = a.to_tables + (int64_t)b * a.to_max_blocks, *kept = p.kept + ((int64_t)b * a.KVH + g) * a.budget;
    const int64_t row = (int64_t)a.KVH * p.row_bytes, off = (int64_t)g * p.row_bytes + piece * 16;
    const int64_t from = row_in(p, table, kept[i]) * row + off, at = row_in(p, to, i) * row + off;
    const float4_t k = *reinterpret_cast<const float4_t *>((const char *)a.k + from), v = *reinterpret_cast<const float4_t *>((const char *)a.v + from);
    *reinterpret_cast<float4_t *>((char *)a.k + at) = k;
    *reinterpret_cast<float4_t *>((char *)a.v + at) = v;
}

size_t kv_evict_workspace_bytes(int64_t B, int64_t KVH, int64_t budget, int64_t max_ctx) {
    (void)max_ctx;
    return B <= 0 || KVH <= 0 || budget <= 0 ? 0 : (size_t)(B * KVH * budget * 4);
}
int kv_evict(int dt, const EvictArgs &a, hipStream_t s) {
    const char *me = "nvr_kv_evict";
    if (a.B < 0 || a.KVH <= 0 || a.D <= 0 || a.block_size <= 0 || a.max_blocks < 0 || a.num_blocks < 0 || a.max_ctx < 0 || a.to_max_blocks < 0)
        return nvr::fail(NVR_ERR_INVALID_ARG, "%s: batch %d, %d kv heads of %d, blocks of %d", me, a.B, a.KVH, a.D, a.block_size);
    if (a.budget <= 0 || a.first < 0 || a.last < 0 || (int64_t)a.first + a.last > a.budget)
        return nvr::fail(NVR_ERR_INVALID_ARG, "%s: a budget of %d keys with the first %d and the last %d", me, a.budget, a.first, a.last);
    const int64_t bytes = (int64_t)a.D * (dt == DT_F32 ? 4 : 2);
    if (bytes % 16 || bytes > 1024) return nvr::fail(NVR_ERR_UNSUPPORTED, "%s: rows of %ld bytes a head (multiples of 16 up to 1024)", me, (long)bytes);
    if (a.num_blocks * a.block_size > 0x7fffffffll || a.B > 65535 || a.KVH > 65535) return nvr::fail(NVR_ERR_UNSUPPORTED, "%s: a pool of 2^31 rows and more, or more than 65535 sequences", me);
    // (sums of 32 bits over a sequence's keys, and the threads of the copy, stay below 2^32)
    const int64_t longest = std::min<int64_t>(a.max_ctx, (int64_t)a.max_blocks * a.block_size);
    if (longest > kLongest) return nvr::fail(NVR_ERR_UNSUPPORTED, "%s: contexts of %ld keys (the bound and the tables together allow up to %d)", me, (long)longest, kLongest);
    if (a.B == 0) return 0;
    if (!a.k || !a.v || !a.scores || !a.ctx_lens || !a.block_tables || !a.new_lens || (!a.kept && !a.workspace)) return nvr::fail(NVR_ERR_INVALID_ARG, "%s: null argument", me);
    if (a.new_lens == a.ctx_lens) return nvr::fail(NVR_ERR_INVALID_ARG, "%s: new_lens is the context_lens that other workgroups still read", me);
    if (a.to_tables == a.block_tables) return nvr::fail(NVR_ERR_INVALID_ARG, "%s: in place is asked for with to_tables null", me);
    if ((((uintptr_t)a.k | (uintptr_t)a.v) & 15) != 0) return nvr::fail(NVR_ERR_INVALID_ARG, "%s: the caches have to be aligned to 16 bytes", me);
    EvictParams p{};
    p.a = a;
    p.kept = a.kept ? a.kept : (int32_t *)a.workspace;
    p.row_bytes = (int32_t)bytes;
    p.per_block = (uint32_t)std::min<uint64_t>(0xffffffffull, (1ull << 32) / (uint64_t)a.block_size);
    p.strip = bytes % 128 == 0 ? 128 : (int32_t)bytes;
    const unsigned G = (unsigned)a.KVH, B = (unsigned)a.B;
    p.held = (int32_t)std::min<int64_t>((longest + 3) / 4 * 4, kHeld);
    const int64_t most = std::min<int64_t>(a.budget, longest);
    const bool move = longest <= kHeld && most <= kHere * (kPick / (p.row_bytes / 16));
    const auto kernel = move ? &kv_evict_select_kernel<true> : &kv_evict_select_kernel<false>;
    static std::atomic<uint64_t> allowed[2];
    if (const int rc = allow_lds(me, reinterpret_cast<const void *>(kernel), kHeld * 4, allowed[move])) return rc;
    kernel<<<dim3(G, B), kPick, (size_t)p.held * 4, s>>>(p);
    if (move) {
        NVR_KX_LAUNCHED("kv_evict");
        return 0;
    }
    if (a.to_tables) {
        const int rows = 256 / (p.row_bytes / 16);
        if (most > 0) kv_evict_copy_kernel<<<dim3((unsigned)((most + rows - 1) / rows), G, B), 256, 0, s>>>(p);
    } else if (longest > a.budget) kv_evict_close_kernel<<<dim3((unsigned)(2 * (p.row_bytes / p.strip)), G, B), kPick, 0, s>>>(p);
    NVR_KX_LAUNCHED("kv_evict");
    return 0;
}

}}  // namespace nvr::kx
