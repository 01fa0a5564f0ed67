// serving.h — launchers of the operators around a serving step of many requests.  Each takes the storage type as an argument (elem.h) and
// enqueues on `s`; 0 or a status.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace nvr { namespace kx {

struct RopeArgs {
    const void *q, *k, *v; int64_t ldq, ldk, ldv;            // rows of a token, ld numbers apart, heads contiguous
    const int64_t *positions; const int32_t *slots;          // slots: row of the caches (outside them: not stored)
    int64_t T; int32_t H, KVH, D, rotary; bool pairs;
    const double *turns; float amplitude;                    // [rotary / 2]
    void *q_out, *k_out; int64_t ldqo, ldko;                 // may be q and k themselves; k_out null: the cache alone
    void *k_cache, *v_cache; int64_t num_slots;              // [num_slots][KVH][D], null: no cache
};
int rope_rotate_store(int dt, const RopeArgs &a, hipStream_t s);

struct LoraArgs {
    const void *x; int64_t ldx;
    const void *A, *B;                                       // [n][R][K], [n][N][R]
    const float *scales; const int32_t *ids; int64_t n;      // ids: an adapter a row (outside 0 .. n - 1: none)
    int64_t T, K, N, R;
    const void *base; int64_t ldb; void *y; int64_t ldy;     // base may be y itself
    void *workspace;
};
size_t lora_workspace_bytes(int64_t T, int64_t K, int64_t N, int64_t R);
int lora_add(int dt, const LoraArgs &a, hipStream_t s);

struct SampleArgs {
    const float *logits; int64_t ld, B, V;
    const float *temperature; const int64_t *top_k; const float *top_p, *min_p, *uniform;
    int64_t *ids; float *logprobs;
    void *workspace;
};
size_t sample_uniform_workspace_bytes(int64_t B, int64_t V);
int sample_uniform(const SampleArgs &a, hipStream_t s);

struct ScoredArgs {
    const void *q; int64_t ldq;
    const void *k, *v; const int32_t *ctx_lens, *block_tables; int32_t max_blocks, block_size; int64_t num_blocks;
    int32_t B, H, KVH, D, max_ctx; float scale;
    const float *scores; const int32_t *scored; float decay; float *new_scores;   // [num_blocks][KVH][block_size]
    void *out; void *workspace;
};
size_t paged_attn_scored_workspace_bytes(int64_t B, int64_t H, int64_t KVH, int64_t D, int64_t max_ctx);
int paged_attn_scored(int dt, const ScoredArgs &a, hipStream_t s);

struct EvictArgs {
    void *k, *v; float *scores;
    const int32_t *ctx_lens, *block_tables; int32_t max_blocks, block_size; int64_t num_blocks;
    int32_t B, KVH, D, max_ctx, budget, first, last;
    const int32_t *to_tables; int32_t to_max_blocks;         // null: in place
    int32_t *new_lens, *kept;                                // kept null: the workspace
    void *workspace;
};
size_t kv_evict_workspace_bytes(int64_t B, int64_t KVH, int64_t budget, int64_t max_ctx);
int kv_evict(int dt, const EvictArgs &a, hipStream_t s);

}}  // namespace nvr::kx
