// Decode attention of a batch whose sequences share their prompts: what its kernels have in common.
#pragma once
#include "common.cuh"

namespace hira {

// Row r of a (prompt, kv head) is query token t of query head g of branch j: r = (j * group + g) * n_q + t.  Partials
// are kept per output row ((b * n_kv + h) * group + g) * n_q + t with b = prompt * n_branches + j: part i of row R has
// its unnormalised output at part_o[(i * n_rows + R) * vdim] and its (maximum, denominator) at part_ml[i * n_rows + R].
// Logits and maxima are in units of log2: x = (q . k) * sm_scale * log2(e), p = 2^(x - m).
struct SharedAttn {
    const void* q;
    const void* pk;
    const void* pv;
    const void* tk;
    const void* tv;
    void* out;
    const int32_t* prefix_lens;   // [n_prompts] or null: prefix_len
    const int32_t* tail_lens;     // [n_prompts * n_branches] or null: tail_len
    float* part_o;
    float2* part_ml;
    int n_prompts, n_branches, n_kv, group, n_q, dim, vdim;
    int prefix_len, tail_len;
    int prefix_parts;             // partials of the prefix (at most, see `shares`), then the tail's
    int tail_parts;
    int fused;                    // the tail's kernel joins the parts itself
    int n_rows;                   // output rows
    float scale_log2;             // sm_scale * log2(e)
    long long qs[3], os[3];       // elements between branches, heads, tokens
    long long pks[3], pvs[3];     // prompts, heads, rows
    long long tks[3], tvs[3];     // branches, heads, rows
    // The tensor-core kernel deals the key tiles of all (prompt, kv head) items out in `shares` equal runs, so an item's
    // number of partials follows from its position (0: every item has prefix_parts of them).
    int shares, item_tiles;
    int32_t* status;              // or null: where a wait that ran out is reported
};

__device__ __forceinline__ int shared_prefix_len(const SharedAttn& P, int prompt) {
    if (!P.prefix_lens) return P.prefix_len;
    return min(max(P.prefix_lens[prompt], 0), P.prefix_len);
}
__device__ __forceinline__ int shared_tail_len(const SharedAttn& P, int branch) {
    if (!P.tail_lens) return P.tail_len;
    return min(max(P.tail_lens[branch], 0), P.tail_len);
}
// output row of row r of (prompt, kv head)
__device__ __forceinline__ int shared_row(const SharedAttn& P, int prompt, int h, int r) {
    const int per = P.group * P.n_q, j = r / per;
    return ((prompt * P.n_branches + j) * P.n_kv + h) * per + (r - j * per);
}
// offset of output row R in a (branch, head, token) tensor with strides s
__device__ __forceinline__ long long shared_row_offset(const SharedAttn& P, int R, const long long (&s)[3]) {
    const int heads = P.n_kv * P.group, t = R % P.n_q, bh = R / P.n_q;
    return (long long)(bh / heads) * s[0] + (long long)(bh % heads) * s[1] + (long long)t * s[2];
}
// the run of tiles that an item begins in (run s is tiles s * total / shares .. (s + 1) * total / shares), and its partials
__device__ __forceinline__ int shared_share_of(const SharedAttn& P, long long tile) {
    const long long total = (long long)P.n_prompts * P.n_kv * P.item_tiles;
    return (int)(((tile + 1) * P.shares - 1) / total);
}
__device__ __forceinline__ int shared_first_share(const SharedAttn& P, int item) { return shared_share_of(P, (long long)item * P.item_tiles); }
__device__ __forceinline__ int shared_item_parts(const SharedAttn& P, int item) {
    if (P.shares == 0) return P.prefix_parts;
    return shared_share_of(P, (long long)(item + 1) * P.item_tiles - 1) - shared_first_share(P, item) + 1;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr int SA_MAX_PARTS = 512;      // of an output row, prefix and tail together: what the join's kernel has room for

bool shared_tc_supported(const SharedAttn& P);
void shared_tc_plan(SharedAttn& P);
int shared_tc_launch(const SharedAttn& P, cudaStream_t s);
bool shared_mma_prefers(const SharedAttn& P);
int shared_mma_splits(const SharedAttn& P, bool tail);
bool shared_tail_joins(const SharedAttn& P);
// chained: behind the prefix's kernel, beside which it may run
int shared_mma_launch(const SharedAttn& P, bool tail, bool chained, cudaStream_t s);

}  // namespace hira
