// Norms of the query and key heads and the rotation by position, in one pass.
//
//   x^ = x * rsqrt(mean(x^2) + eps) * w                       (w given; else x^ = x)
//   y_i = x^_i cos_i - x^_p sin_i,  y_p = x^_p cos_p + x^_i sin_p      for the pairs (i, p) of the first R channels:
//   (i, i + R/2), or (2i, 2i + 1) when interleaved; the channels behind R pass through.
//
// Bound by memory: each head row is read and written once, a token's row of the tables once for all its heads.  Eight
// lanes hold a row, 8 channels a chunk, as elsewhere in this library; everything is fp32 and rounded once, at the end.
#include "common.cuh"

namespace hira {

constexpr int RP_THREADS = 128;
constexpr int RP_GROUPS = RP_THREADS / GROUP;

struct RopeSide {           // the queries, or the keys
    const void* x;
    void* y;
    const void* w;
    int heads;
    long long xs[3], ys[3]; // elements between sequences, heads, tokens
};
struct RopeParams {
    RopeSide side[2];
    const void* cos;
    const void* sin;
    long long cs[2], ss[2]; // sequences, tokens
    int n_tokens, dim, rotary, interleaved;
    float eps;
};

template <typename T> __device__ __forceinline__ float load_one(const T* p) { return (float)*p; }

// the pair partner of channel i of the rotated ones, and whether i is the first of its pair
__device__ __forceinline__ int rope_partner(const RopeParams& P, int i, bool& first) {
    if (P.interleaved) {
        first = (i & 1) == 0;
        return i ^ 1;
    }
    first = i < P.rotary / 2;
    return first ? i + P.rotary / 2 : i - P.rotary / 2;
}

template <typename T, typename TT, int NCH>
__global__ void __launch_bounds__(RP_THREADS)
rope_kernel(const RopeParams P) {
    const int lane = threadIdx.x & (GROUP - 1), grp = threadIdx.x / GROUP;
    const int token = blockIdx.x, b = blockIdx.y;
    const int heads = P.side[0].heads + P.side[1].heads;
    const TT* cos = reinterpret_cast<const TT*>(P.cos) + b * P.cs[0] + token * P.cs[1];
    const TT* sin = reinterpret_cast<const TT*>(P.sin) + b * P.ss[0] + token * P.ss[1];
    for (int hh = grp; hh < heads; hh += RP_GROUPS) {
        const RopeSide& S = P.side[hh >= P.side[0].heads];
        const int h = hh >= P.side[0].heads ? hh - P.side[0].heads : hh;
        const T* x = reinterpret_cast<const T*>(S.x) + b * S.xs[0] + h * S.xs[1] + token * S.xs[2];
        T* y = reinterpret_cast<T*>(S.y) + b * S.ys[0] + h * S.ys[1] + token * S.ys[2];
        const T* w = reinterpret_cast<const T*>(S.w);
        float v[NCH][8], o[NCH][8];
        Acc2 acc{0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = lane + GROUP * i;
            if (c * 8 < P.dim) {
                to_float(load_chunk_coherent<T>(x, c), v[i]);
                chunk_fma(acc, v[i], v[i]);
            }
        }
        float r = 1.f;
        if (w) r = rsqrtf(group_sum(acc.e + acc.o) / (float)P.dim + P.eps);
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = lane + GROUP * i;
            if (c * 8 >= P.dim) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int ch = c * 8 + e;
                const float a = w ? v[i][e] * r * load_one(w + ch) : v[i][e];
                o[i][e] = a;
                if (ch < P.rotary) {
                    bool first;
                    const int p = rope_partner(P, ch, first);
                    const float xp = w ? load_one(x + p) * r * load_one(w + p) : load_one(x + p);
                    o[i][e] = __fmaf_rn(first ? -xp : xp, load_one(sin + ch), a * load_one(cos + ch));
                }
            }
        }
        __syncwarp(group_mask());      // y may be x: every lane has read its partners
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = lane + GROUP * i;
            if (c * 8 < P.dim) store_chunk(y, c, o[i]);
        }
    }
}

template <typename T, typename TT>
static int launch_rope(const RopeParams& P, int batch, cudaStream_t s) {
    const dim3 grid((unsigned)P.n_tokens, (unsigned)batch);
    const int nch = chunks_per_lane(P.dim);
    if (nch == 1) rope_kernel<T, TT, 1><<<grid, RP_THREADS, 0, s>>>(P);
    else if (nch == 2) rope_kernel<T, TT, 2><<<grid, RP_THREADS, 0, s>>>(P);
    else rope_kernel<T, TT, 4><<<grid, RP_THREADS, 0, s>>>(P);
    HIRA_CHECK_LAUNCH("hira_qk_norm_rope launch");
    return HIRA_OK;
}

}  // namespace hira

using namespace hira;

extern "C" int hira_qk_norm_rope(const hira_rope_t* a, void* stream) {
    HIRA_CHECK_ARG(a != nullptr, HIRA_ERR_ARG, "hira_qk_norm_rope: arguments are NULL");
    HIRA_CHECK_ARG((a->dtype == HIRA_F32 || a->dtype == HIRA_BF16) && (a->table_dtype == HIRA_F32 || a->table_dtype == HIRA_BF16),
                   HIRA_ERR_DTYPE, "hira_qk_norm_rope: dtype %d or table_dtype %d is neither HIRA_F32 nor HIRA_BF16", a->dtype,
                   a->table_dtype);
    HIRA_CHECK_ARG(a->batch >= 0 && a->n_tokens >= 0 && a->q_heads >= 0 && a->k_heads >= 0 && a->batch <= 65535, HIRA_ERR_SHAPE,
                   "hira_qk_norm_rope: batch=%d (at most 65535) n_tokens=%d q_heads=%d k_heads=%d", a->batch, a->n_tokens, a->q_heads,
                   a->k_heads);
    HIRA_CHECK_ARG(a->dim >= 8 && a->dim <= 256 && a->dim % 8 == 0, HIRA_ERR_SHAPE,
                   "hira_qk_norm_rope: dim=%d must be a multiple of 8 in 8..256", a->dim);
    HIRA_CHECK_ARG(a->rotary >= 0 && a->rotary <= a->dim && a->rotary % 2 == 0, HIRA_ERR_SHAPE,
                   "hira_qk_norm_rope: rotary=%d must be even and in 0..dim (%d)", a->rotary, a->dim);
    if (a->batch == 0 || a->n_tokens == 0 || a->q_heads + a->k_heads == 0) return HIRA_OK;
    HIRA_CHECK_ARG((a->q_heads == 0 || (a->q && a->q_out)) && (a->k_heads == 0 || (a->k && a->k_out)) &&
                   (a->rotary == 0 || (a->cos && a->sin)), HIRA_ERR_ARG, "hira_qk_norm_rope: NULL argument");
    const int es = (int)elem_size(a->dtype);
    uintptr_t mis = 0;
    const int64_t* st[4] = {a->q_stride, a->q_out_stride, a->k_stride, a->k_out_stride};
    const void* ptr[4] = {a->q, a->q_out, a->k, a->k_out};
    for (int i = 0; i < 4; ++i)
        if (i < 2 ? a->q_heads : a->k_heads) mis |= (uintptr_t)ptr[i] | (uintptr_t)((st[i][0] | st[i][1] | st[i][2]) * es);
    HIRA_CHECK_ARG((mis & 15) == 0, HIRA_ERR_ARG, "hira_qk_norm_rope: every row must start on a 16-byte boundary");
    RopeParams P = {};
    P.side[0] = RopeSide{a->q, a->q_out, a->q_weight, a->q_heads, {st[0][0], st[0][1], st[0][2]}, {st[1][0], st[1][1], st[1][2]}};
    P.side[1] = RopeSide{a->k, a->k_out, a->k_weight, a->k_heads, {st[2][0], st[2][1], st[2][2]}, {st[3][0], st[3][1], st[3][2]}};
    P.cos = a->cos; P.sin = a->sin;
    P.cs[0] = a->cos_stride[0]; P.cs[1] = a->cos_stride[1];
    P.ss[0] = a->sin_stride[0]; P.ss[1] = a->sin_stride[1];
    P.n_tokens = a->n_tokens; P.dim = a->dim; P.rotary = a->rotary; P.interleaved = a->interleaved; P.eps = a->eps;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == HIRA_BF16)
        return a->table_dtype == HIRA_BF16 ? launch_rope<__nv_bfloat16, __nv_bfloat16>(P, a->batch, s) : launch_rope<__nv_bfloat16, float>(P, a->batch, s);
    return a->table_dtype == HIRA_BF16 ? launch_rope<float, __nv_bfloat16>(P, a->batch, s) : launch_rope<float, float>(P, a->batch, s);
}
