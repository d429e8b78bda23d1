// Norms of the query and key heads and the rotation by position, in one pass.
//
//   x^ = x * rsqrt(mean(x^2) + eps) * w                       (w given; else x^ = x)
//   y_i = x^_i cos_i - x^_p sin_i,  y_p = x^_p cos_p + x^_i sin_p      for the pairs (i, p) of the first R channels:
//   (i, i + R/2), or (2i, 2i + 1) when interleaved; the channels behind R pass through.
//
// Bound by memory: each head row is read and written once, a token's row of the tables once for all its heads.  Eight
// lanes hold a row, 8 channels a chunk, as elsewhere in this library; everything is fp32 and rounded once, at the end.
// A group of eight lanes takes up to four heads of one token: their rows are all loaded before the first is used, and
// the token's tables and the weights sit in registers for all four.
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
// how the partner of a rotated channel is come by
enum RopePairs {
    ROPE_LANE,          // R/2 = 64: the lane's other chunk holds the partners of each of its chunks
    ROPE_CHUNK,         // R/2 a multiple of 8: a whole other chunk of the row
    ROPE_INTERLEAVED,   // inside the chunk (R even: a chunk may be rotated in part)
    ROPE_SINGLE         // channel by channel (R/2 not a multiple of 8)
};
struct RopeParams {
    RopeSide side[2];
    const void* cos;
    const void* sin;
    long long cs[2], ss[2]; // sequences, tokens
    long long units;        // groups of heads of all tokens
    int n_tokens, dim, rotary, pairs, per_token;
    int wide_tables;        // 16-byte loads of the tables
    float eps;
};

// channels 8c .. 8c + 7 of a table row; those from R on as cos = 1, sin = 0: they pass through
template <typename TT>
__device__ __forceinline__ void load_table(const TT* row, int c, int rotary, int wide, float other, float (&f)[8]) {
    if (wide && c * 8 + 8 <= rotary) {
        to_float(load_chunk<TT>(row, c), f);
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = c * 8 + e < rotary ? (float)row[c * 8 + e] : other;
}

template <typename T, typename TT, int NCH, int HPG>
__global__ void __launch_bounds__(RP_THREADS)
rope_kernel(const RopeParams P) {
    const int lane = threadIdx.x & (GROUP - 1);
    const long long unit = (long long)blockIdx.x * RP_GROUPS + threadIdx.x / GROUP;
    if (unit >= P.units) return;
    const long long bt = unit / P.per_token;
    const int h0 = (int)(unit - bt * P.per_token) * HPG, b = (int)(bt / P.n_tokens), token = (int)(bt - (long long)b * P.n_tokens);
    const int nq = P.side[0].heads, heads = nq + P.side[1].heads;
    RawChunk<T> raw[HPG][NCH];
    const T* x[HPG];
#pragma unroll
    for (int j = 0; j < HPG; ++j) {
        const int hh = min(h0 + j, heads - 1);
        const RopeSide& S = P.side[hh >= nq];
        x[j] = reinterpret_cast<const T*>(S.x) + b * S.xs[0] + (hh >= nq ? hh - nq : hh) * S.xs[1] + token * S.xs[2];
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = lane + GROUP * i;
            if (c * 8 < P.dim) raw[j][i] = load_chunk_coherent<T>(x[j], c);
            else raw[j][i] = zero_chunk<T>();
        }
    }
    float cs[NCH][8], sn[NCH][8];
    const TT* cos = reinterpret_cast<const TT*>(P.cos) + b * P.cs[0] + token * P.cs[1];
    const TT* sin = reinterpret_cast<const TT*>(P.sin) + b * P.ss[0] + token * P.ss[1];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = lane + GROUP * i;
        load_table<TT>(cos, c, P.rotary, P.wide_tables, 1.f, cs[i]);
        load_table<TT>(sin, c, P.rotary, P.wide_tables, 0.f, sn[i]);
    }
    const int half = P.rotary / 2;
#pragma unroll
    for (int j = 0; j < HPG; ++j) {
        const int hh = h0 + j;
        if (hh >= heads) break;          // the same for the group
        const RopeSide& S = P.side[hh >= nq];
        const T* w = reinterpret_cast<const T*>(S.w);
        float v[NCH][8], r = 1.f;
        Acc2 acc{0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            to_float(raw[j][i], v[i]);
            chunk_fma(acc, v[i], v[i]);
        }
        // the norm of chunk c's channels (v itself, or partners read again) with their weights
        auto scale = [&](float (&y)[8], int c) {
            float ww[8];
            to_float(load_chunk<T>(w, c), ww);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = y[e] * r * ww[e];
        };
        if (w) {
            r = rsqrtf(group_sum(acc.e + acc.o) / (float)P.dim + P.eps);
#pragma unroll
            for (int i = 0; i < NCH; ++i)
                if ((lane + GROUP * i) * 8 < P.dim) scale(v[i], lane + GROUP * i);
        }
        float o[NCH][8];
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = lane + GROUP * i;
            float p[8];                  // partners, with the sign they enter with
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = 0.f;
            if (c * 8 < P.rotary) {
                if (P.pairs == ROPE_INTERLEAVED) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        if (c * 8 + e < P.rotary) {
                            p[e] = -v[i][e + 1];
                            p[e + 1] = v[i][e];
                        }
                } else if (NCH == 2 && P.pairs == ROPE_LANE) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = i == 0 ? -v[NCH - 1][e] : v[0][e];
                } else if (P.pairs == ROPE_SINGLE) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int ch = c * 8 + e;
                        if (ch < P.rotary) {
                            const int q = ch < half ? ch + half : ch - half;
                            const float y = w ? (float)x[j][q] * r * (float)w[q] : (float)x[j][q];
                            p[e] = ch < half ? -y : y;
                        }
                    }
                } else {
                    const bool first = c * 8 < half;
                    const int q = first ? c + half / 8 : c - half / 8;
                    to_float(load_chunk_coherent<T>(x[j], q), p);      // this row again, from L1
                    if (w) scale(p, q);
                    if (first)
#pragma unroll
                        for (int e = 0; e < 8; ++e) p[e] = -p[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) o[i][e] = __fmaf_rn(p[e], sn[i][e], v[i][e] * cs[i][e]);
        }
        __syncwarp(group_mask());        // the output may be the input: every lane has read its partners
        T* y = reinterpret_cast<T*>(S.y) + b * S.ys[0] + (hh >= nq ? hh - nq : hh) * S.ys[1] + token * S.ys[2];
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = lane + GROUP * i;
            if (c * 8 < P.dim) store_chunk(y, c, o[i]);
        }
    }
}

template <typename T, typename TT, int NCH>
static int launch_rope_n(RopeParams& P, int batch, cudaStream_t s) {
    const int heads = P.side[0].heads + P.side[1].heads;
    const long long tokens = (long long)batch * P.n_tokens;
    // One head a group while that does not fill the GPU with threads several times over; else four.
    const bool four = tokens * heads > 8ll * SM_COUNT * RP_GROUPS;
    P.per_token = four ? (heads + 3) / 4 : heads;
    P.units = tokens * P.per_token;
    const long long blocks = (P.units + RP_GROUPS - 1) / RP_GROUPS;
    HIRA_CHECK_ARG(blocks < (1ll << 31), HIRA_ERR_SHAPE, "hira_qk_norm_rope: %lld head rows exceed the grid limit", tokens * heads);
    if (four) rope_kernel<T, TT, NCH, 4><<<(unsigned)blocks, RP_THREADS, 0, s>>>(P);
    else rope_kernel<T, TT, NCH, 1><<<(unsigned)blocks, RP_THREADS, 0, s>>>(P);
    HIRA_CHECK_LAUNCH("hira_qk_norm_rope launch");
    return HIRA_OK;
}
template <typename T, typename TT>
static int launch_rope(RopeParams& P, int batch, cudaStream_t s) {
    const int nch = chunks_per_lane(P.dim);
    return nch == 1 ? launch_rope_n<T, TT, 1>(P, batch, s) : nch == 2 ? launch_rope_n<T, TT, 2>(P, batch, s) : launch_rope_n<T, TT, 4>(P, batch, s);
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
    mis |= (uintptr_t)a->q_weight | (uintptr_t)a->k_weight;
    HIRA_CHECK_ARG((mis & 15) == 0, HIRA_ERR_ARG, "hira_qk_norm_rope: the weights and every row must start on a 16-byte boundary");
    RopeParams P = {};
    P.side[0] = RopeSide{a->q, a->q_out, a->q_weight, a->q_heads, {st[0][0], st[0][1], st[0][2]}, {st[1][0], st[1][1], st[1][2]}};
    P.side[1] = RopeSide{a->k, a->k_out, a->k_weight, a->k_heads, {st[2][0], st[2][1], st[2][2]}, {st[3][0], st[3][1], st[3][2]}};
    P.cos = a->cos; P.sin = a->sin;
    P.cs[0] = a->cos_stride[0]; P.cs[1] = a->cos_stride[1];
    P.ss[0] = a->sin_stride[0]; P.ss[1] = a->sin_stride[1];
    P.n_tokens = a->n_tokens; P.dim = a->dim; P.rotary = a->rotary; P.eps = a->eps;
    // a token's tables may start anywhere, its weights too (they are loaded in 16-byte pieces)
    const int ts = (int)elem_size(a->table_dtype);
    P.wide_tables = (((uintptr_t)a->cos | (uintptr_t)a->sin | (uintptr_t)((P.cs[0] | P.cs[1] | P.ss[0] | P.ss[1]) * ts)) & 15) == 0;
    P.pairs = a->interleaved ? ROPE_INTERLEAVED : a->rotary % 16 ? ROPE_SINGLE : a->rotary == 128 && a->dim <= 128 ? ROPE_LANE : ROPE_CHUNK;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == HIRA_BF16)
        return a->table_dtype == HIRA_BF16 ? launch_rope<__nv_bfloat16, __nv_bfloat16>(P, a->batch, s) : launch_rope<__nv_bfloat16, float>(P, a->batch, s);
    return a->table_dtype == HIRA_BF16 ? launch_rope<float, __nv_bfloat16>(P, a->batch, s) : launch_rope<float, float>(P, a->batch, s);
}
