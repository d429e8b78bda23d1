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
//
// 8,191 tokens x 40 heads of 128 bf16 with norm (168 MB): 35 us (4.8 TB/s) with 64 rotated channels, 41 with 128; a plain
// copy of as many bytes takes 32.  What is left is issue slots: two channels an instruction, partners by shuffles instead
// of the row read again and no division took it from 45 to 35; twice the heads a group, or its next four loaded while
// four are worked on, leave fewer warps and took 43 to 57.  One token of 40 heads: 6 us, the launch and one round trip.  Other
// forms of the same 8,191 tokens: 32 channels 35, interleaved 35 to 42 whatever is rotated; 48 channels 46 and 96 channels 55, whose
// partners are looked for among all of the group's chunks; 24 channels 77 (half of
// them no multiple of 8: one head a group, partners read again one by one).  fp32 57 to 68, 66 and 86, 82.
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
    ROPE_LANE,          // R/2 = 64 or 128: another chunk of the lane holds the partners of each of its chunks
    ROPE_XOR,           // R/2 = 8, 16 or 32: the first chunk of another of the group's lanes
    ROPE_CHUNK,         // any other multiple of 8: some chunk of another lane
    ROPE_INTERLEAVED,   // inside the chunk (R even: a chunk may be rotated in part)
    ROPE_SINGLE         // channel by channel (R/2 not a multiple of 8)
};
struct RopeParams {
    RopeSide side[2];
    const void* cos;
    const void* sin;
    long long cs[2], ss[2]; // sequences, tokens
    long long units;        // groups of heads of all tokens
    int n_tokens, dim, rotary;
    int q_units, per_token; // groups of a token's query heads, of all its heads
    int wide_tables;        // 16-byte loads of the tables
    float eps, inv_dim;
};

// chunks as pairs of channels: the arithmetic goes by two
template <typename T>
__device__ __forceinline__ void to_pairs(const RawChunk<T>& r, float2 (&f)[4]) {
    float x[8];
    to_float(r, x);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = make_float2(x[2 * e], x[2 * e + 1]);
}
// the chunk that lane `from` of the group holds
__device__ __forceinline__ RawChunk<__nv_bfloat16> chunk_of_lane(const RawChunk<__nv_bfloat16>& r, int from) {
    const unsigned m = group_mask();
    RawChunk<__nv_bfloat16> o;
    o.a = make_uint4(__shfl_sync(m, r.a.x, from, GROUP), __shfl_sync(m, r.a.y, from, GROUP), __shfl_sync(m, r.a.z, from, GROUP),
                     __shfl_sync(m, r.a.w, from, GROUP));
    return o;
}
__device__ __forceinline__ RawChunk<float> chunk_of_lane(const RawChunk<float>& r, int from) {
    const unsigned m = group_mask();
    RawChunk<float> o;
    o.a = make_float4(__shfl_sync(m, r.a.x, from, GROUP), __shfl_sync(m, r.a.y, from, GROUP), __shfl_sync(m, r.a.z, from, GROUP),
                      __shfl_sync(m, r.a.w, from, GROUP));
    o.b = make_float4(__shfl_sync(m, r.b.x, from, GROUP), __shfl_sync(m, r.b.y, from, GROUP), __shfl_sync(m, r.b.z, from, GROUP),
                      __shfl_sync(m, r.b.w, from, GROUP));
    return o;
}
// channels 8c .. 8c + 7 of a table row; those from R on as `other`
template <typename TT>
__device__ __forceinline__ void load_table(const TT* row, int c, int rotary, int wide, float other, float2 (&f)[4]) {
    if (c * 8 >= rotary) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = make_float2(other, other);
    } else if (wide && c * 8 + 8 <= rotary) {
        to_pairs(load_chunk<TT>(row, c), f);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)      // R is even
            f[e] = c * 8 + 2 * e < rotary ? make_float2((float)row[c * 8 + 2 * e], (float)row[c * 8 + 2 * e + 1]) : make_float2(other, other);
    }
}
// With the norm's factor r of a row, y_i = r (x_i a_i + x_p b_i), where a_i = w_i cos_i and b_i = +-w_p sin_i belong to the
// token and are formed once for the group's heads.
template <typename T, int NCH, int HPG, int PAIRS>
constexpr int rope_blocks() {      // an SM's: as many as leave a thread the registers for its rows and factors
    if (HPG == 1) return 1;
    return (NCH == 4 ? 3 : PAIRS == ROPE_CHUNK && NCH == 2 ? 4 : 5) - (sizeof(T) == 4);
}
template <typename T, typename TT, int NCH, int HPG, int PAIRS>
__global__ void __launch_bounds__(RP_THREADS, rope_blocks<T, NCH, HPG, PAIRS>())
rope_kernel(const RopeParams P) {
    const int lane = threadIdx.x & (GROUP - 1);
    const long long unit = (long long)blockIdx.x * RP_GROUPS + threadIdx.x / GROUP;
    if (unit >= P.units) return;
    const long long bt = unit / P.per_token;
    const int b = (int)(bt / P.n_tokens), token = (int)(bt - (long long)b * P.n_tokens);
    int h0 = (int)(unit - bt * P.per_token) * HPG;
    const bool keys = h0 >= P.q_units * HPG;          // a group's heads are all of one side
    if (keys) h0 -= P.q_units * HPG;
    const RopeSide& S = P.side[keys];
    const int n = min(S.heads - h0, HPG), half = P.rotary / 2;
    const T* x0 = reinterpret_cast<const T*>(S.x) + b * S.xs[0] + h0 * S.xs[1] + token * S.xs[2];
    const T* w = reinterpret_cast<const T*>(S.w);
    bool in[NCH];      // chunks of the row
#pragma unroll
    for (int i = 0; i < NCH; ++i) in[i] = (lane + GROUP * i) * 8 < P.dim;
    RawChunk<T> raw[HPG][NCH];
#pragma unroll
    for (int j = 0; j < HPG; ++j)
#pragma unroll
        for (int i = 0; i < NCH; ++i)
            raw[j][i] = in[i] && j < n ? load_chunk_coherent<T>(x0 + j * S.xs[1], lane + GROUP * i) : zero_chunk<T>();
    float2 ca[NCH][4], cb[NCH][4];
    const TT* cos = reinterpret_cast<const TT*>(P.cos) + b * P.cs[0] + token * P.cs[1];
    const TT* sin = reinterpret_cast<const TT*>(P.sin) + b * P.ss[0] + token * P.ss[1];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        const int c = lane + GROUP * i;
        load_table<TT>(cos, c, P.rotary, P.wide_tables, 1.f, ca[i]);
        if (PAIRS != ROPE_XOR || i == 0) load_table<TT>(sin, c, P.rotary, P.wide_tables, 0.f, cb[i]);
        float2 other[4];      // weights of the chunk's channels, then of their partners
#pragma unroll
        for (int e = 0; e < 4; ++e) other[e] = make_float2(1.f, 1.f);
        if (w && in[i]) {
            to_pairs(load_chunk<T>(w, c), other);
#pragma unroll
            for (int e = 0; e < 4; ++e) ca[i][e] = __fmul2_rn(ca[i][e], other[e]);
            if (c * 8 < P.rotary) {
                if (PAIRS == ROPE_CHUNK || PAIRS == ROPE_LANE || PAIRS == ROPE_XOR) {
                    to_pairs(load_chunk<T>(w, c * 8 < half ? c + half / 8 : c - half / 8), other);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int ch = c * 8 + 2 * e;
                        if (PAIRS == ROPE_INTERLEAVED) other[e] = make_float2(other[e].y, other[e].x);
                        else if (ch < P.rotary) other[e] = make_float2((float)w[ch < half ? ch + half : ch - half], (float)w[ch + 1 < half ? ch + 1 + half : ch + 1 - half]);
                    }
                }
            }
        }
        if ((PAIRS != ROPE_XOR || i == 0) && c * 8 < P.rotary) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // minus for the first of a pair
                if (PAIRS == ROPE_INTERLEAVED) other[e].x = -other[e].x;
                else if (PAIRS == ROPE_SINGLE)
                    other[e] = make_float2(c * 8 + 2 * e < half ? -other[e].x : other[e].x, c * 8 + 2 * e + 1 < half ? -other[e].y : other[e].y);
                else if (c * 8 < half)
                    other[e] = make_float2(-other[e].x, -other[e].y);
                cb[i][e] = __fmul2_rn(cb[i][e], other[e]);
            }
        }
    }
    T* y0 = reinterpret_cast<T*>(S.y) + b * S.ys[0] + h0 * S.ys[1] + token * S.ys[2];
#pragma unroll
    for (int j = 0; j < HPG; ++j) {
        if (j >= n) break;               // the same for the group
        const T* x = x0 + j * S.xs[1];
        float2 v[NCH][4], r = make_float2(1.f, 1.f);
#pragma unroll
        for (int i = 0; i < NCH; ++i) to_pairs(raw[j][i], v[i]);
        if (w) {
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc = __ffma2_rn(v[i][e], v[i][e], acc);
            r.x = r.y = rsqrtf(__fmaf_rn(group_sum(acc.x + acc.y), P.inv_dim, P.eps));
        }
        float2 o[NCH][4];
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = lane + GROUP * i;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] = __fmul2_rn(v[i][e], ca[i][e]);
            if (PAIRS == ROPE_XOR && i > 0) continue;
            float2 p[4];
            if (PAIRS == ROPE_XOR) to_pairs(chunk_of_lane(raw[j][i], lane ^ (half / 8)), p);
            if (PAIRS == ROPE_CHUNK) {
                const int pc = c * 8 < half ? c + half / 8 : c - half / 8;
                RawChunk<T> of = raw[j][i];
#pragma unroll
                for (int k = 0; k < NCH; ++k) {
                    const RawChunk<T> there = chunk_of_lane(raw[j][k], pc & (GROUP - 1));
                    if (pc / GROUP == k) of = there;
                }
                to_pairs(of, p);
            }
            if (c * 8 >= P.rotary) continue;
            if (PAIRS == ROPE_INTERLEAVED) {
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = make_float2(v[i][e].y, v[i][e].x);
            } else if (PAIRS == ROPE_LANE) {
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = NCH == 2 || half == 64 ? v[i ^ (NCH > 1)][e] : v[(i + NCH / 2) % NCH][e];
            } else if (PAIRS == ROPE_SINGLE) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int ch = c * 8 + 2 * e;
                    p[e] = make_float2(0.f, 0.f);
                    if (ch < P.rotary) p[e] = make_float2((float)x[ch < half ? ch + half : ch - half], (float)x[ch + 1 < half ? ch + 1 + half : ch + 1 - half]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)      // a chunk may be rotated in part: what passes through has no partner
                if ((PAIRS != ROPE_INTERLEAVED && PAIRS != ROPE_SINGLE) || c * 8 + 2 * e < P.rotary) o[i][e] = __ffma2_rn(p[e], cb[i][e], o[i][e]);
        }
        if (w)
#pragma unroll
            for (int i = 0; i < NCH; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] = __fmul2_rn(o[i][e], r);
        __syncwarp(group_mask());        // the output may be the input: every lane has read its partners
#pragma unroll
        for (int i = 0; i < NCH; ++i)
            if (in[i]) {
                const float y[8] = {o[i][0].x, o[i][0].y, o[i][1].x, o[i][1].y, o[i][2].x, o[i][2].y, o[i][3].x, o[i][3].y};
                store_chunk(y0 + j * S.ys[1], lane + GROUP * i, y);
            }
    }
}

template <typename T, typename TT, int NCH, int HPG, int PAIRS>
static int launch_rope_hp(RopeParams& P, int batch, cudaStream_t s) {
    P.q_units = (P.side[0].heads + HPG - 1) / HPG;
    P.per_token = P.q_units + (P.side[1].heads + HPG - 1) / HPG;
    P.units = (long long)batch * P.n_tokens * P.per_token;
    const long long blocks = (P.units + RP_GROUPS - 1) / RP_GROUPS;
    HIRA_CHECK_ARG(blocks < (1ll << 31), HIRA_ERR_SHAPE, "hira_qk_norm_rope: %lld groups of heads exceed the grid limit", P.units);
    rope_kernel<T, TT, NCH, HPG, PAIRS><<<(unsigned)blocks, RP_THREADS, 0, s>>>(P);
    HIRA_CHECK_LAUNCH("hira_qk_norm_rope launch");
    return HIRA_OK;
}
template <typename T, typename TT, int NCH>
static int launch_rope_n(RopeParams& P, int pairs, int batch, cudaStream_t s) {
    // One head a group while that does not fill the GPU with threads several times over (64 tokens of 40 heads); else as many
    // as leave enough warps: four of 128 channels (35 us above; one: 47), two of 256 (65 us for 4,096 tokens; one: 78, four: 84).
    constexpr int MANY = NCH <= 2 ? 4 : 2;
    const bool many = (long long)batch * P.n_tokens * (P.side[0].heads + P.side[1].heads) > 8ll * SM_COUNT * RP_GROUPS;
    if (NCH > 1 && pairs == ROPE_LANE)
        return many ? launch_rope_hp<T, TT, NCH, MANY, ROPE_LANE>(P, batch, s) : launch_rope_hp<T, TT, NCH, 1, ROPE_LANE>(P, batch, s);
    if (pairs == ROPE_XOR)
        return many ? launch_rope_hp<T, TT, NCH, MANY, ROPE_XOR>(P, batch, s) : launch_rope_hp<T, TT, NCH, 1, ROPE_XOR>(P, batch, s);
    if (pairs == ROPE_CHUNK)
        return many ? launch_rope_hp<T, TT, NCH, MANY, ROPE_CHUNK>(P, batch, s) : launch_rope_hp<T, TT, NCH, 1, ROPE_CHUNK>(P, batch, s);
    if (pairs == ROPE_INTERLEAVED)
        return many ? launch_rope_hp<T, TT, NCH, MANY, ROPE_INTERLEAVED>(P, batch, s) : launch_rope_hp<T, TT, NCH, 1, ROPE_INTERLEAVED>(P, batch, s);
    return launch_rope_hp<T, TT, NCH, 1, ROPE_SINGLE>(P, batch, s);
}
template <typename T, typename TT>
static int launch_rope(RopeParams& P, int pairs, int batch, cudaStream_t s) {
    const int nch = chunks_per_lane(P.dim);
    return nch == 1 ? launch_rope_n<T, TT, 1>(P, pairs, batch, s) : nch == 2 ? launch_rope_n<T, TT, 2>(P, pairs, batch, s)
                                                                             : launch_rope_n<T, TT, 4>(P, pairs, batch, s);
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
    P.n_tokens = a->n_tokens; P.dim = a->dim; P.rotary = a->rotary; P.eps = a->eps; P.inv_dim = 1.0f / (float)a->dim;
    // a token's tables may start anywhere, its weights too (they are loaded in 16-byte pieces)
    const int ts = (int)elem_size(a->table_dtype);
    P.wide_tables = (((uintptr_t)a->cos | (uintptr_t)a->sin | (uintptr_t)((P.cs[0] | P.cs[1] | P.ss[0] | P.ss[1]) * ts)) & 15) == 0;
    const int pairs = a->interleaved ? ROPE_INTERLEAVED : a->rotary % 16 ? ROPE_SINGLE : a->rotary == 128 || a->rotary == 256 ? ROPE_LANE
                      : a->rotary == 16 || a->rotary == 32 || a->rotary == 64 ? ROPE_XOR : ROPE_CHUNK;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == HIRA_BF16)
        return a->table_dtype == HIRA_BF16 ? launch_rope<__nv_bfloat16, __nv_bfloat16>(P, pairs, a->batch, s) : launch_rope<__nv_bfloat16, float>(P, pairs, a->batch, s);
    return a->table_dtype == HIRA_BF16 ? launch_rope<float, __nv_bfloat16>(P, pairs, a->batch, s) : launch_rope<float, float>(P, pairs, a->batch, s);
}
