// Decode attention of a batch whose sequences ("branches") share their prompts.
//
//   out[b, hq, t] = softmax(sm_scale * q[b, hq, t] . K) V  over the keys K = prefix[prompt(b)] ++ tail[b]
//
// The prefix of a prompt serves all its branches: its keys and values are read once for all query rows of a kv head
// (branches x group x tokens) instead of once a branch.  A tail is a branch's own; its last n_q keys are those of the
// query tokens, so token t sees the first tail_len - (n_q - 1 - t) of them.
//
// Prefix and tails give softmax partials (m, l, o) per output row, which the merge joins:
//   M = max m_i,  out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i,  and 0 for a row that saw no key.
#include "shared_attn.cuh"
#include <math_constants.h>

namespace hira {

constexpr int SA_THREADS = 128;
constexpr int SA_KEYS = 64;       // keys a tile
constexpr int SA_PAD = 4;         // floats behind each row in shared memory: rows 4 banks apart

// ---------------------------------------------------------------------------
// CUDA-core kernel for fp32.
//
// One block takes ROWS = 8 * RPT query rows of one item against a run of the item's keys, in tiles of 64 in
// shared memory.  16 lanes share RPT rows: for the products of a tile a lane has RPT rows x 4 keys in registers
// (RPT + 4 16-byte loads for 16 RPT FMAs), for the weighted sums RPT rows x V / 16 channels.  A row's softmax
// statistics stay with its 16 lanes, so the blocks only meet to exchange tiles.  fp32 products and sums throughout.
// Bound by shared memory's ports and issue slots: 64 rows of 8 heads at 8,192 keys of 128, 137 us (1.07 G multiply-adds of the
// products and as many of the sums: 31 TFLOP/s).
// ---------------------------------------------------------------------------
// Rows k0 .. k0 + 63 of keys or values into shared memory; those from `len` on as 0, nothing of them is read.
// A thread keeps its piece of the rows where the pieces divide the threads.
template <typename F>
__device__ __forceinline__ void sa_pieces(int pieces, F&& f) {
    if (SA_THREADS % pieces == 0) {
        const int c = threadIdx.x % pieces, step = SA_THREADS / pieces;
#pragma unroll 4
        for (int r = threadIdx.x / pieces; r < SA_KEYS; r += step) f(r, c);
    } else {
        for (int i = threadIdx.x; i < SA_KEYS * pieces; i += SA_THREADS) f(i / pieces, i % pieces);
    }
}
__device__ __forceinline__ void sa_load_tile(float* dst, int ld, const float* src, long long stride, int k0, int len, int width) {
    const uint32_t d0 = (uint32_t)__cvta_generic_to_shared(dst);
    sa_pieces(width / 4, [&](int r, int c) {
        const bool there = k0 + r < len;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(d0 + (uint32_t)(r * ld + c * 4) * 4),
                     "l"(there ? src + (k0 + r) * stride + c * 4 : src), "r"(there ? 16 : 0) : "memory");
    });
    asm volatile("cp.async.commit_group;\n" ::: "memory");
}
template <int N>
__device__ __forceinline__ void sa_landed() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

template <int RPT, int NV, bool TAIL>
__global__ void __launch_bounds__(SA_THREADS)
shared_simt_kernel(const SharedAttn P) {
    constexpr int ROWS = 8 * RPT;
    extern __shared__ __align__(16) float sa_smem[];
    const int ldk = P.dim + SA_PAD, ldv = P.vdim + SA_PAD;
    float* s_q = sa_smem;                       // [ROWS][ldk]
    float* s_k = s_q + ROWS * ldk;              // [SA_KEYS][ldk]
    float* s_v = s_k + SA_KEYS * ldk;           // [SA_KEYS][ldv]
    float* s_p = s_v + SA_KEYS * ldv;           // [SA_KEYS][ROWS + SA_PAD]
    constexpr int LDP = ROWS + SA_PAD;

    grid_trigger();             // who follows waits before it reads
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int row0 = blockIdx.x * ROWS, split = blockIdx.y;
    const int item = blockIdx.z, h = item % P.n_kv, owner = item / P.n_kv;      // prompt, or branch of a tail
    const int per = P.group * P.n_q;
    const int n_rows = TAIL ? per : P.n_branches * per;
    const int n_splits = TAIL ? P.tail_parts : P.prefix_parts;
    const int len = TAIL ? shared_tail_len(P, owner) : shared_prefix_len(P, owner);
    const float* gk = reinterpret_cast<const float*>(TAIL ? P.tk : P.pk) + owner * (TAIL ? P.tks[0] : P.pks[0]) + h * (TAIL ? P.tks[1] : P.pks[1]);
    const float* gv = reinterpret_cast<const float*>(TAIL ? P.tv : P.pv) + owner * (TAIL ? P.tvs[0] : P.pvs[0]) + h * (TAIL ? P.tvs[1] : P.pvs[1]);
    const long long ks = TAIL ? P.tks[2] : P.pks[2], vs = TAIL ? P.tvs[2] : P.pvs[2];
    auto out_row = [&](int r) {
        return TAIL ? (owner * P.n_kv + h) * per + r : shared_row(P, owner, h, r);
    };

    const int kc = P.dim / 8;
    for (int i = tid; i < ROWS * kc; i += SA_THREADS) {
        const int r = i / kc, c = i - r * kc;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (row0 + r < n_rows)
            to_float(load_chunk<float>(reinterpret_cast<const float*>(P.q) + shared_row_offset(P, out_row(row0 + r), P.qs), c), f);
        float4* d = reinterpret_cast<float4*>(s_q + r * ldk + c * 8);
        d[0] = make_float4(f[0], f[1], f[2], f[3]);
        d[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
    // keys this row sees
    int seen[RPT];
    float m[RPT], l[RPT], o[RPT][NV][4];
#pragma unroll
    for (int a = 0; a < RPT; ++a) {
        const int r = row0 + ty * RPT + a;
        seen[a] = TAIL ? len - (P.n_q - 1 - r % P.n_q) : len;
        m[a] = -CUDART_INF_F;
        l[a] = 0.f;
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[a][c][e] = 0.f;
    }
    // equal runs of tiles for the splits
    const int tiles = (len + SA_KEYS - 1) / SA_KEYS;
    const int t0 = (int)((long long)split * tiles / n_splits), t1 = (int)((long long)(split + 1) * tiles / n_splits);
    // the values of a tile arrive while its products are formed, the next keys while its values are summed
    if (t0 < t1) sa_load_tile(s_k, ldk, gk, ks, t0 * SA_KEYS, len, P.dim);
    for (int t = t0; t < t1; ++t) {
        const int k0 = t * SA_KEYS;
        sa_load_tile(s_v, ldv, gv, vs, k0, len, P.vdim);
        sa_landed<1>();
        __syncthreads();      // the keys are there (and the queries)
        float s[RPT][4];
#pragma unroll
        for (int a = 0; a < RPT; ++a)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[a][j] = 0.f;
        const float* qrow = s_q + ty * RPT * ldk;
        const float* krow = s_k + tx * ldk;
#pragma unroll 2
        for (int d = 0; d < P.dim; d += 4) {
            float4 kk[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) kk[j] = *reinterpret_cast<const float4*>(krow + 16 * j * ldk + d);
#pragma unroll
            for (int a = 0; a < RPT; ++a) {
                const float4 qq = *reinterpret_cast<const float4*>(qrow + a * ldk + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[a][j] = __fmaf_rn(qq.x, kk[j].x, s[a][j]);
                    s[a][j] = __fmaf_rn(qq.y, kk[j].y, s[a][j]);
                    s[a][j] = __fmaf_rn(qq.z, kk[j].z, s[a][j]);
                    s[a][j] = __fmaf_rn(qq.w, kk[j].w, s[a][j]);
                }
            }
        }
        __syncthreads();      // and used up
        if (t + 1 < t1) {
            sa_load_tile(s_k, ldk, gk, ks, k0 + SA_KEYS, len, P.dim);
            sa_landed<1>();
        } else {
            sa_landed<0>();
        }
#pragma unroll
        for (int a = 0; a < RPT; ++a) {
            float mx = -CUDART_INF_F;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[a][j] = k0 + tx + 16 * j < seen[a] ? s[a][j] * P.scale_log2 : -CUDART_INF_F;
                mx = fmaxf(mx, s[a][j]);
            }
#pragma unroll
            for (int w = 8; w >= 1; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float nm = fmaxf(m[a], mx), base = nm > -CUDART_INF_F ? nm : 0.f;
            const float alpha = exp2_approx(m[a] - base);
            m[a] = nm;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[a][j] = exp2_approx(s[a][j] - base);
                sum += s[a][j];
            }
#pragma unroll
            for (int w = 8; w >= 1; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            l[a] = __fmaf_rn(l[a], alpha, sum);
#pragma unroll
            for (int c = 0; c < NV; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[a][c][e] *= alpha;
#pragma unroll
            for (int j = 0; j < 4; ++j) s_p[(tx + 16 * j) * LDP + ty * RPT + a] = s[a][j];
        }
        __syncthreads();      // the values are there; a row's weights pass between its 16 lanes only
#pragma unroll 2
        for (int k = 0; k < SA_KEYS; ++k) {
            float p[RPT];
#pragma unroll
            for (int a = 0; a < RPT; ++a) p[a] = s_p[k * LDP + ty * RPT + a];
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const int ch = tx * 4 + 64 * c;
                if (ch < P.vdim) {
                    const float4 v = *reinterpret_cast<const float4*>(s_v + k * ldv + ch);
#pragma unroll
                    for (int a = 0; a < RPT; ++a) {
                        o[a][c][0] = __fmaf_rn(p[a], v.x, o[a][c][0]);
                        o[a][c][1] = __fmaf_rn(p[a], v.y, o[a][c][1]);
                        o[a][c][2] = __fmaf_rn(p[a], v.z, o[a][c][2]);
                        o[a][c][3] = __fmaf_rn(p[a], v.w, o[a][c][3]);
                    }
                }
            }
        }
        __syncthreads();      // the values are used up
    }
    const int part = (TAIL ? P.prefix_parts : 0) + split;
#pragma unroll
    for (int a = 0; a < RPT; ++a) {
        const int r = row0 + ty * RPT + a;
        if (r >= n_rows) continue;
        const size_t at = (size_t)part * P.n_rows + out_row(r);
        if (tx == 0) P.part_ml[at] = make_float2(m[a], l[a]);
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int ch = tx * 4 + 64 * c;
            if (ch < P.vdim) *reinterpret_cast<float4*>(P.part_o + at * P.vdim + ch) = make_float4(o[a][c][0], o[a][c][1], o[a][c][2], o[a][c][3]);
        }
    }
    if (!TAIL) grid_wait();     // so that who waits for this waits for the tails too
}

// ---------------------------------------------------------------------------
// The same for few rows (8 or 16 a block), where shared memory's ports bound the kernel above: here a thread forms one
// key's products with ALL rows (half of the channels each; the key is read once, the queries are broadcasts), a warp
// then takes whole rows for their softmax, and for the weighted sums a warp takes 16 of the 64 keys and a lane four
// channels of all rows.  The four warps' sums are added up once, at the end.
// 8 rows of 8 heads at 32,768 keys of 128 (268 MB): 82..86 us (3.2 TB/s), 16 rows 121 (the kernel above: 209 both).  Bound by the
// rows' broadcasts: each costs a warp four cycles of shared memory's port, as a row of its own would.
// ---------------------------------------------------------------------------
template <int ROWS, int NV, bool TAIL>
__global__ void __launch_bounds__(SA_THREADS)
shared_few_kernel(const SharedAttn P) {
    extern __shared__ __align__(16) float sa_smem[];
    const int ldk = P.dim + SA_PAD, ldv = P.vdim + SA_PAD;
    float* s_q = sa_smem;                       // [ROWS][ldk]
    float* s_k = s_q + ROWS * ldk;              // [SA_KEYS][ldk]
    float* s_v = s_k + SA_KEYS * ldk;           // [SA_KEYS][ldv]
    float* s_p = s_v + SA_KEYS * ldv;           // [SA_KEYS][ROWS + SA_PAD]: logits, then weights
    constexpr int LDP = ROWS + SA_PAD;
    __shared__ float s_alpha[ROWS];
    grid_trigger();             // who follows waits before it reads
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row0 = blockIdx.x * ROWS, split = blockIdx.y;
    const int item = blockIdx.z, h = item % P.n_kv, owner = item / P.n_kv;      // prompt, or branch of a tail
    const int per = P.group * P.n_q;
    const int n_rows = TAIL ? per : P.n_branches * per;
    const int n_splits = TAIL ? P.tail_parts : P.prefix_parts;
    const int len = TAIL ? shared_tail_len(P, owner) : shared_prefix_len(P, owner);
    const float* gk = reinterpret_cast<const float*>(TAIL ? P.tk : P.pk) + owner * (TAIL ? P.tks[0] : P.pks[0]) + h * (TAIL ? P.tks[1] : P.pks[1]);
    const float* gv = reinterpret_cast<const float*>(TAIL ? P.tv : P.pv) + owner * (TAIL ? P.tvs[0] : P.pvs[0]) + h * (TAIL ? P.tvs[1] : P.pvs[1]);
    const long long ks = TAIL ? P.tks[2] : P.pks[2], vs = TAIL ? P.tvs[2] : P.pvs[2];
    auto out_row = [&](int r) {
        return TAIL ? (owner * P.n_kv + h) * per + r : shared_row(P, owner, h, r);
    };
    const int tiles = (len + SA_KEYS - 1) / SA_KEYS;
    const int t0 = (int)((long long)split * tiles / n_splits), t1 = (int)((long long)(split + 1) * tiles / n_splits);
    if (t0 < t1) sa_load_tile(s_k, ldk, gk, ks, t0 * SA_KEYS, len, P.dim);
    const int kc = P.dim / 8;
    for (int i = tid; i < ROWS * kc; i += SA_THREADS) {
        const int r = i / kc, c = i - r * kc;
        float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (row0 + r < n_rows)
            to_float(load_chunk<float>(reinterpret_cast<const float*>(P.q) + shared_row_offset(P, out_row(row0 + r), P.qs), c), f);
        float4* d = reinterpret_cast<float4*>(s_q + r * ldk + c * 8);
        d[0] = make_float4(f[0], f[1], f[2], f[3]);
        d[1] = make_float4(f[4], f[5], f[6], f[7]);
    }
    constexpr int WROWS = ROWS / 4;             // rows of a warp's softmax: warp, warp + 4, ...
    float m[WROWS], l[WROWS], o[ROWS][NV][4];
#pragma unroll
    for (int a = 0; a < WROWS; ++a) {
        m[a] = -CUDART_INF_F;
        l[a] = 0.f;
    }
#pragma unroll
    for (int a = 0; a < ROWS; ++a)
#pragma unroll
        for (int c = 0; c < NV; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[a][c][e] = 0.f;
    const int key = tid & 63, half = tid >> 6, d0 = half ? (P.dim / 8 + 1) / 2 * 8 : 0, d1 = half ? P.dim : (P.dim / 8 + 1) / 2 * 8;
    for (int t = t0; t < t1; ++t) {
        const int k0 = t * SA_KEYS;
        sa_load_tile(s_v, ldv, gv, vs, k0, len, P.vdim);
        sa_landed<1>();
        __syncthreads();      // the keys are there (and the queries)
        float s[ROWS];
#pragma unroll
        for (int a = 0; a < ROWS; ++a) s[a] = 0.f;
#pragma unroll 2
        for (int d = d0; d < d1; d += 4) {
            const float4 kk = *reinterpret_cast<const float4*>(s_k + key * ldk + d);
#pragma unroll
            for (int a = 0; a < ROWS; ++a) {
                const float4 qq = *reinterpret_cast<const float4*>(s_q + a * ldk + d);
                s[a] = __fmaf_rn(qq.x, kk.x, s[a]);
                s[a] = __fmaf_rn(qq.y, kk.y, s[a]);
                s[a] = __fmaf_rn(qq.z, kk.z, s[a]);
                s[a] = __fmaf_rn(qq.w, kk.w, s[a]);
            }
        }
        if (half)
#pragma unroll
            for (int a = 0; a < ROWS; a += 4) *reinterpret_cast<float4*>(s_p + key * LDP + a) = make_float4(s[a], s[a + 1], s[a + 2], s[a + 3]);
        __syncthreads();      // the keys are used up, the second halves there
        if (t + 1 < t1) sa_load_tile(s_k, ldk, gk, ks, k0 + SA_KEYS, len, P.dim);
        if (!half)
#pragma unroll
            for (int a = 0; a < ROWS; a += 4) {
                float4* at = reinterpret_cast<float4*>(s_p + key * LDP + a);
                const float4 x = *at;
                *at = make_float4(s[a] + x.x, s[a + 1] + x.y, s[a + 2] + x.z, s[a + 3] + x.w);
            }
        __syncthreads();
#pragma unroll
        for (int a = 0; a < WROWS; ++a) {
            const int r = warp + 4 * a, seen = TAIL ? len - (P.n_q - 1 - (row0 + r) % P.n_q) : len;
            float x[2], mx;
#pragma unroll
            for (int j = 0; j < 2; ++j) x[j] = k0 + lane + 32 * j < seen ? s_p[(lane + 32 * j) * LDP + r] * P.scale_log2 : -CUDART_INF_F;
            mx = fmaxf(x[0], x[1]);
#pragma unroll
            for (int w = 16; w >= 1; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float nm = fmaxf(m[a], mx), base = nm > -CUDART_INF_F ? nm : 0.f;
            const float alpha = exp2_approx(m[a] - base);
            m[a] = nm;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                x[j] = exp2_approx(x[j] - base);
                sum += x[j];
                s_p[(lane + 32 * j) * LDP + r] = x[j];
            }
#pragma unroll
            for (int w = 16; w >= 1; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            l[a] = __fmaf_rn(l[a], alpha, sum);
            if (lane == 0) s_alpha[r] = alpha;
        }
        if (t + 1 < t1) sa_landed<1>();
        else sa_landed<0>();
        __syncthreads();      // the values and the weights are there
#pragma unroll
        for (int a = 0; a < ROWS; ++a) {
            const float alpha = s_alpha[a];
#pragma unroll
            for (int c = 0; c < NV; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[a][c][e] *= alpha;
        }
#pragma unroll 2
        for (int k = warp * (SA_KEYS / 4); k < (warp + 1) * (SA_KEYS / 4); ++k) {
            float4 v[NV];
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const int ch = lane * 4 + 128 * c;
                v[c] = ch < P.vdim ? *reinterpret_cast<const float4*>(s_v + k * ldv + ch) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int a = 0; a < ROWS; a += 4) {
                const float4 p = *reinterpret_cast<const float4*>(s_p + k * LDP + a);
                const float pp[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int c = 0; c < NV; ++c) {
                        o[a + b][c][0] = __fmaf_rn(pp[b], v[c].x, o[a + b][c][0]);
                        o[a + b][c][1] = __fmaf_rn(pp[b], v[c].y, o[a + b][c][1]);
                        o[a + b][c][2] = __fmaf_rn(pp[b], v[c].z, o[a + b][c][2]);
                        o[a + b][c][3] = __fmaf_rn(pp[b], v[c].w, o[a + b][c][3]);
                    }
            }
        }
        __syncthreads();      // the values are used up
    }
    // the warps' sums added up, in the tiles' place
    float* s_o = s_k;         // [4][ROWS][ldv]
    __syncthreads();
#pragma unroll
    for (int a = 0; a < ROWS; ++a)
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int ch = lane * 4 + 128 * c;
            if (ch < P.vdim) *reinterpret_cast<float4*>(s_o + (warp * ROWS + a) * ldv + ch) = make_float4(o[a][c][0], o[a][c][1], o[a][c][2], o[a][c][3]);
        }
    __syncthreads();
    const int part = (TAIL ? P.prefix_parts : 0) + split;
#pragma unroll
    for (int a = 0; a < WROWS; ++a) {
        const int r = warp + 4 * a;
        if (row0 + r >= n_rows) continue;
        const size_t at = (size_t)part * P.n_rows + out_row(row0 + r);
        if (lane == 0) P.part_ml[at] = make_float2(m[a], l[a]);
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int ch = lane * 4 + 128 * c;
            if (ch >= P.vdim) continue;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(s_o + (w * ROWS + r) * ldv + ch);
                y.x += x.x; y.y += x.y; y.z += x.z; y.w += x.w;
            }
            *reinterpret_cast<float4*>(P.part_o + at * P.vdim + ch) = y;
        }
    }
    if (!TAIL) grid_wait();     // so that who waits for this waits for the tails too
}

// ---------------------------------------------------------------------------
// The partials of an output row joined, by W warps: each weighs all parts (a lane a part), sums every W-th and the
// first adds the sums up.  A few megabytes out of L2: bound by the round trips, so all loads of a round are issued at
// once, and where a row has many parts four warps share them.  540 rows of some 13 parts: 4 us behind the last part.
// ---------------------------------------------------------------------------
constexpr int SA_MERGE_WARPS = 4;
constexpr int SA_FLIGHT = 8;      // parts of a row on their way at once, for each warp

template <typename T, int W>
__global__ void __launch_bounds__(32 * SA_MERGE_WARPS)
shared_merge_kernel(const SharedAttn P) {
    __shared__ float s_w[SA_MERGE_WARPS / W][SA_MAX_PARTS];
    __shared__ float4 s_o[SA_MERGE_WARPS][64];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wi = warp % W, slot = warp / W;
    const int R = blockIdx.x * (SA_MERGE_WARPS / W) + slot;
    const bool there = R < P.n_rows;
    const int row = there ? R : P.n_rows - 1, bh = row / P.n_q, heads = P.n_kv * P.group;
    const int item = bh / heads / P.n_branches * P.n_kv + bh % heads / P.group;
    // the partials there are: the item's own, then (from prefix_parts on) the tail's
    const int np = P.prefix_parts > 0 ? shared_item_parts(P, item) : 0, n = np + P.tail_parts, gap = P.prefix_parts - np;
    auto part = [&](int i) { return (size_t)(i < np ? i : i + gap) * P.n_rows + row; };
    grid_wait();
    // the first parts' rows are asked for together with the maxima that weigh them: one round trip less
    float4 x[SA_FLIGHT];
    auto load = [&](int c, int i0) {
        const int ch = lane * 4 + c * 128;
        const float* src = P.part_o + (ch < P.vdim ? ch : 0);
#pragma unroll
        for (int j = 0; j < SA_FLIGHT; ++j) x[j] = *reinterpret_cast<const float4*>(src + part(min(i0 + j * W, n - 1)) * P.vdim);
    };
    if (n > 0) load(0, wi);
    float M = -CUDART_INF_F;
    bool bad = false;
    for (int i = lane; i < n; i += 32) {
        const float2 ml = P.part_ml[part(i)];
        bad |= ml.x != ml.x || ml.y != ml.y;       // a NaN among the logits, which a maximum passes over
        M = fmaxf(M, ml.x);
    }
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
    const float base = M > -CUDART_INF_F ? M : 0.f;
    float L = 0.f;
    for (int i = lane; i < n; i += 32) {
        const float2 ml = P.part_ml[part(i)];
        const float w = ml.x > -CUDART_INF_F ? exp2_approx(ml.x - base) : 0.f;      // a part without keys has no sums either
        L += w > 0.f ? w * ml.y : 0.f;
        if (i % W == wi) s_w[slot][i] = w;         // the parts this warp sums
    }
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1) L += __shfl_xor_sync(0xffffffffu, L, w);
    if (__any_sync(0xffffffffu, bad)) L = CUDART_NAN_F;
    __syncwarp();
    float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        if (c * 128 >= P.vdim) break;
        for (int i0 = wi; i0 < n; i0 += W * SA_FLIGHT) {
            if (c > 0 || i0 != wi) load(c, i0);
#pragma unroll
            for (int j = 0; j < SA_FLIGHT; ++j) {
                const float w = i0 + j * W < n ? s_w[slot][i0 + j * W] : 0.f;
                if (w != 0.f) {      // what a part without keys has there is not used, whatever it is
                    acc[c].x = __fmaf_rn(w, x[j].x, acc[c].x); acc[c].y = __fmaf_rn(w, x[j].y, acc[c].y);
                    acc[c].z = __fmaf_rn(w, x[j].z, acc[c].z); acc[c].w = __fmaf_rn(w, x[j].w, acc[c].w);
                }
            }
        }
    }
    if (W > 1) {
        s_o[warp][lane] = acc[0];
        s_o[warp][lane + 32] = acc[1];
        __syncthreads();
        if (wi != 0) return;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int w = 1; w < W; ++w) {
                const float4 x = s_o[warp + w][lane + 32 * c];
                acc[c].x += x.x; acc[c].y += x.y; acc[c].z += x.z; acc[c].w += x.w;
            }
    }
    if (!there) return;
    T* out = reinterpret_cast<T*>(P.out) + shared_row_offset(P, R, P.os);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int ch = lane * 4 + c * 128;
        if (ch >= P.vdim) continue;
        float4 y;      // no key seen: 0 (a NaN stays one)
        y.x = L == 0.f ? 0.f : acc[c].x / L; y.y = L == 0.f ? 0.f : acc[c].y / L;
        y.z = L == 0.f ? 0.f : acc[c].z / L; y.w = L == 0.f ? 0.f : acc[c].w / L;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(out + ch) = y;
        } else {
            __nv_bfloat162 lo = __floats2bfloat162_rn(y.x, y.y), hi = __floats2bfloat162_rn(y.z, y.w);
            *reinterpret_cast<uint2*>(out + ch) = make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
        }
    }
}

template <int RPT, int NV, bool TAIL>
static auto simt_kernel() {      // NV: 64 channels each of 16 lanes, or (few rows) 128 each of a warp
    if constexpr (RPT <= 2) return shared_few_kernel<8 * RPT, NV / 2, TAIL>;
    else return shared_simt_kernel<RPT, NV, TAIL>;
}
static size_t simt_smem(int block_rows, int dim, int vdim) {
    return sizeof(float) * ((size_t)(block_rows + SA_KEYS) * (dim + SA_PAD) + (size_t)SA_KEYS * (vdim + SA_PAD) +
                            (size_t)SA_KEYS * (block_rows + SA_PAD));
}

template <int RPT, int NV, bool TAIL>
static int launch_simt(const SharedAttn& P, bool chained, cudaStream_t s) {
    auto kern = simt_kernel<RPT, NV, TAIL>();
    const int per = P.group * P.n_q, rows = TAIL ? per : P.n_branches * per;
    const size_t smem = simt_smem(8 * RPT, P.dim, P.vdim);
    static SmemLimit limit;
    cudaError_t e = limit.raise(kern, (int)smem);
    if (e != cudaSuccess) {
        set_error("hira_shared_attn: cudaFuncSetAttribute(%zu B smem): %s", smem, cudaGetErrorString(e));
        return HIRA_ERR_CUDA;
    }
    const dim3 grid((unsigned)((rows + 8 * RPT - 1) / (8 * RPT)), (unsigned)(TAIL ? P.tail_parts : P.prefix_parts),
                    (unsigned)((TAIL ? P.n_prompts * P.n_branches : P.n_prompts) * P.n_kv));
    if (chained) {
        e = launch_chained(kern, grid, dim3(SA_THREADS), smem, s, P);
    } else {
        kern<<<grid, SA_THREADS, smem, s>>>(P);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) {
        set_error("hira_shared_attn launch: %s", cudaGetErrorString(e));
        return HIRA_ERR_CUDA;
    }
    return HIRA_OK;
}

// rows a block takes: no more than there are, so that a few rows do not pay for the products of many
static int simt_rows(int rows, int vdim) { return rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 || vdim > 128 ? 32 : 64; }

template <bool TAIL>
static int launch_simt_rows(const SharedAttn& P, bool chained, cudaStream_t s) {
    const int per = P.group * P.n_q, rows = simt_rows(TAIL ? per : P.n_branches * per, P.vdim);
    if (P.vdim > 128) {
        if (rows == 8) return launch_simt<1, 4, TAIL>(P, chained, s);
        if (rows == 16) return launch_simt<2, 4, TAIL>(P, chained, s);
        return launch_simt<4, 4, TAIL>(P, chained, s);
    }
    if (rows == 8) return launch_simt<1, 2, TAIL>(P, chained, s);
    if (rows == 16) return launch_simt<2, 2, TAIL>(P, chained, s);
    if (rows == 32) return launch_simt<4, 2, TAIL>(P, chained, s);
    return launch_simt<8, 2, TAIL>(P, chained, s);
}

// Splits of the keys: as many blocks as are resident at once -- what an SM's shared memory holds, but no more than three of those
// with few rows and two of the others --, none with fewer than two tiles.  128 channels (three an SM of 8 rows, two of 16 and 32, one
// of 64), us with one / two / three an SM: 8 heads, 32,768 keys, 8 rows 123 / 88 / 82, 16 rows 162 / 121 / 158, 32 rows 311 / 203 /
// 272; 9,000 keys, 64 rows 131 / 141 / 162; one head, 32,768 keys, 16 rows 37 / 39 / 35.  256 channels (one), 8 heads, 9,000 keys,
// 8 rows 61 / 68 / 80.
constexpr int SA_SM_SMEM = 228 * 1024, SA_BLOCK_RESERVE = 1024;      // bytes an SM has, and keeps for itself of each block's
static int simt_splits(int rows, int items, int len, int dim, int vdim) {
    if (len <= 0) return 0;
    const int block_rows = simt_rows(rows, vdim), tiles = (len + SA_KEYS - 1) / SA_KEYS;
    const long long blocks = (long long)((rows + block_rows - 1) / block_rows) * items;
    long long resident = SA_SM_SMEM / (long long)(simt_smem(block_rows, dim, vdim) + SA_BLOCK_RESERVE);
    if (resident > (block_rows <= 16 ? 3 : 2)) resident = block_rows <= 16 ? 3 : 2;
    if (resident < 1) resident = 1;
    long long splits = resident * SM_COUNT / blocks;
    if (splits > (tiles + 1) / 2) splits = (tiles + 1) / 2;
    if (splits > SA_MAX_PARTS / 2) splits = SA_MAX_PARTS / 2;
    return splits < 1 ? 1 : (int)splits;
}

static int shared_plan(const hira_shared_attn_t* a, SharedAttn& P) {
    HIRA_CHECK_ARG(a != nullptr, HIRA_ERR_ARG, "hira_shared_attn: arguments are NULL");
    HIRA_CHECK_ARG(a->dtype == HIRA_F32 || a->dtype == HIRA_BF16, HIRA_ERR_DTYPE,
                   "hira_shared_attn: dtype %d is neither HIRA_F32 nor HIRA_BF16", a->dtype);
    HIRA_CHECK_ARG(a->n_prompts >= 1 && a->n_branches >= 1 && a->n_kv >= 1 && a->group >= 1 && a->n_q >= 1, HIRA_ERR_SHAPE,
                   "hira_shared_attn: n_prompts=%d n_branches=%d n_kv=%d group=%d n_q=%d must be >= 1", a->n_prompts,
                   a->n_branches, a->n_kv, a->group, a->n_q);
    HIRA_CHECK_ARG(a->dim >= 8 && a->dim <= 256 && a->dim % 8 == 0 && a->vdim >= 8 && a->vdim <= 256 && a->vdim % 8 == 0,
                   HIRA_ERR_SHAPE, "hira_shared_attn: dim=%d and vdim=%d must be multiples of 8 in 8..256", a->dim, a->vdim);
    HIRA_CHECK_ARG(a->prefix_len >= 0 && a->tail_len >= 0 && a->prefix_len < (1 << 30) && a->tail_len < (1 << 30), HIRA_ERR_SHAPE,
                   "hira_shared_attn: prefix_len=%d tail_len=%d outside 0..2^30", a->prefix_len, a->tail_len);
    const long long rows = (long long)a->n_prompts * a->n_branches * a->n_kv * a->group * a->n_q;
    HIRA_CHECK_ARG(rows < (1ll << 30) && (long long)a->n_prompts * a->n_branches * a->n_kv <= 65535, HIRA_ERR_SHAPE,
                   "hira_shared_attn: %lld query rows, or %lld (branch, kv head) pairs, exceed 2^30 or 65535", rows,
                   (long long)a->n_prompts * a->n_branches * a->n_kv);
    HIRA_CHECK_ARG(a->q && a->out, HIRA_ERR_ARG, "hira_shared_attn: q and out must not be NULL");
    HIRA_CHECK_ARG(a->prefix_len == 0 || (a->prefix_k && a->prefix_v), HIRA_ERR_ARG, "hira_shared_attn: prefix_k / prefix_v is NULL");
    HIRA_CHECK_ARG(a->tail_len == 0 || (a->tail_k && a->tail_v), HIRA_ERR_ARG, "hira_shared_attn: tail_k / tail_v is NULL");
    const int es = (int)elem_size(a->dtype);
    HIRA_CHECK_ARG(((uintptr_t)a->status & 3) == 0, HIRA_ERR_ARG, "hira_shared_attn: status is no 4-byte word");
    uintptr_t mis = (uintptr_t)a->q | (uintptr_t)a->out;
    const void* kv[4] = {a->prefix_k, a->prefix_v, a->tail_k, a->tail_v};
    const int64_t* st[6] = {a->prefix_k_stride, a->prefix_v_stride, a->tail_k_stride, a->tail_v_stride, a->q_stride, a->out_stride};
    for (int i = 0; i < 4; ++i)
        if (i < 2 ? a->prefix_len : a->tail_len) mis |= (uintptr_t)kv[i] | (uintptr_t)((st[i][0] | st[i][1] | st[i][2]) * es);
    for (int i = 4; i < 6; ++i) mis |= (uintptr_t)((st[i][0] | st[i][1] | st[i][2]) * es);
    HIRA_CHECK_ARG((mis & 15) == 0, HIRA_ERR_ARG, "hira_shared_attn: every row must start on a 16-byte boundary");
    P = SharedAttn{};
    P.q = a->q; P.out = a->out;
    P.pk = a->prefix_k; P.pv = a->prefix_v; P.tk = a->tail_k; P.tv = a->tail_v;
    P.prefix_lens = a->prefix_lens; P.tail_lens = a->tail_lens; P.status = a->status;
    P.n_prompts = a->n_prompts; P.n_branches = a->n_branches; P.n_kv = a->n_kv; P.group = a->group; P.n_q = a->n_q;
    P.dim = a->dim; P.vdim = a->vdim; P.prefix_len = a->prefix_len; P.tail_len = a->tail_len;
    P.n_rows = (int)rows;
    P.scale_log2 = (float)((double)a->sm_scale * 1.4426950408889634074);     // log2(e)
    for (int i = 0; i < 3; ++i) {
        P.pks[i] = st[0][i]; P.pvs[i] = st[1][i]; P.tks[i] = st[2][i]; P.tvs[i] = st[3][i]; P.qs[i] = st[4][i]; P.os[i] = st[5][i];
    }
    const int per = a->group * a->n_q;
    const int branches = a->n_prompts * a->n_branches * a->n_kv;
    if (a->dtype == HIRA_BF16) {
        P.tail_parts = shared_mma_splits(P, true);
        if (shared_tc_supported(P) && !shared_mma_prefers(P)) shared_tc_plan(P);
        else P.prefix_parts = shared_mma_splits(P, false);
        P.fused = shared_tail_joins(P);
    } else {
        P.tail_parts = simt_splits(per, branches, a->tail_len, a->dim, a->vdim);
        P.prefix_parts = simt_splits(a->n_branches * per, a->n_prompts * a->n_kv, a->prefix_len, a->dim, a->vdim);
    }
    return HIRA_OK;
}
static size_t shared_parts_bytes(const SharedAttn& P) {
    return (size_t)(P.prefix_parts + (P.fused ? 0 : P.tail_parts)) * P.n_rows * (P.vdim + 2) * sizeof(float);
}

template <typename T>
static int run_shared(const SharedAttn& P, cudaStream_t s) {
    // The first kernel starts when all before it on the stream is done; the ones behind it may start beside it, so each
    // waits for the one before it by its end (the merge: at its start).  With bf16 the prefix's kernel takes whole SMs, and
    // the tail's joins the parts where it can: the tails come second.  With fp32 they come first, so that their few blocks run
    // beside the prefix's instead of behind them (2 prompts x 4 branches of 8 heads, 4,100 keys: 29 us, the other way 35).
    int rc = HIRA_OK;
    if (sizeof(T) == 2) {
        if (P.prefix_parts > 0) rc = P.shares > 0 ? shared_tc_launch(P, s) : shared_mma_launch(P, false, false, s);
        if (rc == HIRA_OK && P.tail_parts > 0) rc = shared_mma_launch(P, true, P.prefix_parts > 0, s);
    } else {
        if (P.tail_parts > 0) rc = launch_simt_rows<true>(P, false, s);
        if (rc == HIRA_OK && P.prefix_parts > 0) rc = launch_simt_rows<false>(P, P.tail_parts > 0, s);
    }
    if (rc != HIRA_OK || P.fused) return rc;
    const int parts = P.prefix_parts + P.tail_parts;
    // four warps a row where its parts fill their flights (36 rows of some 30 parts: 28.7 us the whole call, 32.8 with one), one
    // where they do not (2,048 rows of 2 parts: 41 us, 45 with four)
    const bool many = parts > SA_FLIGHT;
    const int rows = many ? 1 : SA_MERGE_WARPS;
    const dim3 grid((unsigned)((P.n_rows + rows - 1) / rows));
    auto merge = many ? shared_merge_kernel<T, SA_MERGE_WARPS> : shared_merge_kernel<T, 1>;
    cudaError_t e;
    if (parts > 0) {
        e = launch_chained(merge, grid, dim3(32 * SA_MERGE_WARPS), 0, s, P);
    } else {
        merge<<<grid, 32 * SA_MERGE_WARPS, 0, s>>>(P);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) {
        set_error("hira_shared_attn merge launch: %s", cudaGetErrorString(e));
        return HIRA_ERR_CUDA;
    }
    return HIRA_OK;
}

}  // namespace hira

using namespace hira;

extern "C" size_t hira_shared_attn_workspace_bytes(const hira_shared_attn_t* a) {
    SharedAttn P;
    return shared_plan(a, P) == HIRA_OK ? shared_parts_bytes(P) : 0;
}

extern "C" int hira_shared_attn(const hira_shared_attn_t* a, void* workspace, size_t workspace_bytes, void* stream) {
    SharedAttn P;
    const int rc = shared_plan(a, P);
    if (rc != HIRA_OK) return rc;
    const size_t need = shared_parts_bytes(P);
    HIRA_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), HIRA_ERR_CAPACITY,
                   "hira_shared_attn: a 16-byte aligned workspace of %zu bytes is needed, %zu given", need, workspace_bytes);
    P.part_o = reinterpret_cast<float*>(workspace);
    P.part_ml = reinterpret_cast<float2*>(P.part_o + (size_t)(P.prefix_parts + (P.fused ? 0 : P.tail_parts)) * P.n_rows * P.vdim);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return a->dtype == HIRA_BF16 ? run_shared<__nv_bfloat16>(P, s) : run_shared<float>(P, s);
}
