// The tails of hira_shared_attn for bf16, and the prefixes that the tcgen05 kernel does not take (rows wider than 128, strides
// that a tensor map does not take, few keys): few query rows against keys of their own.
//
// Bound by the keys' bytes: 16 query rows cost 16-bit matrix products that hide behind the loads.  A block of four
// warps takes 16 rows of one item -- (branch, kv head) or (prompt, kv head) -- against a run of its keys; each warp takes 16
// keys of every 64, through a ring of its own (cp.async, no barrier between warps), with softmax statistics of its own, and
// the four join once, at the end.  Products by mma.sync m16n8k16: a tail's rows are too few for a tcgen05 tile, which would be
// 7/8 empty.
//
// Measured behind a prefix of 131,072 keys: 64 branches x 8 heads x 256 keys (134 MB) and the join of 19 parts in 20 us
// (6.7 TB/s of the tails alone); 16 branches x 64 keys 6 us, a chain of latencies.  As the prefix's kernel: rows of 256 channels,
// 8 heads at 16,384 keys (134 MB), 8 rows a head 33 us, 16 rows 34 (CUDA cores: 213 and 250), 64 rows 83, 256 rows 309: the keys are
// read again for every 16 rows.  The weights' second bf16 term (2^-16 of a weight between the two) costs 1 us of 33, 12 of 83.
#include "shared_attn.cuh"
#include "tc_common.cuh"
#include <math_constants.h>

namespace hira {

constexpr int TL_WARPS = 4;
constexpr int TL_ROWS = 16;
constexpr int TL_KEYS = 16;                     // keys a warp takes a step
constexpr int TL_STEP = TL_WARPS * TL_KEYS;
constexpr int TL_STAGES = 3;
constexpr float TL_SLACK = 8.0f;
constexpr int TL_FLIGHT = 8;                    // parts of a row on their way at once

template <int HD>
struct TlLayout {
    static constexpr int ROW = HD * 2;                              // bytes
    static constexpr int STAGE = 2 * TL_KEYS * ROW;                 // keys, then values, of one warp
    static constexpr int STAGES = HD == 256 ? 2 : TL_STAGES;
    static constexpr int BYTES = TL_WARPS * STAGES * STAGE;         // the joined sums (16 x HD floats a warp) fit too
};

__device__ __forceinline__ void tl_cp16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void tl_ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tl_ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tl_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tl_pack(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// A block's rows: the tail's sums (in shared memory, of each warp) and the prefix's n parts joined and written.  A warp
// takes R rows at a time, a lane four channels of each.
template <int HD, int R>
__device__ __forceinline__ void tl_join(const SharedAttn& P, const float (*s_m)[TL_ROWS], const float (*s_l)[TL_ROWS], const float* s_o, int n,
                                        int rows, int first_row) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, ch = lane * 4;
    for (int r0 = warp; r0 < rows; r0 += R * TL_WARPS) {
        int row[R];
        float base[R], w_t[R], l_t[R], L[R], wi[R];
        float4 acc[R];
        // the first parts' rows are asked for together with the maxima that weigh them: one round trip less
        float4 x[R][TL_FLIGHT];
        const float* src = P.part_o + (ch < P.vdim ? ch : 0);
        auto load = [&](int i0) {
#pragma unroll
            for (int k = 0; k < R; ++k)
#pragma unroll
                for (int j = 0; j < TL_FLIGHT; ++j)
                    x[k][j] = *reinterpret_cast<const float4*>(src + ((size_t)min(i0 + j, n - 1) * P.n_rows + row[k]) * P.vdim);
        };
#pragma unroll
        for (int k = 0; k < R; ++k) row[k] = first_row + min(r0 + k * TL_WARPS, rows - 1);
        if (n > 0) load(0);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const int r = min(r0 + k * TL_WARPS, rows - 1);
            float m_t = -CUDART_INF_F;
            l_t[k] = L[k] = 0.f;
            for (int w = 0; w < TL_WARPS; ++w) m_t = fmaxf(m_t, s_m[w][r]);
            for (int w = 0; w < TL_WARPS; ++w) l_t[k] += s_m[w][r] > -CUDART_INF_F ? s_l[w][r] * exp2_approx(s_m[w][r] - m_t) : s_l[w][r];
            float M = m_t;
            for (int i = lane; i < n; i += 32) M = fmaxf(M, P.part_ml[(size_t)i * P.n_rows + row[k]].x);
#pragma unroll
            for (int w = 16; w >= 1; w >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, w));
            base[k] = M > -CUDART_INF_F ? M : 0.f;
            w_t[k] = m_t > -CUDART_INF_F ? exp2_approx(m_t - base[k]) : 0.f;
            acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (ch < HD)
                for (int w = 0; w < TL_WARPS; ++w) {
                    const float4 x = *reinterpret_cast<const float4*>(s_o + (w * TL_ROWS + r) * HD + ch);
                    acc[k].x += x.x; acc[k].y += x.y; acc[k].z += x.z; acc[k].w += x.w;
                }
            acc[k].x *= w_t[k]; acc[k].y *= w_t[k]; acc[k].z *= w_t[k]; acc[k].w *= w_t[k];
        }
        for (int i0 = 0; i0 < n; i0 += 32) {
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const float2 ml = i0 + lane < n ? P.part_ml[(size_t)(i0 + lane) * P.n_rows + row[k]] : make_float2(-CUDART_INF_F, 0.f);
                wi[k] = ml.x > -CUDART_INF_F ? exp2_approx(ml.x - base[k]) : 0.f;
                // a NaN among a part's logits, which a maximum passes over, is in its sum (or its maximum)
                L[k] += wi[k] > 0.f ? wi[k] * ml.y : ml.x != ml.x ? ml.x : ml.y != ml.y ? ml.y : 0.f;
            }
            const int count = min(n - i0, 32);
            for (int j0 = 0; j0 < count; j0 += TL_FLIGHT) {
                if (i0 + j0 > 0) load(i0 + j0);
#pragma unroll
                for (int k = 0; k < R; ++k)
#pragma unroll
                    for (int j = 0; j < TL_FLIGHT; ++j) {
                        const float wj = __shfl_sync(0xffffffffu, wi[k], (j0 + j) & 31);
                        if (j0 + j < count && wj != 0.f) {      // what a part without keys has there is not used
                            acc[k].x = __fmaf_rn(wj, x[k][j].x, acc[k].x); acc[k].y = __fmaf_rn(wj, x[k][j].y, acc[k].y);
                            acc[k].z = __fmaf_rn(wj, x[k][j].z, acc[k].z); acc[k].w = __fmaf_rn(wj, x[k][j].w, acc[k].w);
                        }
                    }
            }
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
#pragma unroll
            for (int w = 16; w >= 1; w >>= 1) L[k] += __shfl_xor_sync(0xffffffffu, L[k], w);
            L[k] += w_t[k] > 0.f ? w_t[k] * l_t[k] : l_t[k] != l_t[k] ? l_t[k] : 0.f;
            if (ch < P.vdim && r0 + k * TL_WARPS < rows) {   // no key seen: 0 (a NaN stays one)
                const float inv = L[k] == 0.f ? 0.f : 1.f / L[k];
                const uint2 y = make_uint2(tl_pack(acc[k].x * inv, acc[k].y * inv), tl_pack(acc[k].z * inv, acc[k].w * inv));
                *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(P.out) + shared_row_offset(P, row[k], P.os) + ch) = y;
            }
        }
    }
}

template <int HD, bool TAIL>
__global__ void __launch_bounds__(32 * TL_WARPS, HD == 256 ? 1 : HD == 128 ? 2 : 3)
shared_mma_kernel(const SharedAttn P) {
    using Lay = TlLayout<HD>;
    extern __shared__ __align__(128) unsigned char tl_smem[];
    __shared__ float s_m[TL_WARPS][TL_ROWS], s_l[TL_WARPS][TL_ROWS];
    grid_trigger();      // the merge waits before it reads
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
    const int row0 = blockIdx.x * TL_ROWS, split = blockIdx.y;
    const int owner = blockIdx.z / P.n_kv, h = blockIdx.z % P.n_kv, per = P.group * P.n_q;      // a tail's branch, or a prompt
    const int n_rows = TAIL ? per : P.n_branches * per, n_splits = TAIL ? P.tail_parts : P.prefix_parts;
    const int len = TAIL ? shared_tail_len(P, owner) : shared_prefix_len(P, owner);
    const __nv_bfloat16* gk = reinterpret_cast<const __nv_bfloat16*>(TAIL ? P.tk : P.pk) + owner * (TAIL ? P.tks[0] : P.pks[0]) + h * (TAIL ? P.tks[1] : P.pks[1]);
    const __nv_bfloat16* gv = reinterpret_cast<const __nv_bfloat16*>(TAIL ? P.tv : P.pv) + owner * (TAIL ? P.tvs[0] : P.pvs[0]) + h * (TAIL ? P.tvs[1] : P.pvs[1]);
    const long long ks = TAIL ? P.tks[2] : P.pks[2], vs = TAIL ? P.tvs[2] : P.pvs[2];
    const int out_row0 = (owner * P.n_kv + h) * per;      // of a tail
    auto out_row = [&](int r) { return TAIL ? out_row0 + r : shared_row(P, owner, h, r); };

    // this warp's steps: 16 keys of every 64
    const int steps_all = (len + TL_STEP - 1) / TL_STEP;
    const int t0 = (int)((long long)split * steps_all / n_splits), t1 = (int)((long long)(split + 1) * steps_all / n_splits);
    const uint32_t ring = smem_u32(tl_smem) + warp * Lay::STAGES * Lay::STAGE;
    // A lane copies the same 16 bytes of every RPI-th of a step's keys and values.
    constexpr int CH = HD / 8, RPI = 32 / CH, ITER = TL_KEYS / RPI;
    const int lr = lane / CH, lc = lane % CH;
    const uint32_t dst0 = ring + lr * Lay::ROW;
    const bool in_k = lc * 8 < P.dim, in_v = lc * 8 < P.vdim;      // behind the row's channels: 0
    auto load = [&](int t, int stage) {
        const int k0 = t * TL_STEP + warp * TL_KEYS;
        if (t < t1 && k0 < len) {
            const __nv_bfloat16* src_k = gk + (k0 + lr) * ks + lc * 8;
            const __nv_bfloat16* src_v = gv + (k0 + lr) * vs + lc * 8;
            const long long step_k = RPI * ks, step_v = RPI * vs;
            const uint32_t dst = dst0 + stage * Lay::STAGE;
            const bool whole = k0 + TL_KEYS <= len;
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                const uint32_t at = dst + i * RPI * Lay::ROW + ((lc ^ ((lr + i * RPI) & 7)) << 4);
                const bool row = whole || k0 + lr + i * RPI < len;       // behind the last key: 0
                tl_cp16(at, row && in_k ? src_k : gk, row && in_k);
                tl_cp16(at + TL_KEYS * Lay::ROW, row && in_v ? src_v : gv, row && in_v);
                src_k += step_k;
                src_v += step_v;
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < Lay::STAGES - 1; ++i) load(t0 + i, i);

    // queries as the products want them: rows g and g + 8, two channels a register
    uint32_t q[HD / 16][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int r = row0 + g + 8 * j;
        const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(P.q) + (r < n_rows ? shared_row_offset(P, out_row(r), P.qs) : 0);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int ch = k * 16 + u * 8 + tig * 2;
                q[k][j + 2 * u] = r < n_rows && ch < P.dim ? *reinterpret_cast<const uint32_t*>(src + ch) : 0u;
            }
    }
    int seen[2];
    float m[2], l[2], o[HD / 8][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        seen[j] = TAIL ? len - (P.n_q - 1 - (row0 + g + 8 * j) % P.n_q) : len;
        m[j] = -CUDART_INF_F;
        l[j] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    for (int t = t0; t < t1; ++t) {
        const int stage = (t - t0) % Lay::STAGES;
        load(t + Lay::STAGES - 1, (t - t0 + Lay::STAGES - 1) % Lay::STAGES);
        asm volatile("cp.async.wait_group %0;\n" ::"n"(Lay::STAGES - 1) : "memory");
        __syncwarp();
        const int k0 = t * TL_STEP + warp * TL_KEYS;
        if (k0 < len) {          // the same for the warp
            const uint32_t sk = ring + stage * Lay::STAGE, sv = sk + TL_KEYS * Lay::ROW;
            float s[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int k = 0; k < HD / 32; ++k) {
                    uint32_t kk[4];
                    const int r = n * 8 + (lane & 7), c = k * 4 + (lane >> 3);
                    tl_ldm4(kk, sk + r * Lay::ROW + ((c ^ (r & 7)) << 4));
                    tl_mma(s[n], q[2 * k], kk[0], kk[1]);
                    tl_mma(s[n], q[2 * k + 1], kk[2], kk[3]);
                }
            // The reference maximum of a row moves only when a step exceeds it by 2^8, as in the prefix's kernel.
            float mx[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                mx[j] = -CUDART_INF_F;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = s[n][2 * j + e];
                        x = k0 + n * 8 + tig * 2 + e < seen[j] ? x * P.scale_log2 : -CUDART_INF_F;
                        mx[j] = fmaxf(mx[j], x);
                    }
                mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 1));
                mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 2));
            }
            if (__any_sync(0xffffffffu, mx[0] > m[0] + TL_SLACK || mx[1] > m[1] + TL_SLACK)) {
                float f[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bool rise = mx[j] > m[j] + TL_SLACK;       // from -inf on: always, unless the step is -inf too
                    f[j] = rise ? exp2_approx(m[j] - mx[j]) : 1.f;
                    if (rise) m[j] = mx[j];
                    l[j] *= f[j];
                }
#pragma unroll
                for (int n = 0; n < HD / 8; ++n) {
                    o[n][0] *= f[0]; o[n][1] *= f[0];
                    o[n][2] *= f[1]; o[n][3] *= f[1];
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float base = m[j] > -CUDART_INF_F ? m[j] : 0.f;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = s[n][2 * j + e];
                        x = exp2_approx(x - base);
                        l[j] += x;      // this lane's keys; the four lanes of a row are added at the end
                    }
            }
            const uint32_t p[4] = {tl_pack(s[0][0], s[0][1]), tl_pack(s[0][2], s[0][3]), tl_pack(s[1][0], s[1][1]), tl_pack(s[1][2], s[1][3])};
            uint32_t lo[4];      // what the rounding left: the weights' second terms
#pragma unroll
            for (int x = 0; x < 4; ++x)
                lo[x] = tl_pack(s[x >> 1][2 * (x & 1)] - __uint_as_float(p[x] << 16), s[x >> 1][2 * (x & 1) + 1] - __uint_as_float(p[x] & 0xffff0000u));
#pragma unroll
            for (int n = 0; n < HD / 16; ++n) {
                uint32_t vv[4];
                const int r = ((lane >> 3) & 1) * 8 + (lane & 7), c = n * 2 + (lane >> 4);
                tl_ldm4t(vv, sv + r * Lay::ROW + ((c ^ (r & 7)) << 4));
                tl_mma(o[2 * n], p, vv[0], vv[1]);
                tl_mma(o[2 * n + 1], p, vv[2], vv[3]);
                tl_mma(o[2 * n], lo, vv[0], vv[1]);
                tl_mma(o[2 * n + 1], lo, vv[2], vv[3]);
            }
        }
        __syncwarp();            // the stage is read before it is filled again
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
        if (tig == 0) {
            s_m[warp][g + 8 * j] = m[j];
            s_l[warp][g + 8 * j] = l[j];
        }
    }
    __syncthreads();             // statistics of all warps; and no ring is in use any more
    float* s_o = reinterpret_cast<float*>(tl_smem);      // [warp][row][HD]
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float top = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < TL_WARPS; ++w) top = fmaxf(top, s_m[w][g + 8 * j]);
        const float w = top > -CUDART_INF_F ? exp2_approx(m[j] - top) : 0.f;
        float* dst = s_o + (warp * TL_ROWS + g + 8 * j) * HD + tig * 2;
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * j] * w, o[n][2 * j + 1] * w);
    }
    __syncthreads();
    if constexpr (TAIL && HD <= 128) if (P.fused) {
        // the tail's only part: what the merge would do with it and the prefix's parts, done here
        const int rows = min(per - row0, TL_ROWS);
        const int item = owner / P.n_branches * P.n_kv + h;
        const int n = P.prefix_parts > 0 ? shared_item_parts(P, item) : 0;
        grid_wait();             // the prefix's parts are there
        if (rows <= TL_WARPS) tl_join<HD, 1>(P, s_m, s_l, s_o, n, rows, out_row0 + row0);
        else tl_join<HD, 2>(P, s_m, s_l, s_o, n, rows, out_row0 + row0);
        return;
    }
    const size_t part = (size_t)((TAIL ? P.prefix_parts : 0) + split) * P.n_rows;
    for (int i = tid; i < TL_ROWS * (HD / 4); i += 32 * TL_WARPS) {
        const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
        if (row0 + r >= n_rows || c >= P.vdim) continue;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < TL_WARPS; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(s_o + (w * TL_ROWS + r) * HD + c);
            a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
        }
        const size_t at = part + out_row(row0 + r);
        *reinterpret_cast<float4*>(P.part_o + at * P.vdim + c) = a;
        if (c == 0) {
            float top = -CUDART_INF_F, sum = 0.f;
            for (int w = 0; w < TL_WARPS; ++w) top = fmaxf(top, s_m[w][r]);
            for (int w = 0; w < TL_WARPS; ++w) sum += s_m[w][r] > -CUDART_INF_F ? s_l[w][r] * exp2_approx(s_m[w][r] - top) : s_l[w][r];
            P.part_ml[at] = make_float2(top, sum);
        }
    }
    if (TAIL) grid_wait();       // so that who waits for this waits for the prefix too
}

// A block that joins the parts of its rows itself saves a launch and its round trips, as long as its warps have no more
// than the two rows each that they join at a time (15 branches of 9 rows: 30 us that way, 25 with the merge's kernel).
bool shared_tail_joins(const SharedAttn& P) { return P.tail_parts == 1 && P.group * P.n_q <= 2 * TL_WARPS && P.dim <= 128 && P.vdim <= 128; }

static int tl_width(const SharedAttn& P) { return P.dim > 128 || P.vdim > 128 ? 256 : P.dim > 64 || P.vdim > 64 ? 128 : 64; }
// Prefixes of few rows or keys: 16 rows a block, each block row reading the keys again, start sooner than tcgen05 tiles.  8 heads
// on the device, this way and the other: 8 to 32 rows a head 300 keys 12.3 / 14.4 us, 2,000 keys 14.3..16.4 / 16.4..20.5, 9,000
// keys 20.5..22.6 / 22.5..24.6; 64 rows 2,000 keys 18.4 / 20.5, 9,000 keys 28.7 / 26.6, 32,768 keys 57 / 37.
bool shared_mma_prefers(const SharedAttn& P) {
    const long long row_blocks = ((long long)P.n_branches * P.group * P.n_q + TL_ROWS - 1) / TL_ROWS;
    return row_blocks * P.n_prompts * P.n_kv * P.prefix_len <= 1280ll * SM_COUNT;
}
// Splits of the keys: two blocks an SM (one of 256 channels), none with less than two steps of its own, and beyond 32 none with less
// than sixteen: each split is a part that the join reads.  One key head, 8 rows, at most 32 splits against this and tcgen05
// tiles: 128 channels, 65,536 keys 28.7 / 22.6 / 30.7 us, 131,072 keys 45.1 / 28.7 / 38.9; 256 channels, 131,072 keys 75.8 / 47.1.
// With eight steps instead of sixteen 131,072 keys take 32.8 (two heads 45.2, with sixteen 42.9).
int shared_mma_splits(const SharedAttn& P, bool tail) {
    const int len = tail ? P.tail_len : P.prefix_len, rows = P.group * P.n_q * (tail ? 1 : P.n_branches);
    if (len <= 0) return 0;
    const long long blocks = (long long)((rows + TL_ROWS - 1) / TL_ROWS) * P.n_prompts * (tail ? P.n_branches : 1) * P.n_kv;
    const int steps = (len + TL_STEP - 1) / TL_STEP;
    long long s = (tl_width(P) == 256 ? 1 : 2) * SM_COUNT / blocks;
    if (s > steps / 2) s = steps / 2;
    if (s > 32 && s > steps / 16) s = steps / 16 > 32 ? steps / 16 : 32;
    if (s > SA_MAX_PARTS / 2) s = SA_MAX_PARTS / 2;
    return s < 1 ? 1 : (int)s;
}

template <int HD, bool TAIL>
static int tl_launch(const SharedAttn& P, bool chained, cudaStream_t s) {
    auto kern = shared_mma_kernel<HD, TAIL>;
    const int smem = TlLayout<HD>::BYTES, rows = P.group * P.n_q * (TAIL ? 1 : P.n_branches);
    static SmemLimit limit;
    cudaError_t e = limit.raise(kern, smem);
    if (e == cudaSuccess) {
        const dim3 grid((unsigned)((rows + TL_ROWS - 1) / TL_ROWS), (unsigned)(TAIL ? P.tail_parts : P.prefix_parts),
                        (unsigned)(P.n_prompts * (TAIL ? P.n_branches : 1) * P.n_kv));
        if (chained) {
            e = launch_chained(kern, grid, dim3(32 * TL_WARPS), smem, s, P);
        } else {
            kern<<<grid, 32 * TL_WARPS, smem, s>>>(P);
            e = cudaGetLastError();
        }
    }
    if (e != cudaSuccess) {
        set_error("hira_shared_attn launch: %s", cudaGetErrorString(e));
        return HIRA_ERR_CUDA;
    }
    return HIRA_OK;
}
template <bool TAIL>
static int tl_launch_width(const SharedAttn& P, bool chained, cudaStream_t s) {
    const int w = tl_width(P);
    return w == 256 ? tl_launch<256, TAIL>(P, chained, s) : w == 128 ? tl_launch<128, TAIL>(P, chained, s) : tl_launch<64, TAIL>(P, chained, s);
}
int shared_mma_launch(const SharedAttn& P, bool tail, bool chained, cudaStream_t s) {
    return tail ? tl_launch_width<true>(P, chained, s) : tl_launch_width<false>(P, chained, s);
}

}  // namespace hira
