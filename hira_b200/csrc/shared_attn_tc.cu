// The prefix of hira_shared_attn on the tensor cores (bf16, rows of up to 128).
//
// A block takes the query rows of one (prompt, kv head) -- 128, or 256 where there are more -- through a run of key
// tiles of 128.  One warp streams the tiles in by TMA, one thread issues the products
//   S = Q K^T  (tcgen05.mma, operands in shared memory, fp32 accumulator in TMEM)
//   O += P V   (P = 2^(S - m) as two bf16 terms in TMEM, where S was; V in shared memory as it lies in memory)
// and two groups of four warps turn S into P, each thread one row: no exchange between threads for maximum and sum.
// The two groups are two independent chains, so that one group's exponentials run under the other's products:
//   256 rows: a group has 128 rows of its own, both see every tile;
//   128 rows: the groups take the tiles alternately, and their sums are joined at the end.
// The reference maximum of a row moves only when a tile exceeds it by 2^8: until then O and the sum stay as they are
// (weights up to 256 lose nothing in floating point), and O in TMEM is rescaled in rare tiles instead of each.
//
// The tiles of all items are dealt out in equal runs, one to each SM, whatever the items' number: a run may end
// inside an item and go on in the next one.  Every wait is bounded; a block whose wait ran out leaves NaN and says so in the
// status word.
//
// P takes two bf16 terms, 2^-15 of a weight between them: one alone is off by 2^-8, and the outputs' error against 64 bits
// was 0.0023 with it where rounding them costs 0.0017 (now 0.0017).  The second term is a third product on the same V.
//
// Measured, launch after launch (8 heads of 128): 16 branches x 4 heads a key head at 32,768 keys 30.7 us (134 MB: 4.4 TB/s; some
// 1.7 us before the first product and 1.6 behind the last), with one term 29.0; 64 branches at 131,072 keys 157 us (3.4 TB/s and
// 1.31 PFLOP/s, the rate that matrix products keep up under the power limit), with one term 123 (1.11 PFLOP/s of two products).
#include "shared_attn.cuh"
#include "tc_common.cuh"

#include <cuda.h>
#include <math_constants.h>

namespace hira {

constexpr int ST_KEYS = 128;                 // keys a tile
constexpr int ST_ROWS = 128;                 // query rows of a group
constexpr int ST_WG = 128;                   // threads of a softmax group
constexpr int ST_THREADS = 3 * ST_WG;        // the third group: the TMA warp, the MMA warp, two that idle
constexpr int ST_MAX_STAGES = 12;
constexpr int ST_SMEM = 227 * 1024;
// Registers: 384 threads start with 168 each; the softmax groups hold a row of 128 scores and take what the others leave
// (2 x 208 + 88 = 3 x 168).
constexpr float ST_SLACK = 8.0f;             // log2 of how far a row may rise above its reference maximum

template <int HD>
struct StLayout {
    static constexpr int BOXES = HD / 64;                       // 128-byte swizzled boxes of 64 channels
    static constexpr int BOX_BYTES = ST_KEYS * 128;
    static constexpr int TILE_BYTES = BOXES * BOX_BYTES;        // 128 rows of keys, values or queries
};
template <int HD, int NT>
constexpr int st_stages() {
    const int n = (ST_SMEM - 2048 - NT * StLayout<HD>::TILE_BYTES) / StLayout<HD>::TILE_BYTES;
    return n > ST_MAX_STAGES ? ST_MAX_STAGES : n;
}

__device__ __forceinline__ void st_tma_load(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar) : "memory");
}
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void st_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void st_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// Values as the B operand: channels one behind another in memory (N), a key a row (K).  128-byte swizzle; 64 channels a
// box, the next 64 a box further; 8 keys are 1024 bytes.
template <int HD>
__device__ __forceinline__ uint64_t st_desc_v(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3ffff) >> 4);
    d |= (uint64_t)(StLayout<HD>::BOX_BYTES >> 4) << 16;     // to the next 64 channels
    d |= (uint64_t)(1024 >> 4) << 32;                        // to the next 8 keys
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// fp32 accumulator, bf16 operands, 128 x n
constexpr uint32_t st_idesc(int n, bool b_transposed) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_transposed ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(ST_ROWS >> 4) << 24);
}
__device__ __forceinline__ void st_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
// the registers of a st_ld32 are valid behind this; they are its operands, so that no use moves ahead of it
__device__ __forceinline__ void st_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}
__device__ __forceinline__ void st_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        :: "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
           "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
           "r"(taddr) : "memory");
}
// load and wait
__device__ __forceinline__ void st_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr) : "memory");
}
// A whole warp waits, and all lanes get the same answer.  The clock is looked at only where the phase is not complete yet:
// a wait that need not wait lies on the path between two products.
__device__ __forceinline__ bool st_wait(uint32_t bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    const long long t0 = clock64();
    while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
        if (__any_sync(0xffffffffu, (unsigned long long)(clock64() - t0) > TC_WAIT_CYCLES)) return false;
    return true;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}

// One segment: a block's run of tiles inside one item.  All roles walk the same segments.
struct StSegment {
    int item, first, n;       // n tiles from `first` on that hold keys (0: none)
    int part;                 // index among the item's runs
    int len;                  // keys of the prompt
};
struct StWalk {
    long long at, end;
    __device__ __forceinline__ StWalk(const SharedAttn& P, int share) {
        const long long total = (long long)P.n_prompts * P.n_kv * P.item_tiles;
        at = share * total / P.shares;
        end = (share + 1) * total / P.shares;
    }
    __device__ __forceinline__ bool next(const SharedAttn& P, int share, StSegment& s) {
        if (at >= end) return false;
        s.item = (int)(at / P.item_tiles);
        const long long base = (long long)s.item * P.item_tiles;
        s.first = (int)(at - base);
        const int stop = (int)min(end - base, (long long)P.item_tiles);
        s.len = shared_prefix_len(P, s.item / P.n_kv);
        s.n = max(0, min(stop, (s.len + ST_KEYS - 1) / ST_KEYS) - s.first);
        s.part = share - shared_first_share(P, s.item);
        at = base + stop;
        return true;
    }
};

// where keys tile j and values tile j of a segment of n tiles lie in the order of their loads: K0 K1 V0 K2 V1 ... V(n-1),
// which is the order of their products
__device__ __forceinline__ int st_pos_k(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int st_pos_v(int j, int n) { return j == n - 1 ? 2 * n - 1 : 2 * j + 2; }

template <int HD, int NT>
__global__ void __launch_bounds__(ST_THREADS, 1)
shared_tc_kernel(const SharedAttn P, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, int row_blocks) {
    using Lay = StLayout<HD>;
    constexpr int STAGES = st_stages<HD, NT>();
    extern __shared__ unsigned char st_smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(st_smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t s_q = smem_u32(sm), s_ring = s_q + NT * Lay::TILE_BYTES;
    __shared__ __align__(8) unsigned long long s_bar[2 * ST_MAX_STAGES + 11];
    __shared__ uint32_t s_tmem;
    __shared__ int s_fail;
    const uint32_t bars = smem_u32(s_bar);
    const uint32_t bar_full = bars, bar_empty = bars + 8 * ST_MAX_STAGES;      // [STAGES] tile landed, tile used up
    const uint32_t bar_q = bars + 16 * ST_MAX_STAGES;                            // the segment's queries are in place
    const uint32_t bar_done = bar_q + 8;                                         // all products of the segment are complete
    const uint32_t bar_s = bar_q + 16, bar_p = bar_q + 32, bar_o = bar_q + 48;   // [2] S written, P written, O complete
    const uint32_t bar_pa = bar_q + 64, bar_exit = bar_q + 80;                   // [2] the first half of P written

    const int tid = threadIdx.x, warp = tid >> 5;
    const int rb = blockIdx.x % row_blocks, share = blockIdx.x / row_blocks;
    if (tid == 0) {
        s_fail = 0;
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(bar_full + 8 * i, 1);
            mbar_init(bar_empty + 8 * i, 1);
        }
        mbar_init(bar_q, 2 * ST_WG);
        mbar_init(bar_done, 1);
        mbar_init(bar_exit, 1);
        for (int w = 0; w < 2; ++w) {
            mbar_init(bar_s + 8 * w, 1);
            mbar_init(bar_p + 8 * w, ST_WG);
            mbar_init(bar_pa + 8 * w, ST_WG);
            mbar_init(bar_o + 8 * w, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s_tmem);
    volatile int* fail = &s_fail;
    const uint32_t tm_s = tmem, tm_o = tmem + 2 * ST_KEYS;      // S and P of the chains, then O of the chains
    grid_trigger();      // what follows on the stream reads nothing of this before it waits

    StWalk walk(P, share);
    StSegment seg;
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8) {
            // ---- tiles in, in the order of their products ---------------------------------------------------
            if ((tid & 31) == 0) {
                uint32_t pos = 0;
                auto load = [&](const CUtensorMap* map, int tile, const StSegment& s) {
                    const uint32_t stage = pos % STAGES, round = pos / STAGES;
                    if (round > 0 && (!mbar_wait(bar_empty + 8 * stage, (round - 1) & 1))) return false;
                    const uint32_t bar = bar_full + 8 * stage, dst = s_ring + stage * Lay::TILE_BYTES;
                    mbar_expect_tx(bar, Lay::TILE_BYTES);
    #pragma unroll
                    for (int b = 0; b < Lay::BOXES; ++b)
                        st_tma_load(dst + b * Lay::BOX_BYTES, map, b * 64, tile * ST_KEYS, s.item % P.n_kv, s.item / P.n_kv, bar);
                    ++pos;
                    return true;
                };
                bool ok = true;
                while (ok && walk.next(P, share, seg)) {
                    if (seg.n == 0) continue;
                    ok = load(&map_k, seg.first, seg);
                    for (int j = 0; ok && j < seg.n; ++j) {
                        if (j + 1 < seg.n) ok = load(&map_k, seg.first + j + 1, seg);
                        ok = ok && load(&map_v, seg.first + j, seg);
                    }
                }
                if (!ok) *fail = 1;
                // No copy may be in flight when the shared memory is given back, and who waits for a tile may give up after the
                // last one is asked for: the tiles that the ring still holds are waited for here, whatever became of the others.
                // (Where all went well the products of the last one come after this, so it costs nothing.)
                for (uint32_t p = pos > STAGES ? pos - STAGES : 0; p < pos; ++p) mbar_wait(bar_full + 8 * (p % STAGES), (p / STAGES) & 1);
            }
        } else if (warp == 9) {
            // ---- products ------------------------------------------------------------------------------------
            // The whole warp walks the loop, so that everything the instructions take is known to be the same in all
            // lanes and lies in uniform registers; one lane issues.  (With one lane walking, each product waited some
            // 120 cycles for its operands, twice the 64 that it takes.)
            uint32_t leader;
            asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
            uint32_t base = 0, segs = 0, n_p[2] = {0, 0};      // loads, segments and P tiles so far
            bool ok = true;
            while (ok && walk.next(P, share, seg)) {
                const int n = seg.n;
                if (n == 0) continue;
                ok = st_wait(bar_q, segs & 1);
                const int count[2] = {NT == 2 ? n : (n + 1) / 2, NT == 2 ? n : n / 2};
                auto tile_of = [&](int w, int i) { return NT == 2 ? i : 2 * i + w; };
                auto full = [&](uint32_t pos) { return st_wait(bar_full + 8 * (pos % STAGES), (pos / STAGES) & 1); };
                auto qk = [&](int w, uint32_t pos) {
                    const uint32_t stage = pos % STAGES, a0 = s_q + (NT == 2 ? w : 0) * Lay::TILE_BYTES, b0 = s_ring + stage * Lay::TILE_BYTES;
                    if (leader) {
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k) {
                            const uint32_t off = (k >> 2) * Lay::BOX_BYTES + (k & 3) * 32;
                            st_mma_ss(tm_s + w * ST_KEYS, umma_desc(a0 + off), umma_desc(b0 + off), st_idesc(ST_KEYS, false), k > 0);
                        }
                        umma_commit(bar_s + 8 * w);
                        if (NT == 1 || w == 1) umma_commit(bar_empty + 8 * stage);
                    }
                };
                // 16 keys' part of P V: the weights' first terms, then their second ones
                auto pv = [&](int w, int k, uint32_t b0, bool accumulate) {
                    const uint32_t p = tm_s + w * ST_KEYS + k * 8;
                    const uint64_t v = st_desc_v<HD>(b0 + k * 2048);
                    st_mma_ts(tm_o + w * HD, p, v, st_idesc(HD, true), accumulate);
                    st_mma_ts(tm_o + w * HD, p + ST_KEYS / 2, v, st_idesc(HD, true), 1);
                };
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    if (ok && count[w] > 0) {
                        const uint32_t pos = base + st_pos_k(tile_of(w, 0));
                        ok = full(pos);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (ok) qk(w, pos);
                    }
                for (int i = 0; ok && i < count[0]; ++i)
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        if (!ok || i >= count[w]) continue;
                        // P V of tile i (its first half as soon as that half of P is there) and Q K of the chain's next, back
                        // to back: the second is behind the first in the pipe, so it may write S where P was.  The tiles are
                        // waited for first, P last.
                        const bool more = i + 1 < count[w];
                        const uint32_t pos_k = base + st_pos_k(tile_of(w, more ? i + 1 : i)), pos_v = base + st_pos_v(tile_of(w, i), n);
                        const uint32_t stage = pos_v % STAGES, b0 = s_ring + stage * Lay::TILE_BYTES;
                        ok = full(pos_v) && (!more || full(pos_k)) && st_wait(bar_pa + 8 * w, n_p[w] & 1);
                        if (!ok) continue;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (leader) {
#pragma unroll
                            for (int k = 0; k < ST_KEYS / 32; ++k) pv(w, k, b0, i > 0 || k > 0);
                        }
                        ok = st_wait(bar_p + 8 * w, n_p[w] & 1);
                        if (!ok) continue;
                        ++n_p[w];
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (leader) {
#pragma unroll
                            for (int k = ST_KEYS / 32; k < ST_KEYS / 16; ++k) pv(w, k, b0, i > 0 || k > 0);
                            if (NT == 1 || w == 1) umma_commit(bar_empty + 8 * stage);
                            if (!more) umma_commit(bar_o + 8 * w);
                        }
                        if (more) qk(w, pos_k);
                    }
                if (ok && leader) umma_commit(bar_done);
                base += 2 * n;
                ++segs;
            }
            // nothing of the tensor cores may be under way when shared memory and TMEM are given back
            if (!ok) {
                *fail = 1;
                if (leader) umma_commit(bar_exit);
                mbar_wait(bar_exit, 0);
            } else if (segs > 0) {
                mbar_wait(bar_done, (segs - 1) & 1);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- softmax: thread t of group w has row t of its chain (TMEM lane t) -----------------------------
        const int w = warp >> 2, t = tid & (ST_WG - 1);
        const int per = P.group * P.n_q, n_rows = P.n_branches * per;
        const int row0 = (rb * NT + (NT == 2 ? w : 0)) * ST_ROWS;       // first row of the chain
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t my_s = tm_s + w * ST_KEYS + lanes, my_o = tm_o + w * HD + lanes;
        const bool warp_used = row0 + (warp & 3) * 32 < n_rows;          // rows behind the last: nothing to compute
        const int row = row0 + t;
        const float scale = fmaxf(fabsf(P.scale_log2), 1.2e-38f);        // never 0, which a masked score's -inf would turn into NaN
        const uint32_t flip = P.scale_log2 < 0.f ? 0x80008000u : 0u;     // a negative scale turns the queries round
        uint32_t base = 0, segs = 0, n_s = 0, n_o[2] = {0, 0};
        bool ok = true;
        while (walk.next(P, share, seg)) {
            const int prompt = seg.item / P.n_kv, h = seg.item % P.n_kv, n = seg.n;
            const int count = NT == 2 ? n : (n + 1 - w) / 2;
            float m = -CUDART_INF_F, l = 0.f;
            if (n > 0 && ok) {
                // queries into the swizzled layout of the products; the products of the segment before have read theirs
                if (segs > 0) ok = st_wait(bar_done, (segs - 1) & 1);
                // a thread takes a row (or half of one), all of it on its way at once
                constexpr int CHUNKS = HD / 8 / (NT == 2 ? 1 : 2);
                const int c0 = NT == 2 ? 0 : w * CHUNKS, have = row < n_rows ? P.dim / 8 : 0;
                uint4 x[CHUNKS];
                const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(P.q) +
                                                                  (have ? shared_row_offset(P, shared_row(P, prompt, h, row), P.qs) : 0));
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) x[c] = c0 + c < have ? src[c0 + c] : make_uint4(0, 0, 0, 0);
                unsigned char* dst = sm + (NT == 2 ? w : 0) * Lay::TILE_BYTES + t * 128;
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c)
                    *reinterpret_cast<uint4*>(dst + ((c0 + c) >> 3) * Lay::BOX_BYTES + ((((c0 + c) & 7) ^ (t & 7)) << 4)) =
                        make_uint4(x[c].x ^ flip, x[c].y ^ flip, x[c].z ^ flip, x[c].w ^ flip);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(bar_q);
                for (int i = 0; i < count && ok; ++i) {
                    const int j = NT == 2 ? i : 2 * i + w, k0 = (seg.first + j) * ST_KEYS;
                    ok = st_wait(bar_s + 8 * w, n_s & 1);
                    if (!ok) break;
                    ++n_s;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const int valid = min(seg.len - k0, ST_KEYS);
                    if (k0 + valid < min(P.prefix_len, k0 + ST_KEYS)) {
                        // rows of the value tile behind the prompt's keys, whatever they hold: 0, as what TMA fills in
                        // behind the array (0 x NaN would be NaN)
                        const uint32_t pos = base + st_pos_v(j, n), stage = pos % STAGES;
                        ok = st_wait(bar_full + 8 * stage, (pos / STAGES) & 1);
                        unsigned char* v = sm + (NT + stage) * Lay::TILE_BYTES;
                        for (int q = valid * 8 + t; q < ST_KEYS * 8; q += ST_WG)
#pragma unroll
                            for (int b = 0; b < Lay::BOXES; ++b) *reinterpret_cast<uint4*>(v + b * Lay::BOX_BYTES + q * 16) = make_uint4(0, 0, 0, 0);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    if (warp_used) {
                        uint32_t s[4][32];
#pragma unroll
                        for (int q = 0; q < 4; ++q) st_ld32(my_s + q * 32, s[q]);
#pragma unroll
                        for (int q = 0; q < 4; ++q) st_ld_wait(s[q]);
                        if (valid < ST_KEYS) {
#pragma unroll
                            for (int q = 0; q < 4; ++q)
#pragma unroll
                                for (int e = 0; e < 32; ++e)
                                    if (q * 32 + e >= valid) s[q][e] = 0xff800000u;      // -inf
                        }
                        float mx[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            mx[q] = __uint_as_float(s[q][0]);
#pragma unroll
                            for (int e = 1; e < 31; e += 2) mx[q] = max3f(mx[q], __uint_as_float(s[q][e]), __uint_as_float(s[q][e + 1]));
                            mx[q] = fmaxf(mx[q], __uint_as_float(s[q][31]));
                        }
                        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
                        const bool rise = top > m + ST_SLACK;      // from -inf on: always, unless the tile is -inf too
                        if (__any_sync(0xffffffffu, rise)) {
                            const float to = rise ? top : m;
                            const float f = rise ? exp2_approx(m - top) : 1.f;      // 0 from -inf on
                            m = to;
                            l *= f;
                            if (i > 0) {
                                // the product before last is complete: S of this tile was committed behind it
                                uint32_t o[16];
#pragma unroll 1
                                for (int c = 0; c < HD; c += 16) {
                                    st_ld16(my_o + c, o);
#pragma unroll
                                    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                    st_st16(my_o + c, o);
                                }
                            }
                        }
                        const float nm = m > -CUDART_INF_F ? -m : 0.f;
                        const float2 sc2 = make_float2(scale, scale), nm2 = make_float2(nm, nm);
                        float2 sum2 = make_float2(0.f, 0.f);
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            uint32_t hi[16], lo[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float2 y = __ffma2_rn(make_float2(__uint_as_float(s[q][2 * e]), __uint_as_float(s[q][2 * e + 1])), sc2, nm2);
                                const float2 z = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                                sum2 = __fadd2_rn(sum2, z);
                                // the upper 16 bits of each are its first term, what that leaves (exact in fp32) rounded its second
                                const uint32_t a = __float_as_uint(z.x), b = __float_as_uint(z.y);
                                hi[e] = __byte_perm(a, b, 0x7632);
                                const float2 rest = __ffma2_rn(make_float2(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u)),
                                                               make_float2(-1.f, -1.f), z);
                                lo[e] = pack_bf16(rest.x, rest.y);
                            }
                            st_st16(my_s + q * 16, hi);
                            st_st16(my_s + ST_KEYS / 2 + q * 16, lo);
                            if (q == 1) {
                                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                                mbar_arrive(bar_pa + 8 * w);
                            }
                        }
                        l += sum2.x + sum2.y;
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    } else {
                        mbar_arrive(bar_pa + 8 * w);
                    }
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    mbar_arrive(bar_p + 8 * w);
                }
#pragma unroll
                for (int v = 0; v < 2; ++v)
                    if (NT == 2 ? v == w : n > v) {      // the chains whose sums this group is going to read
                        ok = ok && st_wait(bar_o + 8 * v, n_o[v] & 1);
                        ++n_o[v];
                    }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                base += 2 * n;
                ++segs;
            }
            if (!ok) *fail = 1;
            // What the run adds to its rows.  Chains with rows of their own leave them as they are; two chains over the same rows
            // are joined here, each group writing half of the channels.
            const bool mine = warp_used && row < n_rows;
            const size_t at = (size_t)seg.part * P.n_rows + (mine ? shared_row(P, prompt, h, row) : 0);
            float f[2] = {1.f, 1.f};       // factors of the chains' sums
            if (NT == 1) {
                float2* s_ml = reinterpret_cast<float2*>(sm);      // in the queries' place: the products have read them
                s_ml[tid] = ok ? make_float2(m, l) : make_float2(CUDART_NAN_F, CUDART_NAN_F);
                asm volatile("bar.sync 1, %0;" ::"n"(2 * ST_WG) : "memory");
                const float2 c0 = s_ml[t], c1 = s_ml[ST_WG + t];
                m = fmaxf(c0.x, c1.x);
                const float base_m = m > -CUDART_INF_F ? m : 0.f;
                f[0] = c0.x > -CUDART_INF_F ? exp2_approx(c0.x - base_m) : 0.f;
                f[1] = c1.x > -CUDART_INF_F ? exp2_approx(c1.x - base_m) : 0.f;
                // (a sum is NaN without a maximum where all logits were; a maximum is where a wait ran out)
                l = (c0.x > -CUDART_INF_F ? f[0] * c0.y : c0.y) + (c1.x > -CUDART_INF_F ? f[1] * c1.y : c1.y);
                if (c0.x != c0.x || c1.x != c1.x) m = CUDART_NAN_F;
            } else if (!ok) {
                m = CUDART_NAN_F;
            }
            if (mine && (NT == 2 || w == 0)) P.part_ml[at] = make_float2(m, l);
            if (warp_used && n > 0 && ok) {
                const int chains = NT == 2 || n < 2 ? 1 : 2, from = NT == 2 ? 0 : w * (HD / 2);
                uint32_t o[16], o1[16];
#pragma unroll 1
                for (int c = from; c < from + (NT == 2 ? HD : HD / 2); c += 16) {
                    st_ld16(tm_o + (NT == 2 ? w * HD : 0) + lanes + c, o);
                    if (NT == 1) {
                        if (chains == 2) st_ld16(tm_o + HD + lanes + c, o1);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float y = __uint_as_float(o[e]) * f[0];
                            if (chains == 2) y = __fmaf_rn(__uint_as_float(o1[e]), f[1], y);
                            o[e] = __float_as_uint(y);
                        }
                    }
                    if (mine)
#pragma unroll
                        for (int e = 0; e < 16; e += 4)
                            if (c + e < P.vdim)
                                *reinterpret_cast<float4*>(P.part_o + at * P.vdim + c + e) =
                                    make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                }
            }
            if (NT == 1) {      // the other group's sums and statistics are read before they are written again
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                asm volatile("bar.sync 1, %0;" ::"n"(2 * ST_WG) : "memory");
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (tid == 0 && *fail && P.status) atomicOr(P.status, HIRA_STATUS_ATTN_FAILED);
    if (warp == 9) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

typedef CUresult (*StEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static StEncodeFn st_encode_fn() {
    static const StEncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess
                   ? reinterpret_cast<StEncodeFn>(p) : nullptr;
    }();
    return fn;
}
// (prompts, heads, rows, width) bf16 with the given strides; boxes of 64 channels x 128 rows
static bool st_make_map(CUtensorMap* map, const void* base, int width, const SharedAttn& P, const long long (&s)[3]) {
    const StEncodeFn fn = st_encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)width, (cuuint64_t)P.prefix_len, (cuuint64_t)P.n_kv, (cuuint64_t)P.n_prompts};
    // a stride along a dimension of one is not used, but has to be one that the encoder takes
    const cuuint64_t row = (cuuint64_t)(P.prefix_len > 1 ? s[2] : width) * 2;
    const cuuint64_t strides[3] = {row, P.n_kv > 1 ? (cuuint64_t)s[1] * 2 : row, P.n_prompts > 1 ? (cuuint64_t)s[0] * 2 : row};
    const cuuint32_t box[4] = {64, (cuuint32_t)ST_KEYS, 1, 1}, one[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Strides that a tensor map takes: forward, rows that do not overlap, and below 2^40 bytes.
bool shared_tc_supported(const SharedAttn& P) {
    if (P.prefix_len == 0 || P.dim > 128 || P.vdim > 128 || (P.dim > 64) != (P.vdim > 64)) return false;
    const int n[3] = {P.n_prompts, P.n_kv, P.prefix_len};
    for (int i = 0; i < 3; ++i)
        if (n[i] > 1 && (P.pks[i] < 1 || P.pvs[i] < 1 || P.pks[i] >= (1ll << 39) || P.pvs[i] >= (1ll << 39))) return false;
    return P.prefix_len == 1 || (P.pks[2] >= P.dim && P.pvs[2] >= P.vdim);
}

void shared_tc_plan(SharedAttn& P) {
    const int rows = P.n_branches * P.group * P.n_q, nt = rows > ST_ROWS ? 2 : 1, row_blocks = (rows + nt * ST_ROWS - 1) / (nt * ST_ROWS);
    P.item_tiles = (P.prefix_len + ST_KEYS - 1) / ST_KEYS;
    const long long total = (long long)P.n_prompts * P.n_kv * P.item_tiles;
    const long long items = (long long)P.n_prompts * P.n_kv;
    long long shares = SM_COUNT / row_blocks;
    if (shares < 1) shares = 1;
    // A run that goes on in a second item pays for filling and draining the pipe again, about four tiles' time (64
    // branches of 8 heads at 131,072 keys: such blocks ended 12 us behind the others' 128).  Runs that end with their
    // items are taken where they cost no more than that.
    if (items <= shares) {
        const long long each = shares / items;
        if ((P.item_tiles + each - 1) / each <= (total + shares - 1) / shares + 4) shares = each * items;
    }
    if (shares > total) shares = total;
    P.shares = (int)shares;
    // an item of T tiles spans at most this many runs of total / shares tiles
    const long long run = total / P.shares;
    long long runs = (P.item_tiles + run - 1) / run + 1;
    if (runs > P.shares) runs = P.shares;
    P.prefix_parts = (int)runs;
}

template <int HD, int NT>
static int st_launch(const SharedAttn& P, int row_blocks, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t s) {
    auto kern = shared_tc_kernel<HD, NT>;
    const size_t smem = (size_t)(NT + st_stages<HD, NT>()) * StLayout<HD>::TILE_BYTES + 1024;
    static SmemLimit limit;
    const cudaError_t e = limit.raise(kern, (int)smem);
    if (e != cudaSuccess) {
        set_error("hira_shared_attn: cudaFuncSetAttribute(%zu B smem): %s", smem, cudaGetErrorString(e));
        return HIRA_ERR_CUDA;
    }
    kern<<<(unsigned)(P.shares * row_blocks), ST_THREADS, smem, s>>>(P, mk, mv, row_blocks);
    HIRA_CHECK_LAUNCH("hira_shared_attn launch");
    return HIRA_OK;
}

int shared_tc_launch(const SharedAttn& P, cudaStream_t s) {
    CUtensorMap mk, mv;
    if (!st_make_map(&mk, P.pk, P.dim, P, P.pks) || !st_make_map(&mv, P.pv, P.vdim, P, P.pvs)) {
        set_error("hira_shared_attn: cuTensorMapEncodeTiled failed or is unavailable");
        return HIRA_ERR_CUDA;
    }
    const int rows = P.n_branches * P.group * P.n_q, nt = rows > ST_ROWS ? 2 : 1, row_blocks = (rows + nt * ST_ROWS - 1) / (nt * ST_ROWS);
    const bool wide = P.dim > 64;
    if (nt == 1) return wide ? st_launch<128, 1>(P, row_blocks, mk, mv, s) : st_launch<64, 1>(P, row_blocks, mk, mv, s);
    return wide ? st_launch<128, 2>(P, row_blocks, mk, mv, s) : st_launch<64, 2>(P, row_blocks, mk, mv, s);
}

}  // namespace hira
