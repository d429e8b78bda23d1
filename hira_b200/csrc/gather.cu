// Sequences of a cache forked, reordered or compacted: out[j] = in[index[j]] for every array of it, in one launch.
//
// An array holds, for each sequence, n_seg parts (heads) of which only the first `bytes` are in use.  Nothing is
// computed; the floor is reading each picked sequence once and writing each changed one, and only what is in use.
//
// A block takes a strip of columns -- the same bytes of a head's part -- of ALL sequences at once:
//   * into other memory, a thread loads its column of a sequence once and stores it for every sequence that picks it;
//   * in place, the strip of every sequence that changes is staged in shared memory before the first is overwritten, so
//     any index is right (cycles, one sequence picked many times) without a second copy of the cache; sequences that
//     pick themselves are neither read nor written.  Where no changed sequence is another's source, nothing is staged.
//
// Bound by memory.  One sequence of an index of 8 heads, 32,768 keys of 128 bf16 in room for 40,000, forked into 8 (1.9 GB with
// the int8 copy and the cleared room): 322 us, 5.9 TB/s.  In place, two of 8 sequences of 16,384 keys replaced (340 MB): 64 us,
// 5.3 TB/s, nothing staged.  Staged, which any changed sequence that another picks asks for: two of the 8 swapped 99 us, permuted (6
// changed) 276, all 8 rotated 381, 3.4 to 3.7 TB/s: a strip's loads, a barrier, its stores and another barrier, with only the SM's
// other blocks in flight meanwhile.  Tails of 100 tokens, 4 of 8 replaced: 7 us, the launch and two round trips; rotated 28.
#include "common.cuh"

namespace hira {

constexpr int GA_THREADS = 256;
constexpr int GA_ITEMS = 24;              // arrays a launch takes
constexpr int GA_STAGE_BYTES = 48 * 1024; // staged strips of a block; 64 bytes a sequence where that is more
constexpr int GA_MAX_SEQ = 2048;

struct GatherItems {
    hira_gather_item_t it[GA_ITEMS];
    long long first[GA_ITEMS + 1];        // first strip of each array
    int wide[GA_ITEMS];                   // 16-byte columns (4-byte ones where a part starts or ends between)
    int n;
};

template <typename W>
__device__ __forceinline__ W gather_fill(uint32_t f);
template <> __device__ __forceinline__ uint4 gather_fill<uint4>(uint32_t f) { return make_uint4(f, f, f, f); }
template <> __device__ __forceinline__ uint32_t gather_fill<uint32_t>(uint32_t f) { return f; }

// strip `strip` of one array into other memory: 4 columns a thread
constexpr int GA_COLS = 4;
template <typename W>
__device__ __forceinline__ void gather_strip(const hira_gather_item_t& g, long long strip, const int* s_idx, int n_dst) {
    const long long strips = (g.bytes_filled + GA_THREADS * GA_COLS * (long long)sizeof(W) - 1) / (GA_THREADS * GA_COLS * (long long)sizeof(W));
    const long long seg = strip / strips, col0 = (strip - seg * strips) * GA_THREADS * GA_COLS + threadIdx.x;
    const long long used = g.bytes / sizeof(W), total = g.bytes_filled / sizeof(W);
    const char* src = reinterpret_cast<const char*>(g.src) + seg * g.src_seg_stride;
    char* dst = reinterpret_cast<char*>(g.dst) + seg * g.dst_seg_stride;
    W v[GA_COLS];
    int have = -2;      // the sequence whose columns v holds
    for (int j = 0; j < n_dst; ++j) {
        const int from = s_idx[j];
        if (from != have) {
            have = from;
#pragma unroll
            for (int c = 0; c < GA_COLS; ++c) {
                const long long col = col0 + c * GA_THREADS;
                v[c] = from >= 0 && col < used ? reinterpret_cast<const W*>(src + from * g.src_seq_stride)[col] : gather_fill<W>(g.fill);
            }
        }
#pragma unroll
        for (int c = 0; c < GA_COLS; ++c) {
            const long long col = col0 + c * GA_THREADS;
            if (col < total) reinterpret_cast<W*>(dst + j * g.dst_seq_stride)[col] = v[c];
        }
    }
}

__global__ void __launch_bounds__(GA_THREADS)
gather_kernel(const __grid_constant__ GatherItems items, const long long* __restrict__ index, int n_src, int n_dst,
              const int32_t* __restrict__ status_from, int32_t* status) {
    __shared__ int s_idx[GA_MAX_SEQ];
    int bad = 0;
    for (int j = threadIdx.x; j < n_dst; j += GA_THREADS) {
        const long long i = index[j];
        const bool ok = i >= 0 && i < n_src;
        bad |= !ok;
        s_idx[j] = ok ? (int)i : -1;      // a sequence that is not there: left empty
    }
    bad = __syncthreads_or(bad);
    if (status && blockIdx.x == 0 && threadIdx.x == 0) {
        const int now = bad ? HIRA_STATUS_BAD_INDEX : 0;
        if (status_from) *status = *status_from | now;
        else if (now) atomicOr(status, now);
    }
    for (long long strip = blockIdx.x; strip < items.first[items.n]; strip += gridDim.x) {
        int a = 0;
        while (strip >= items.first[a + 1]) ++a;
        if (items.wide[a]) gather_strip<uint4>(items.it[a], strip - items.first[a], s_idx, n_dst);
        else gather_strip<uint32_t>(items.it[a], strip - items.first[a], s_idx, n_dst);
    }
}

// In place, `cols` columns of the m sequences that change.
//   staged: all read before the first is written;
//   direct (no changed sequence is another's source): copied right away, a source that follows itself read once.
template <typename W, bool STAGED>
__device__ __forceinline__ void permute_strip(const hira_gather_item_t& g, long long strip, const int* s_dst, const int* s_src, int moved,
                                              int cols, W* s_stage) {
    const long long used = g.bytes / sizeof(W), strips = (used + cols - 1) / cols;
    const long long seg = strip / strips, col0 = (strip - seg * strips) * cols;
    char* base = reinterpret_cast<char*>(g.dst) + seg * g.dst_seg_stride;
    if (STAGED) {
        const int n = moved * cols;
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += GA_THREADS) {
            const int k = i / cols;
            const long long col = col0 + (i - k * cols);
            if (col < used) s_stage[i] = reinterpret_cast<const W*>(base + s_src[k] * g.dst_seq_stride)[col];
        }
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < n; i += GA_THREADS) {
            const int k = i / cols;
            const long long col = col0 + (i - k * cols);
            if (col < used) reinterpret_cast<W*>(base + s_dst[k] * g.dst_seq_stride)[col] = s_stage[i];
        }
        __syncthreads();
    } else {
        W v[GA_COLS];
        int have = -1;
        for (int k = 0; k < moved; ++k) {
            if (s_src[k] != have) {
                have = s_src[k];
#pragma unroll
                for (int c = 0; c < GA_COLS; ++c) {
                    const long long col = col0 + threadIdx.x + c * GA_THREADS;
                    if (col < used) v[c] = reinterpret_cast<const W*>(base + have * g.dst_seq_stride)[col];
                }
            }
#pragma unroll
            for (int c = 0; c < GA_COLS; ++c) {
                const long long col = col0 + threadIdx.x + c * GA_THREADS;
                if (col < used) reinterpret_cast<W*>(base + s_dst[k] * g.dst_seq_stride)[col] = v[c];
            }
        }
    }
}

// The strips' width follows from how many sequences change, which only the device knows; so the strips are counted here.
__global__ void __launch_bounds__(GA_THREADS)
permute_kernel(const __grid_constant__ GatherItems items, const long long* __restrict__ index, int n_seq, int stage_bytes, int32_t* status) {
    extern __shared__ __align__(16) unsigned char ga_stage[];
    __shared__ int s_dst[GA_MAX_SEQ], s_src[GA_MAX_SEQ];
    __shared__ unsigned char s_moves[GA_MAX_SEQ];
    __shared__ long long s_first[GA_ITEMS + 1];
    __shared__ int s_n, s_hazard;
    const int tid = threadIdx.x;
    if (tid == 0) s_n = s_hazard = 0;
    for (int j = tid; j < n_seq; j += GA_THREADS) {
        const long long i = index[j];
        const bool ok = i >= 0 && i < n_seq;
        if (!ok && status && blockIdx.x == 0) atomicOr(status, HIRA_STATUS_BAD_INDEX);      // left as it was
        s_src[j] = ok ? (int)i : j;
        s_moves[j] = ok && i != j;
    }
    __syncthreads();
    // the list of those that change, packed by the first warp in their order
    for (int j = tid; j < n_seq; j += GA_THREADS)
        if (s_moves[j] && s_moves[s_src[j]]) s_hazard = 1;
    __syncthreads();
    if (tid < 32) {
        int n = 0;
        for (int j0 = 0; j0 < n_seq; j0 += 32) {
            const int j = j0 + tid, src = j < n_seq ? s_src[j] : 0;
            const unsigned m = __ballot_sync(0xffffffffu, j < n_seq && s_moves[j]);
            __syncwarp();
            if (m >> tid & 1) {       // never ahead of what is still to be read: n + rank <= j
                const int k = n + __popc(m & ((1u << tid) - 1));
                s_dst[k] = j;
                s_src[k] = src;
            }
            n += __popc(m);
            __syncwarp();
        }
        if (tid == 0) s_n = n;
    }
    __syncthreads();
    const int moved = s_n;
    if (moved == 0) return;
    const bool staged = s_hazard != 0;
    int cols = GA_THREADS * GA_COLS;
    if (staged) {
        cols = stage_bytes / 16 / moved;
        if (cols > GA_THREADS) cols = cols / GA_THREADS * GA_THREADS;
    }
    if (tid == 0) {
        long long n = 0;
        for (int a = 0; a < items.n; ++a) {
            s_first[a] = n;
            const long long words = items.it[a].bytes / (items.wide[a] ? 16 : 4);
            n += (words + cols - 1) / cols * items.it[a].n_seg;
        }
        s_first[items.n] = n;
    }
    __syncthreads();
    for (long long strip = blockIdx.x; strip < s_first[items.n]; strip += gridDim.x) {
        int a = 0;
        while (strip >= s_first[a + 1]) ++a;
        const long long at = strip - s_first[a];
        uint4* s16 = reinterpret_cast<uint4*>(ga_stage);
        uint32_t* s4 = reinterpret_cast<uint32_t*>(ga_stage);
        if (items.wide[a]) {
            if (staged) permute_strip<uint4, true>(items.it[a], at, s_dst, s_src, moved, cols, s16);
            else permute_strip<uint4, false>(items.it[a], at, s_dst, s_src, moved, cols, s16);
        } else {
            if (staged) permute_strip<uint32_t, true>(items.it[a], at, s_dst, s_src, moved, cols, s4);
            else permute_strip<uint32_t, false>(items.it[a], at, s_dst, s_src, moved, cols, s4);
        }
    }
}

}  // namespace hira

using namespace hira;

static int run_gather(const hira_gather_item_t* items, int32_t n_items, const int64_t* index, int32_t n_src, int32_t n_dst,
                      int32_t in_place, const int32_t* status_from, int32_t* status, void* stream) {
    HIRA_CHECK_ARG(items && index, HIRA_ERR_ARG, "hira_gather: items and index must not be NULL");
    HIRA_CHECK_ARG(n_items >= 0 && n_items <= GA_ITEMS, HIRA_ERR_SHAPE, "hira_gather: %d arrays outside 0..%d", n_items, GA_ITEMS);
    HIRA_CHECK_ARG(n_src >= 1 && n_dst >= 1 && n_src <= GA_MAX_SEQ && n_dst <= GA_MAX_SEQ, HIRA_ERR_SHAPE,
                   "hira_gather: %d sequences picked from %d, 1..%d are served", n_dst, n_src, GA_MAX_SEQ);
    HIRA_CHECK_ARG(!in_place || n_src == n_dst, HIRA_ERR_SHAPE, "hira_gather: in place %d sequences cannot become %d", n_src, n_dst);
    GatherItems G = {};
    for (int i = 0; i < n_items; ++i) {
        const hira_gather_item_t& g = items[i];
        HIRA_CHECK_ARG(g.n_seg >= 0 && g.bytes >= 0 && g.bytes_filled >= g.bytes, HIRA_ERR_SHAPE,
                       "hira_gather: array %d has n_seg=%d bytes=%lld bytes_filled=%lld", i, g.n_seg, (long long)g.bytes,
                       (long long)g.bytes_filled);
        const long long span = in_place ? g.bytes : g.bytes_filled;
        if (g.n_seg == 0 || span == 0) continue;
        HIRA_CHECK_ARG(g.dst && (in_place ? g.src == g.dst && g.src_seq_stride == g.dst_seq_stride && g.src_seg_stride == g.dst_seg_stride
                                          : g.src && g.src != g.dst),
                       HIRA_ERR_ARG, "hira_gather: array %d is NULL, or source and destination do not fit in_place=%d", i, in_place);
        const uintptr_t mix = (uintptr_t)g.src | (uintptr_t)g.dst | (uintptr_t)g.src_seq_stride | (uintptr_t)g.dst_seq_stride |
                              (uintptr_t)g.src_seg_stride | (uintptr_t)g.dst_seg_stride | (uintptr_t)g.bytes | (uintptr_t)g.bytes_filled;
        HIRA_CHECK_ARG((mix & 3) == 0, HIRA_ERR_ARG, "hira_gather: array %d is not made of 4-byte words", i);
        G.it[G.n] = g;
        G.wide[G.n] = (mix & 15) == 0;
        const long long word = G.wide[G.n] ? 16 : 4, strip = word * GA_THREADS * GA_COLS;
        G.first[G.n + 1] = G.first[G.n] + (span + strip - 1) / strip * g.n_seg;
        ++G.n;
    }
    if (G.n == 0) return HIRA_OK;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const long long strips = G.first[G.n];
    const long long* idx = reinterpret_cast<const long long*>(index);
    if (in_place) {
        const int smem = n_dst * 64 > GA_STAGE_BYTES ? n_dst * 64 : GA_STAGE_BYTES;
        static SmemLimit limit;
        const cudaError_t e = limit.raise(permute_kernel, smem);
        if (e != cudaSuccess) {
            set_error("hira_gather: cudaFuncSetAttribute(%d B smem): %s", smem, cudaGetErrorString(e));
            return HIRA_ERR_CUDA;
        }
        // strips of the direct copy; staged ones are more
        const long long blocks = strips < 3 * SM_COUNT ? strips : 3 * SM_COUNT;
        permute_kernel<<<(unsigned)blocks, GA_THREADS, smem, s>>>(G, idx, n_dst, smem, status);
    } else {
        const long long blocks = strips < 8 * SM_COUNT ? strips : 8 * SM_COUNT;
        gather_kernel<<<(unsigned)blocks, GA_THREADS, 0, s>>>(G, idx, n_src, n_dst, status_from, status);
    }
    HIRA_CHECK_LAUNCH("hira_gather launch");
    return HIRA_OK;
}

extern "C" int hira_gather(const hira_gather_item_t* items, int32_t n_items, const int64_t* index, int32_t n_src, int32_t n_dst,
                           int32_t in_place, int32_t* status, void* stream) {
    return run_gather(items, n_items, index, n_src, n_dst, in_place, nullptr, status, stream);
}

extern "C" int hira_gather_index(const hira_index_t* from, const hira_index_t* to, int32_t n_src, int32_t n_dst, const int64_t* index,
                                 void* samples, int64_t sample_bytes, const int32_t* status_from, int32_t* status, void* stream) {
    int rc = validate_index(from, false);
    if (rc == HIRA_OK) rc = validate_index(to, false);
    if (rc != HIRA_OK) return rc;
    HIRA_CHECK_ARG(n_src >= 1 && n_dst >= 1 && from->n_heads % n_src == 0 && to->n_heads % n_dst == 0 &&
                   from->n_heads / n_src == to->n_heads / n_dst, HIRA_ERR_SHAPE,
                   "hira_gather_index: %d and %d heads are not the same number for each of %d and %d sequences", from->n_heads,
                   to->n_heads, n_src, n_dst);
    HIRA_CHECK_ARG(from->dtype == to->dtype && from->vdtype == to->vdtype && from->depth == to->depth && from->bf == to->bf &&
                   from->dim == to->dim && from->vdim == to->vdim && from->cap_parents == to->cap_parents, HIRA_ERR_SHAPE,
                   "hira_gather_index: the two indexes differ in more than their heads");
    const bool in_place = from->children == to->children;
    const int heads = from->n_heads / n_src;
    const long long p = from->active_parents > 0 ? from->active_parents : from->cap_parents, cp = from->cap_parents, bf = from->bf;
    const long long g = from->depth == 3 ? (p + bf - 1) / bf : 0, cg = from->cap_gp;
    const long long es = (long long)elem_size(from->dtype), ves = (long long)elem_size(from->vdtype);
    hira_gather_item_t it[GA_ITEMS];
    int n = 0;
    // the parents in use, and what belongs to them, lie before `p` in every head; behind is nothing
    auto add = [&](const void* src, void* dst, long long row, long long rows, long long cap, uint32_t fill, bool clear = true) {
        if (!src || !dst) return;
        it[n++] = hira_gather_item_t{src, dst, heads * cap * row, heads * cap * row, cap * row, cap * row, rows * row,
                                     (clear ? cap : rows) * row, heads, fill};
    };
    add(from->children, to->children, from->dim * es, p * bf, cp * bf, 0);
    add(from->values, to->values, from->vdim * ves, p * bf, cp * bf, 0);
    add(from->children_q8, to->children_q8, 128, p * bf, cp * bf, 0, false);      // of free slots nothing is kept there
    add(from->slot2token, to->slot2token, 4, p * bf, cp * bf, 0xffffffffu);
    add(from->children_q8_meta, to->children_q8_meta, 4, p * bf, cp * bf, 0, false);
    add(from->parents, to->parents, from->dim * es, p, cp, 0);
    add(from->parent_radii, to->parent_radii, 4, p, cp, 0);
    add(from->parent_sqnorm, to->parent_sqnorm, 4, p, cp, 0);
    add(from->child_counts, to->child_counts, 4, p, cp, 0);
    if (from->depth == 3) {
        add(from->grand_parents, to->grand_parents, from->dim * es, g, cg, 0);
        add(from->gp_radii, to->gp_radii, 4, g, cg, 0);
        add(from->gp_sqnorm, to->gp_sqnorm, 4, g, cg, 0);
        add(from->gp_counts, to->gp_counts, 4, g, cg, 0);
    }
    add(from->used, to->used, 4, 4, 4, 0);
    add(from->q8_chan_scale, to->q8_chan_scale, 4, HIRA_Q8_CHAN, HIRA_Q8_CHAN, 0);
    if (samples) {
        HIRA_CHECK_ARG(in_place && sample_bytes >= 0, HIRA_ERR_ARG, "hira_gather_index: samples move in place only");
        it[n++] = hira_gather_item_t{samples, samples, heads * sample_bytes, heads * sample_bytes, sample_bytes, sample_bytes,
                                     sample_bytes, sample_bytes, heads, 0};
    }
    return run_gather(it, n, index, n_src, n_dst, in_place, in_place ? nullptr : status_from, status, stream);
}
