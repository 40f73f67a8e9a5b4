// Decode attention of a batch whose sequences share a prefix: one token per sequence attends the prefix's rows (one copy for the
// batch) and the rows of its own cache. Optionally the weight that each own row received, summed over the query heads of its
// kv head, is added to an accumulator (what an eviction by attention weight looks at).
//
// Mathematics: o = sum_t p_t v_t with p the softmax over prefix and own rows. The rows are cut into pieces; each gives its own
// softmax-normalised sum and log-sum-exp, and the pieces merge by weights exp(lse_i - LSE). All B * G query rows of a kv head meet the
// prefix together as one matrix, so a prefix row is read once for the batch and not once per sequence.
//
// Two launches. With a long prefix and many query rows the first is the prefix's own kernel (attn_shared_prefix.cu), on some of whose CTAs
// the split pass (shared_split.cuh) takes the own rows:
//   split   tiles of 64 (row, head) pairs of K and V, prefix tiles first, then the own rows of sequence after sequence, are dealt to the
//           CTAs in contiguous runs of equal cost (two CTAs per SM). A warp streams K and V tiles through a ring in shared memory, a TMA
//           box each; four warps multiply by mma.sync (16 query rows x 16 keys x 8 at a time). A warp owns 16 query rows of one kv
//           head and a share of the tile's keys: with few query rows the four warps take four heads (whose slices of a cache row are
//           contiguous) or four shares of the keys, with many rows of the prefix product four blocks of 16 rows.
//   merge   folds the pieces of an output row, by a warp, a CTA, or a CTA per slice of the row; further CTAs turn the scaled scores that
//           the split pass left in the workspace into weights (exp2(s - LSE)), sum them over the heads and add them to the accumulators.
// The scores of own rows cost 4 bytes per query head and row each way through L2, next to 4 * head_dim bytes of K and V per kv head.
// P enters the second product rounded once to the caches' type when the output is 16 bits wide too, which adds about as much error as the
// output's own rounding (together 1.4 times the error of that alone; the residual would be a second product), and for fp32 outputs in three
// parts of bf16 (24 bits) or two of fp16 (23 bits, or 2^-32 of the row's maximum where p is small: fp16 probabilities are lifted by 2^7, to
// the upper end of fp16's range).
//
// Bound by HBM where there is enough to read: 16 ragged caches of up to 4096 rows (168 MB, with weights) take 38.9 us in a graph of
// calls, of which the streaming alone takes 30; 7 sequences over 131072 shared rows (543 MB) 96 us = 5.6 TB/s. Smaller calls are a chain
// of latencies: lengths and dealing 1.1 us, query rows and first tile 2.5, a tile 1.2 us from barrier to barrier, pieces and merge 4.
// What that taught: query rows requested behind the tiles' 28 MB came 3 to 5 us late, a chain of eight dependent MMAs and divisions by
// variables show, and a tile in two slots (K is handed back before the softmax) keeps the stream going.
#include <cuda.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <type_traits>

#include "shared_split.cuh"

namespace b200 {
namespace {

constexpr int kThreads = 128;
using tc::fast_exp2;

template <int D, bool BF16, bool RES>
__global__ void __launch_bounds__(kSplitThreads, 2)
shared_split_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_kp,
                    const __grid_constant__ CUtensorMap tm_vp, const __grid_constant__ SharedParams p) {
    extern __shared__ unsigned char smem_raw[];
    split_body<D, BF16, RES>(tm_k, tm_v, tm_kp, tm_vp, p, smem_raw, blockIdx.x, threadIdx.x, 0);
}

// The pieces of one query row: of the prefix, then of its own cache.
struct Pieces {
    const float* o[2];
    const float* lse[2];
    uint32_t first[2], ts[2], count[2];
    uint64_t step[2];  // rows between consecutive records of one CTA
};
template <int D>
__device__ __forceinline__ void find_pieces(const SharedParams& p, uint32_t b, uint32_t h, Pieces& x) {
    const uint32_t kvh = fast_div(h, p.div_group), g = h - kvh * p.group;
    x.count[0] = 0;
    if (p.prefix_segs) {
        const Shape& sh = p.pre;
        // (rec_rows and hpc are powers of two here, hpc at most four)
        const uint32_t row = b * p.group + g, rb = row >> (31 - __clz(sh.rec_rows)), r = row & (sh.rec_rows - 1);
        const uint32_t hg = kvh >> (sh.hpc >> 1), hs = kvh & (sh.hpc - 1), seg = hg * p.row_blocks + rb;
        const uint32_t w = p.seg_pre[seg];
        const uint64_t at = (static_cast<uint64_t>((w & 0xffffu) + seg) * sh.ts * sh.hpc + hs) * sh.rec_rows + r;
        x.step[0] = static_cast<uint64_t>(sh.hpc) * sh.rec_rows;
        x.count[0] = (w >> 16) * sh.ts;
        x.o[0] = p.part_pre + at * D;
        x.lse[0] = p.lse_pre + at;
    }
    const Shape& sh = p.own;
    const uint32_t hg = kvh >> (sh.hpc >> 1), hs = kvh & (sh.hpc - 1), seg = b * sh.groups + hg;
    const uint32_t w = p.seg_own[seg];
    const uint64_t at = (static_cast<uint64_t>((w & 0xffffu) + seg) * sh.ts * sh.hpc + hs) * sh.rec_rows + g;
    x.step[1] = static_cast<uint64_t>(sh.hpc) * sh.rec_rows;
    x.count[1] = (w >> 16) * sh.ts;
    x.o[1] = p.part_own + at * D;
    x.lse[1] = p.lse_own + at;
}

// Output CTAs: one per (query row, slice of SLICE floats). Groups of SLICE / 4 lanes take a piece each, several pieces in flight per
// lane; the groups' results merge by shuffles, then over the warps. WARP_ROWS: a warp takes a whole row by itself, four rows a CTA (many
// rows of few pieces: 2048 rows of ten pieces take 11 us with four warps a row). Score CTAs behind them.
template <int D, int SLICE, bool WARP_ROWS, bool SCORED>
__global__ void __launch_bounds__(kThreads, !SCORED ? 1 : SLICE < D ? 8 : 6) shared_merge_kernel(const __grid_constant__ SharedParams p) {
    constexpr int kLanes = SLICE / 4;                                // of a group
    constexpr int kGroups = (WARP_ROWS ? 32 : kThreads) / kLanes;    // pieces at once
    __shared__ __align__(16) float s_o[4][SLICE];
    __shared__ float s_ml[4][2];
    __shared__ float s_lse[64];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    grid_dep_launch_dependents();
    grid_dep_wait();
    if (blockIdx.x < p.out_ctas) {
        const uint32_t row = WARP_ROWS ? blockIdx.x * 4 + warp : blockIdx.x / (D / SLICE), slice = WARP_ROWS ? 0 : blockIdx.x % (D / SLICE);
        if (WARP_ROWS && row >= p.batch * p.n_heads) return;
        const uint32_t b = fast_div(row, p.div_heads), h = row - b * p.n_heads;
        Pieces x;
        find_pieces<D>(p, b, h, x);
        const int in_group = lane % kLanes, group = (WARP_ROWS ? lane : tid) / kLanes;
        float m = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        auto fold = [&](float mo, float lo, float4 v) {  // another state: maximum, sum, weighted sum
            const float mn = fmaxf(m, mo), safe = mn == -INFINITY ? 0.f : mn;
            const float f = fast_exp2(m - safe), w = fast_exp2(mo - safe);
            l = l * f + lo * w;
            acc.x = acc.x * f + v.x * w;
            acc.y = acc.y * f + v.y * w;
            acc.z = acc.z * f + v.z * w;
            acc.w = acc.w * f + v.w * w;
            m = mn;
        };
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            constexpr int kAhead = 4;
            for (uint32_t i0 = group; i0 < x.count[kind]; i0 += kGroups * kAhead) {
                float ls[kAhead];
                float4 v[kAhead];
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    const uint32_t i = i0 + a * kGroups;
                    ls[a] = -INFINITY;
                    v[a] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (i < x.count[kind]) {
                        ls[a] = x.lse[kind][i * x.step[kind]];
                        v[a] = *reinterpret_cast<const float4*>(x.o[kind] + i * x.step[kind] * D + slice * SLICE + in_group * 4);
                    }
                }
#pragma unroll
                for (int a = 0; a < kAhead; ++a) fold(ls[a], 1.f, v[a]);
            }
        }
#pragma unroll
        for (int d = kLanes; d < 32; d *= 2) {
            const float mo = __shfl_xor_sync(0xffffffffu, m, d), lo = __shfl_xor_sync(0xffffffffu, l, d);
            float4 v;
            v.x = __shfl_xor_sync(0xffffffffu, acc.x, d);
            v.y = __shfl_xor_sync(0xffffffffu, acc.y, d);
            v.z = __shfl_xor_sync(0xffffffffu, acc.z, d);
            v.w = __shfl_xor_sync(0xffffffffu, acc.w, d);
            fold(mo, lo, v);
        }
        if constexpr (WARP_ROWS) {
            if (lane < kLanes) {
                const float inv = l == 0.f ? 0.f : 1.f / l;  // no row at all: zeros; NaN stays NaN
                const size_t at = static_cast<size_t>(row) * D + lane * 4;
                acc.x *= inv, acc.y *= inv, acc.z *= inv, acc.w *= inv;
                if (p.o_dtype == ATTN_DTYPE_F32) *reinterpret_cast<float4*>(static_cast<float*>(p.o) + at) = acc;
                else if (p.o_dtype == ATTN_DTYPE_F16) *reinterpret_cast<uint2*>(static_cast<__half*>(p.o) + at) = make_uint2(pack2<false>(acc.x, acc.y), pack2<false>(acc.z, acc.w));
                else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.o) + at) = make_uint2(pack2<true>(acc.x, acc.y), pack2<true>(acc.z, acc.w));
            }
            if (lane == 0 && p.lse) p.lse[row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
            return;
        }
        if (lane < kLanes) *reinterpret_cast<float4*>(&s_o[warp][lane * 4]) = acc;
        if (lane == 0) {
            s_ml[warp][0] = m;
            s_ml[warp][1] = l;
        }
        __syncthreads();
        if (tid < SLICE) {
            const float mm = fmaxf(fmaxf(s_ml[0][0], s_ml[1][0]), fmaxf(s_ml[2][0], s_ml[3][0]));
            const float safe = mm == -INFINITY ? 0.f : mm;
            float sum = 0.f, val = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = fast_exp2(s_ml[w][0] - safe);
                sum += f * s_ml[w][1];
                val += f * s_o[w][tid];
            }
            val = sum == 0.f ? 0.f : val / sum;
            const size_t at = static_cast<size_t>(row) * D + slice * SLICE + tid;
            if (p.o_dtype == ATTN_DTYPE_F32) static_cast<float*>(p.o)[at] = val;
            else if (p.o_dtype == ATTN_DTYPE_F16) static_cast<__half*>(p.o)[at] = __float2half_rn(val);
            else static_cast<__nv_bfloat16*>(p.o)[at] = __float2bfloat16_rn(val);
            if (tid == 0 && slice == 0 && p.lse) p.lse[row] = sum == 0.f ? -INFINITY : (mm + __log2f(sum)) * 0.69314718055994531f;
        }
        return;
    }
    if constexpr (!SCORED) return;
    // ---- weights of the own rows of one (sequence, kv head)
    const uint32_t idx = blockIdx.x - p.out_ctas;
    const uint32_t seg = idx / p.score_chunks, chunk = idx - seg * p.score_chunks;
    const uint32_t b = seg / p.n_kv_heads, kvh = seg - b * p.n_kv_heads;
    const uint32_t len = own_len(p, b);
    const uint32_t begin = chunk * p.score_rows, end = min(len, begin + p.score_rows);
    if (begin >= end) return;
    // Sixteen scores of a thread are requested at once, the first ones ahead of the log-sum-exps: four heads of four rows, kThreads apart, or
    // sixteen heads where a CTA has no more rows than threads (twelve heads per kv head, 128 rows: 5 us with four at a time).
    const float* raw = p.raw + (static_cast<size_t>(b) * p.n_heads + kvh * p.group) * p.raw_stride;
    const float* before = p.scores ? p.scores + seg * p.score_stride : nullptr;
    float* after = p.scores_out + seg * p.score_out_stride;
    const bool one_row = p.score_rows == kThreads;
    const uint32_t heads_at_once = one_row ? 16 : 4;
    float w[4], x[16];
    auto fetch_rows = [&](uint32_t t0) {
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const uint32_t t = t0 + a * kThreads;
            w[a] = before && t < end ? before[t] : 0.f;
        }
    };
    // score i of a thread: row t0 + a * kThreads of head g0 + g
    auto fetch_heads = [&](uint32_t t0, uint32_t g0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t g = g0 + (one_row ? i : i / 4), t = t0 + (one_row ? 0 : i % 4 * kThreads);
            x[i] = t < end && g < p.group ? raw[g * p.raw_stride + t] : -INFINITY;
        }
    };
    fetch_rows(begin + tid);
    fetch_heads(begin + tid, 0);
    // the heads' log-sum-exps: eight lanes a head
    for (uint32_t g0 = 0; g0 < p.group; g0 += kThreads / 8) {
        const uint32_t g = g0 + tid / 8;
        float m = -INFINITY, l = 0.f;
        if (g < p.group) {
            Pieces pc;
            find_pieces<D>(p, b, kvh * p.group + g, pc);
#pragma unroll
            for (int kind = 0; kind < 2; ++kind) {
                constexpr int kAhead = 4;
                for (uint32_t i0 = tid & 7; i0 < pc.count[kind]; i0 += 8 * kAhead) {
                    float ls[kAhead];
#pragma unroll
                    for (int a = 0; a < kAhead; ++a) {
                        const uint32_t i = i0 + 8 * a;
                        ls[a] = i < pc.count[kind] ? pc.lse[kind][i * pc.step[kind]] : -INFINITY;
                    }
                    const float mn = fmaxf(fmaxf(fmaxf(ls[0], ls[1]), fmaxf(ls[2], ls[3])), m), safe = mn == -INFINITY ? 0.f : mn;
                    l = l * fast_exp2(m - safe) + fast_exp2(ls[0] - safe) + fast_exp2(ls[1] - safe) + fast_exp2(ls[2] - safe) +
                        fast_exp2(ls[3] - safe);
                    m = mn;
                }
            }
        }
#pragma unroll
        for (int d = 1; d < 8; d *= 2) {
            const float om = __shfl_xor_sync(0xffffffffu, m, d), ol = __shfl_xor_sync(0xffffffffu, l, d);
            const float mn = fmaxf(m, om), safe = mn == -INFINITY ? 0.f : mn;
            l = l * fast_exp2(m - safe) + ol * fast_exp2(om - safe);
            m = mn;
        }
        if ((tid & 7) == 0 && g < p.group) s_lse[g] = m + __log2f(l);
    }
    __syncthreads();
    for (uint32_t t0 = begin + tid; t0 < end; t0 += 4 * kThreads) {
        if (t0 != begin + tid) {
            fetch_rows(t0);
            fetch_heads(t0, 0);
        }
        float sum[4] = {};
        for (uint32_t g0 = 0; g0 < p.group; g0 += heads_at_once) {
            if (g0) fetch_heads(t0, g0);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t g = g0 + (one_row ? i : i / 4);
                sum[i % 4] += fast_exp2(x[i] - (g < p.group ? s_lse[g] : 0.f));
            }
        }
        if (one_row) {
            if (t0 < end) after[t0] = w[0] + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
        } else {
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const uint32_t t = t0 + a * kThreads;
                if (t < end) after[t] = w[a] + sum[a];
            }
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Dimensions -> how the warps share the tiles, and the pieces of the workspace (in 32-bit words).
struct SharedPlan {
    Shape pre, own;
    uint32_t row_blocks, prefix_segs, own_segs, grid;
    uint32_t pairs, tensor_segs, tensor_grid;  // the prefix on the tensor cores
    uint32_t tiles;  // as `pairs`, in half as many query rows, which is what a segment of an fp32 output has
    size_t lse_pre, part_own, lse_own, seg_pre, seg_own, raw, words;
    uint64_t raw_stride;
};
void set_shape(Shape* s, uint32_t query_rows, uint32_t n_kv_heads) {
    s->wm = query_rows <= 16 ? 1 : query_rows <= 32 ? 2 : 4;
    s->hpc = 4 / s->wm;
    while (n_kv_heads % s->hpc) s->hpc /= 2;
    s->ts = 4 / (s->wm * s->hpc);
    s->keys = kTilePairs / s->hpc;
    s->groups = n_kv_heads / s->hpc;
}
int make_shared_plan(uint32_t batch, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, uint32_t scored_rows, const DeviceInfo& dev,
                     SharedPlan* plan) {
    if (batch == 0 || n_heads == 0 || n_kv_heads == 0 || n_heads % n_kv_heads != 0) return ATTN_ERR_INVALID_ARG;
    const uint32_t group = n_heads / n_kv_heads;
    if ((head_dim != 64 && head_dim != 128) || group > 64 || batch > kMaxBatch || n_heads > 1024) return ATTN_ERR_UNSUPPORTED;
    SharedPlan& s = *plan;  // (sized for either type of output)
    set_shape(&s.own, group, n_kv_heads);
    s.own.rec_rows = group;
    set_shape(&s.pre, batch * group, n_kv_heads);
    s.pre.rec_rows = 16 * s.pre.wm;
    s.row_blocks = (batch * group + s.pre.rec_rows - 1) / s.pre.rec_rows;
    s.prefix_segs = s.pre.groups * s.row_blocks;
    s.own_segs = batch * s.own.groups;
    s.grid = 2 * dev.sm_count;
    s.pairs = (batch * group + kPrefixRows - 1) / kPrefixRows;
    s.tiles = (batch * group + kPrefixRows / 2 - 1) / (kPrefixRows / 2);
    s.tensor_segs = s.pairs * n_kv_heads;
    s.tensor_grid = dev.sm_count;
    const size_t pre_rows = std::max(static_cast<size_t>(s.grid + s.prefix_segs) * s.pre.ts * s.pre.hpc * s.pre.rec_rows,
                                     static_cast<size_t>(s.tensor_grid + s.tensor_segs) * kPrefixRows);
    const size_t own_rows = static_cast<size_t>(s.grid + s.own_segs) * s.own.ts * s.own.hpc * s.own.rec_rows;
    auto round4 = [](size_t n) { return (n + 3) / 4 * 4; };
    s.lse_pre = pre_rows * head_dim;
    s.part_own = s.lse_pre + round4(pre_rows);
    s.lse_own = s.part_own + own_rows * head_dim;
    s.seg_pre = s.lse_own + round4(own_rows);
    s.seg_own = s.seg_pre + round4(std::max(s.prefix_segs, s.tiles * n_kv_heads));
    s.raw = s.seg_own + round4(s.own_segs);
    s.raw_stride = (static_cast<uint64_t>(scored_rows) + 63) / 64 * 64;
    s.words = s.raw + static_cast<size_t>(batch) * n_heads * s.raw_stride;
    return ATTN_OK;
}

// Cache rows as [sequence][128-byte part of a head][kv head][row][64 elements]; a box is a tile: all parts of hpc heads over its
// rows. Rows that the cache does not have read as zeros.
int tile_map(CUtensorMap* map, const void* cache, bool bf16, uint32_t head_dim, uint32_t rows, uint32_t kv_heads, uint32_t batch,
             uint64_t row_stride, uint64_t batch_stride, const Shape& sh) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return ATTN_ERR_CUDA;
    const cuuint64_t dims[5] = {64, rows, kv_heads, head_dim / 64, batch};
    const cuuint64_t strides[4] = {row_stride * 2, head_dim * 2ull, 128, (batch > 1 ? batch_stride : row_stride * rows) * 2};
    const cuuint32_t box[5] = {64, sh.keys, sh.hpc, head_dim / 64, 1};
    const cuuint32_t unit[5] = {1, 1, 1, 1, 1};
    const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, const_cast<void*>(cache), dims,
                           strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return ATTN_OK;
    g_last_cuda_error = static_cast<int>(r);
    return ATTN_ERR_CUDA;
}

// Which kernel takes the prefix, and how the SMs are shared. The split pass can take it along with the own rows in one launch; the
// tensor-core kernel does many query rows or long prefixes faster, but starts and ends more slowly. Where it takes fewer CTAs than there
// are SMs, the split pass of the same launch runs beside it on the others, else as its CTAs end. Times in us, measured on shapes of 64-
// and 128-dimension heads (graphs of calls).
struct PrefixChoice {
    bool tensor;
    uint32_t prefix_ctas, split_ctas;
};
constexpr uint32_t kMinPrefixBlocks = 2;  // of a CTA
constexpr uint32_t kPieceBlocks = 4;
PrefixChoice choose_prefix(const SharedPlan& plan, uint32_t sms, uint32_t head_dim, uint64_t prefix_tiles, uint64_t own_tiles, uint64_t own_most,
                           uint64_t blocks, uint32_t query_rows, bool res) {
    // (times go by the tiles that are expected, the number of CTAs by those that there can be)
    auto ctas_for = [](uint64_t ctas, uint64_t tiles) { return static_cast<uint32_t>(std::max<uint64_t>(1, std::min<uint64_t>(ctas, tiles))); };
    const uint64_t all = prefix_tiles + own_tiles;
    const uint32_t both_ctas = ctas_for(2 * sms, prefix_tiles + own_most);
    PrefixChoice c{false, 0, both_ctas};
    if (prefix_tiles == 0) return c;
#ifdef ATTN_TRACE
    const char* knob = getenv("ATTN_TRACE_PREFIX");  // profiling knob
    if (knob && atoi(knob) == 0) return c;
#endif
    const double dim = head_dim / 128.0, work = res ? 0.4 + 0.6 * dim : 0.75 + 0.25 * dim;
    const double tile_bytes = 32768.0 * dim, bandwidth = 6.2e6;     // bytes per us
    const double own_tile = (res ? 0.85 : 0.6) * work, own_seg = 2.0, launch = 5.0;  // us of an SM per own tile, of a CTA per own segment; a launch's fixed part
    // of a prefix tile in the split pass, of a key block in the tensor-core kernel; fp32 outputs take two or three times the second products
    const double shared_tile = (plan.pre.wm == 4 ? (res ? 2.9 : 1.15) : plan.pre.wm == 2 ? (res ? 1.35 : 0.65) : res ? 0.9 : 0.6) * work;
    const double block = res ? 1.05 : (query_rows > 128 ? 1.1 : 0.8) * (0.4 + 0.6 * dim);
    const double block_bytes = 16384.0 * 2 * dim;
    auto split_time = [&](double ctas) {
        const double segs = std::ceil(plan.own_segs / ctas) * (own_tiles ? own_seg : 0.0);
        return launch + segs + std::max(own_tiles * own_tile / (ctas / 2), own_tiles * tile_bytes / bandwidth);
    };
    auto prefix_time = [&](double ctas) { return launch + 1.0 + std::max(std::ceil(blocks / ctas) * block, blocks / plan.pairs * block_bytes / bandwidth); };
    const double together = launch + std::max((prefix_tiles * shared_tile + own_tiles * own_tile) / sms, all * tile_bytes / bandwidth);
    // one behind the other
    const uint32_t most = ctas_for(sms, blocks / kMinPrefixBlocks);
    double best = prefix_time(most) + split_time(2.0 * sms) - 2.0;
    c.prefix_ctas = most;
    c.split_ctas = ctas_for(2 * sms, own_most);
    // side by side
    const double both = launch + (own_tiles * tile_bytes + blocks / plan.pairs * block_bytes) / bandwidth;
    for (uint32_t n = 8; n < sms; n += 4) {
        if (n > most) break;
        const uint32_t m = ctas_for(2 * (sms - n), own_most);
        const double t = std::max(std::max(prefix_time(n), split_time(m)), both);
        if (t < best) best = t, c.prefix_ctas = n, c.split_ctas = m;
    }
    c.tensor = best + 1.5 < together;
#ifdef ATTN_TRACE
    if (knob) c.tensor = true;
#endif
    if (!c.tensor) c.split_ctas = both_ctas;
    return c;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" size_t attn_decode_shared_workspace_bytes(uint32_t batch, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim,
                                                     uint32_t scored_rows) {
    DeviceInfo dev{};
    if (current_device_info(&dev) != ATTN_OK) return 0;
    SharedPlan plan{};
    if (make_shared_plan(batch, n_heads, n_kv_heads, head_dim, scored_rows, dev, &plan) != ATTN_OK) return 0;
    return plan.words * 4;
}

extern "C" int attn_decode_shared(const AttnDecodeSharedArgs* a, void* stream_v) {
    if (!a || !a->o || !a->q) return ATTN_ERR_INVALID_ARG;
    if ((a->prefix_len && (!a->k_prefix || !a->v_prefix)) || (a->kv_capacity && (!a->k || !a->v))) return ATTN_ERR_INVALID_ARG;
    if (a->dtype != ATTN_DTYPE_F16 && a->dtype != ATTN_DTYPE_BF16) return ATTN_ERR_UNSUPPORTED;
    if (a->o_dtype != ATTN_DTYPE_F32 && a->o_dtype != a->dtype) return ATTN_ERR_UNSUPPORTED;
    if (a->batch == 0 || a->n_heads == 0 || a->n_kv_heads == 0 || a->n_heads % a->n_kv_heads != 0) return ATTN_ERR_INVALID_ARG;
    if (a->batch > 1 && a->kv_capacity && a->kv_batch_stride == 0) return ATTN_ERR_INVALID_ARG;
    if (a->scores && !a->scores_out) return ATTN_ERR_INVALID_ARG;
    if (a->scores_out && a->kv_capacity == 0) return ATTN_ERR_INVALID_ARG;
    const uint64_t width = static_cast<uint64_t>(a->n_kv_heads) * a->head_dim;
    SharedParams p{};
    const uint64_t prefix_row_stride = a->prefix_row_stride ? a->prefix_row_stride : width;
    const uint64_t row_stride = a->kv_row_stride ? a->kv_row_stride : width, batch_stride = a->kv_batch_stride;
    p.score_stride = a->score_stride ? a->score_stride : a->kv_capacity;
    p.score_out_stride = a->score_out_stride ? a->score_out_stride : a->kv_capacity;
    if (prefix_row_stride < width || row_stride < width || p.score_stride < a->kv_capacity || p.score_out_stride < a->kv_capacity)
        return ATTN_ERR_INVALID_ARG;
    if (!aligned16(a->q) || !aligned16(a->k_prefix) || !aligned16(a->v_prefix) || !aligned16(a->k) || !aligned16(a->v) ||
        (prefix_row_stride | row_stride | batch_stride) % 8 != 0)
        return ATTN_ERR_ALIGNMENT;
    DeviceInfo dev{};
    int rc = current_device_info(&dev);
    if (rc != ATTN_OK) return rc;
    if (dev.cc_major != 10) return ATTN_ERR_DEVICE;
    const bool scored = a->scores_out != nullptr;
    SharedPlan plan{};
    rc = make_shared_plan(a->batch, a->n_heads, a->n_kv_heads, a->head_dim, scored ? a->kv_capacity : 0, dev, &plan);
    if (rc != ATTN_OK) return rc;
    if (!a->workspace || a->workspace_bytes < plan.words * 4) return ATTN_ERR_WORKSPACE;
    if (!aligned16(a->workspace)) return ATTN_ERR_ALIGNMENT;

    p.q = static_cast<const uint16_t*>(a->q);
    p.kv_len = a->kv_capacity ? a->kv_len : nullptr;
    p.kv_len_uniform = a->kv_len_uniform;
    p.batch = a->batch;
    p.n_heads = a->n_heads;
    p.n_kv_heads = a->n_kv_heads;
    p.group = a->n_heads / a->n_kv_heads;
    p.div_heads = divider(p.n_heads);
    p.div_group = divider(p.group);
    p.prefix = a->prefix_len;
    p.rows = a->kv_capacity;
    const float scale = a->scale != 0.f ? a->scale : 1.0f / sqrtf(static_cast<float>(a->head_dim));
    p.scale_log2 = scale * 1.4426950408889634f;
    p.pre = plan.pre;
    p.own = plan.own;
    p.row_blocks = plan.row_blocks;
    p.prefix_segs = a->prefix_len ? plan.prefix_segs : 0;
    const uint64_t prefix_tiles = (static_cast<uint64_t>(a->prefix_len) + plan.pre.keys - 1) / plan.pre.keys;
    const uint64_t own_tiles = (static_cast<uint64_t>(a->kv_capacity) + plan.own.keys - 1) / plan.own.keys;
    if (prefix_tiles * plan.prefix_segs + own_tiles * plan.own_segs > 0x7fffffffull) return ATTN_ERR_UNSUPPORTED;  // 32-bit tile numbers
    p.prefix_tiles = static_cast<uint32_t>(prefix_tiles);
    float* ws = static_cast<float*>(a->workspace);
    p.part_pre = ws;
    p.lse_pre = ws + plan.lse_pre;
    p.part_own = ws + plan.part_own;
    p.lse_own = ws + plan.lse_own;
    p.seg_pre = reinterpret_cast<uint32_t*>(ws + plan.seg_pre);
    p.seg_own = reinterpret_cast<uint32_t*>(ws + plan.seg_own);
    p.raw = scored ? ws + plan.raw : nullptr;
    p.raw_stride = plan.raw_stride;
    p.status = a->status;
    p.o = a->o;
    p.lse = a->lse;
    p.o_dtype = a->o_dtype;
    p.scores = a->scores;
    p.scores_out = a->scores_out;
    // A CTA adds up the weights of 128 rows or a multiple of it, so that there are about eight CTAs per SM.
    const uint64_t segs = static_cast<uint64_t>(a->batch) * a->n_kv_heads;
    const uint64_t per_cta = (segs * a->kv_capacity + 8ull * dev.sm_count - 1) / (8ull * dev.sm_count);
    p.score_rows = static_cast<uint32_t>(std::max<uint64_t>(1, (per_cta + kThreads - 1) / kThreads)) * kThreads;
    p.score_chunks = (a->kv_capacity + p.score_rows - 1) / p.score_rows;

    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    const bool bf16 = a->dtype == ATTN_DTYPE_BF16, res = a->o_dtype == ATTN_DTYPE_F32;
    const uint32_t seg_rows = res ? kPrefixRows / 2 : kPrefixRows;
    if (res) {
        plan.pairs = plan.tiles;
        plan.tensor_segs = plan.tiles * a->n_kv_heads;
    }
    const uint64_t blocks = (static_cast<uint64_t>(a->prefix_len) + kPrefixBlock - 1) / kPrefixBlock * plan.tensor_segs;
    // (lengths that lie on the device are taken to be five eighths of the capacity)
    const uint64_t own_guess = a->kv_len ? own_tiles * plan.own_segs * 5 / 8
                                         : (std::min(a->kv_len_uniform, a->kv_capacity) + plan.own.keys - 1ull) / plan.own.keys * plan.own_segs;
    PrefixChoice choice = choose_prefix(plan, dev.sm_count, a->head_dim, prefix_tiles * p.prefix_segs, own_guess, own_tiles * plan.own_segs, blocks,
                                        std::min(a->batch * p.group, seg_rows), res);
    if (blocks > 0x7fffffffull) choice.tensor = false;
    const bool tensor = choice.tensor;
    p.scale_log2 = fabsf(p.scale_log2);
    p.q_sign = scale < 0.f ? 0x80008000u : 0u;
    SharedParams in_split = p;
    SharedPrefixParams t{};
    if (tensor) {
        t.q = a->q;
        t.k = a->k_prefix;
        t.v = a->v_prefix;
        t.part = p.part_pre;
        t.lse = p.lse_pre;
        t.seg_ctas = p.seg_pre;
        t.row_stride = prefix_row_stride;
        t.batch = p.batch;
        t.n_heads = p.n_heads;
        t.n_kv_heads = p.n_kv_heads;
        t.group = p.group;
        t.div_group = p.div_group;
        t.head_dim = a->head_dim;
        t.prefix = p.prefix;
        t.pairs = plan.pairs;
        t.segments = plan.tensor_segs;
        t.grid = choice.prefix_ctas;
        t.q_sign = p.q_sign;
        // A run that crosses from one segment into the next pays a second set of query rows and a second piece, about as much as
        // kPieceBlocks blocks: whole CTAs per segment unless that makes the longest run longer by more.
        const uint64_t seg_blocks = blocks / plan.tensor_segs, per_seg = std::min<uint64_t>(t.grid / plan.tensor_segs, seg_blocks);
        if (per_seg > 0 && (seg_blocks + per_seg - 1) / per_seg <= (blocks + t.grid - 1) / t.grid + kPieceBlocks) {
            t.ctas_per_seg = static_cast<uint32_t>(per_seg);
            t.grid = t.ctas_per_seg * plan.tensor_segs;
        }
        t.scale_log2 = p.scale_log2;
        t.status = p.status;
        t.bf16 = bf16;
        t.residual = res;
        in_split.prefix_segs = in_split.prefix_tiles = 0;
        // how the merge pass finds the pieces: one record of a segment's rows per CTA and segment
        p.pre = Shape{1, 1, 1, kPrefixBlock, p.n_kv_heads, seg_rows};
        p.row_blocks = plan.pairs;
        p.prefix_segs = plan.tensor_segs;
    }
    const uint32_t grid = in_split.ctas = choice.split_ctas;
    CUtensorMap tm_k{}, tm_v{}, tm_kp{}, tm_vp{};
    if (a->kv_capacity) {
        if ((rc = tile_map(&tm_k, a->k, bf16, a->head_dim, p.rows, p.n_kv_heads, p.batch, row_stride, batch_stride, p.own)) != ATTN_OK ||
            (rc = tile_map(&tm_v, a->v, bf16, a->head_dim, p.rows, p.n_kv_heads, p.batch, row_stride, batch_stride, p.own)) != ATTN_OK)
            return rc;
    }
    if (in_split.prefix_segs) {
        if ((rc = tile_map(&tm_kp, a->k_prefix, bf16, a->head_dim, p.prefix, p.n_kv_heads, 1, prefix_row_stride, 0, p.pre)) != ATTN_OK ||
            (rc = tile_map(&tm_vp, a->v_prefix, bf16, a->head_dim, p.prefix, p.n_kv_heads, 1, prefix_row_stride, 0, p.pre)) != ATTN_OK)
            return rc;
    }
    // Shared memory: alignment, the ring, its barriers, the row of zeros, four warps' query rows, s_cum, s_warp; as many slots as fit.
    const size_t slot_bytes = static_cast<size_t>(kTilePairs) * a->head_dim * 2;
    in_split.q_held = in_split.prefix_segs ? 16 : std::min<uint32_t>(16, p.group);
    const size_t fixed = 1024 + kMaxSlots * 16 + (1 + 4 * in_split.q_held) * a->head_dim * 2 + (a->batch + 1 + 6) * 4;
    in_split.slots = static_cast<uint32_t>(std::min<size_t>(kMaxSlots, (kSplitSmem - fixed) / slot_bytes));
    const size_t smem = fixed + in_split.slots * slot_bytes;
    // A prefix tile of four row blocks keeps a CTA as busy as two own tiles; others are as fast as memory in either form.
    // A CTA that meets a second own segment ended 2.5 us, two tiles, behind the others (16 ragged caches of up to 4096 rows). Not counted
    // where a CTA has few tiles: there it would only keep CTAs idle.
    in_split.switch_units = own_guess >= 8ull * grid ? 2 : 0;
    in_split.prefix_weight = plan.pre.wm == 4 && plan.own.wm == 1 ? 2 : 1;
    if (prefix_tiles * in_split.prefix_segs * in_split.prefix_weight + (own_tiles + in_split.switch_units) * plan.own_segs > 0x7fffffffull) return ATTN_ERR_UNSUPPORTED;  // 32-bit units
    auto split = [&](auto kernel) -> int {
        B200_CUDA_TRY(allow_max_smem(kernel));
        B200_CUDA_TRY(launch_dependent(kernel, dim3(grid), dim3(kSplitThreads), smem, stream, tm_k, tm_v, tm_kp, tm_vp, in_split));
        g_launch_count.fetch_add(1, std::memory_order_relaxed);
        return ATTN_OK;
    };
    if (tensor) {
        rc = launch_shared_prefix(t, in_split, tm_k, tm_v, smem, stream);
    } else if (a->head_dim == 128) {
        rc = bf16 ? (res ? split(shared_split_kernel<128, true, true>) : split(shared_split_kernel<128, true, false>))
                  : (res ? split(shared_split_kernel<128, false, true>) : split(shared_split_kernel<128, false, false>));
    } else {
        rc = bf16 ? (res ? split(shared_split_kernel<64, true, true>) : split(shared_split_kernel<64, true, false>))
                  : (res ? split(shared_split_kernel<64, false, true>) : split(shared_split_kernel<64, false, false>));
    }
    if (rc != ATTN_OK) return rc;
    // Few output rows: slices of 32 floats, so that more CTAs take fewer pieces each. Many rows: whole rows, by a warp each where few CTAs
    // share a segment. (16-byte stores need an output aligned to them.)
    const uint64_t rows = static_cast<uint64_t>(a->batch) * a->n_heads;
    const bool sliced = rows * (a->head_dim / 32) <= 8ull * dev.sm_count;
    const uint64_t pieces = (p.prefix_segs ? (tensor ? choice.prefix_ctas : grid) / p.prefix_segs * p.pre.ts + 1 : 0) + grid / plan.own_segs * p.own.ts + 1;
    const bool warp_rows = !sliced && pieces <= 24 && aligned16(a->o);
    p.out_ctas = static_cast<uint32_t>(sliced ? rows * (a->head_dim / 32) : warp_rows ? (rows + 3) / 4 : rows);
    const uint64_t merge_ctas = p.out_ctas + (scored ? segs * p.score_chunks : 0);
    if (merge_ctas > 0x7fffffffull) return ATTN_ERR_UNSUPPORTED;
    auto merge = [&](auto kernel) -> int {
        B200_CUDA_TRY(launch_dependent(kernel, dim3(static_cast<uint32_t>(merge_ctas)), dim3(kThreads), 0, stream, p));
        g_launch_count.fetch_add(1, std::memory_order_relaxed);
        return ATTN_OK;
    };
    auto merge_rows = [&](auto scores) -> int {
        constexpr bool S = decltype(scores)::value;
        if (sliced) return a->head_dim == 128 ? merge(shared_merge_kernel<128, 32, false, S>) : merge(shared_merge_kernel<64, 32, false, S>);
        if (warp_rows) return a->head_dim == 128 ? merge(shared_merge_kernel<128, 128, true, S>) : merge(shared_merge_kernel<64, 64, true, S>);
        return a->head_dim == 128 ? merge(shared_merge_kernel<128, 128, false, S>) : merge(shared_merge_kernel<64, 64, false, S>);
    };
    return scored ? merge_rows(std::true_type{}) : merge_rows(std::false_type{});
}
