// Eviction from a KV cache by accumulated attention weight: of every (sequence, kv head), the first `sink` rows, the last
// `recent` rows and the rows with the largest scores, `keep` in all, stay; their order stays too. Ties go to the lowest row.
//
// Two launches, or one that does both for small calls. (1) Which rows: a CTA or a cluster of them per (sequence, kv head) finds the
// keep-th largest key by a radix selection (digits of 11, 11 and 10 bits, a histogram in shared memory per CTA, summed over the cluster), then counts and writes the
// kept rows in order. A score's key is its bit pattern mapped so that unsigned order is the order of the numbers (NaN below
// everything, -0 = +0); always-kept rows carry the largest key. (2) The copy, bound by memory: kept K and V rows and scores are
// read once and written once. Into another cache it is a plain gather with as many blocks as it has work for. In place, a row only
// moves down, so one CTA per (head, slice of the row) goes through the rows in order: everything it still has to read lies
// behind what it writes.
//
// Graphs of calls: 16 ragged sequences of up to 4096 rows into caches of 1999 (8 kv heads of 128, 246 MB) 49.1 us, of which the
// copy is 39 (6.2 TB/s) and the selection 6; one sequence of 131072 rows to 16384 39.3 us: copy 22, the rest the selection on 64 SMs (48.6
// while every CTA read the others' histograms whole, 2 us a digit); 1024 rows to 256, one launch,
// 6.2 us (two: 9.3), all of it latency. In place: 16 sequences of 2080 rows back to 2048 (268 MB) 91 us, of 4096 to 1999 76, one of
// 131072 to 16384 117: 2.9, 3.5 and 1.1 TB/s, a CTA per (head, slice) going through its rows one batch behind the other.
#include <cooperative_groups.h>

#include <algorithm>

#include "attn_internal.cuh"
#include "operand_memory.cuh"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

namespace cg = cooperative_groups;

struct EvictParams {
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* k_out;
    uint16_t* v_out;
    const float* scores;
    float* scores_out;
    uint32_t* kept;
    const uint32_t* kv_len;
    uint32_t* kv_len_out;
    uint64_t row_stride, batch_stride, out_row_stride, out_batch_stride;
    uint64_t score_stride, score_out_stride;  // floats between the rows of (sequence, kv head)
    uint32_t batch, n_kv_heads, head_dim, rows, out_rows, keep, sink, recent;
    uint32_t* status;
    uint32_t staged;  // keys of a CTA's slice that its shared memory holds
    uint32_t scores_aligned;  // every run of scores starts on 16 bytes
    uint32_t slices;  // in place: pieces of a head's row
    uint32_t in_place;
};

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;
constexpr int kGroups = kBins / 32;
constexpr uint32_t kSelWords = 4 * kBins + 3 * kGroups + 2 * kSelWarps + 4;  // shared memory in front of the keys
constexpr uint32_t kAlways = 0xffffffffu;
constexpr uint64_t kOneLaunchBytes = 256 * 1024, kOneLaunchSmem = 200 * 1024;

// Unsigned order of the keys = order of the scores; NaN gets 0, below -inf. No score maps to kAlways (that pattern would be a NaN).
__device__ __forceinline__ uint32_t score_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);  // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A sequence's rows; a length beyond the cache is clamped to it (and reported by the selection). kv_len_out may be kv_len: the
// selection reads it, and the copy, whose first CTA of a sequence writes the new length, needs only min(length, keep), which is
// the same from either value.
__device__ __forceinline__ uint32_t rows_of(const EvictParams& p, uint32_t b) { return min(p.kv_len ? p.kv_len[b] : p.rows, p.rows); }

// This CTA's share, one of gridDim.x, of what a (sequence, kv head) keeps: K and V, scores, and the list itself.
__device__ __forceinline__ void copy_share(const EvictParams& p, const uint32_t* kept, uint32_t b, uint32_t seg, uint32_t len) {
    __syncthreads();  // the list is complete
    const uint32_t h = seg - b * p.n_kv_heads, after = min(len, p.keep);
    const uint32_t first = blockIdx.x * kSelThreads + threadIdx.x, step = gridDim.x * kSelThreads;
    if (h == 0 && first == 0) p.kv_len_out[b] = after;
    for (uint32_t j = first; j < p.out_rows; j += step) {
        if (j < p.keep) p.kept[static_cast<size_t>(seg) * p.keep + j] = kept[j];
        p.scores_out[seg * p.score_out_stride + j] = j < after ? p.scores[seg * p.score_stride + kept[j]] : 0.f;
    }
    const uint32_t D16 = p.head_dim / 8, total = after * D16;
    const size_t in = b * p.batch_stride + static_cast<size_t>(h) * p.head_dim, out = b * p.out_batch_stride + static_cast<size_t>(h) * p.head_dim;
#pragma unroll 2
    for (uint32_t u = first; u < total; u += step) {
        const uint32_t j = u / D16, c = (u - j * D16) * 8;
        const uint64_t from = in + kept[j] * p.row_stride + c, to = out + j * p.out_row_stride + c;
        const uint4 xk = __ldcs(reinterpret_cast<const uint4*>(p.k + from)), xv = __ldcs(reinterpret_cast<const uint4*>(p.v + from));
        *reinterpret_cast<uint4*>(p.k_out + to) = xk;
        *reinterpret_cast<uint4*>(p.v_out + to) = xv;
    }
}

// One cluster of kCtas per (sequence, kv head) = blockIdx.y. A CTA keeps the keys of its rows in shared memory and goes through them four
// at a time; rows beyond `staged` (more than 40960 rows a CTA) are read again from the scores.
// kCopy, for small calls into other caches: one launch. The CTAs of a (sequence, kv head) do not form a cluster, each selects for itself and
// then copies its share of the kept rows.
template <int kCtas, bool kCopy = false>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
    static_assert(!kCopy || kCtas == 1);
    extern __shared__ __align__(16) uint32_t s_all[];
    uint32_t* s_hist = s_all;                   // [4][kBins]: two for the top digit (even and odd lanes: fewer meet in a bin), one for each other
    uint32_t* s_group = s_hist + 4 * kBins;     // [3][kGroups]: a digit's histogram in sums over 32 bins
    uint32_t* s_gt = s_group + 3 * kGroups;     // [kSelWarps]
    uint32_t* s_eq = s_gt + kSelWarps;          // [kSelWarps]
    uint32_t* s_pick = s_eq + kSelWarps;        // digit, keys above it
    uint32_t* s_counts = s_pick + 2;            // this CTA's keys above the threshold, equal to it
    uint32_t* s_keys = s_counts + 2;            // [staged]
    cg::cluster_group cluster = cg::this_cluster();
    auto meet = [&]() {
        if constexpr (kCtas > 1) cluster.sync();
        else __syncthreads();
    };
    const uint32_t rank = kCopy ? 0u : blockIdx.x;
    const uint32_t seg = blockIdx.y, b = seg / p.n_kv_heads;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    grid_dep_launch_dependents();
    for (int i = tid; i < 4 * kBins / 4; i += kSelThreads) reinterpret_cast<uint4*>(s_hist)[i] = make_uint4(0, 0, 0, 0);
    grid_dep_wait();
    const uint32_t len = rows_of(p, b);
    uint32_t* kept = kCopy ? s_keys + p.staged : p.kept + static_cast<size_t>(seg) * p.keep;
    if (blockIdx.x == 0 && tid == 0 && p.kv_len && p.kv_len[b] > p.rows && p.status) atomicOr(p.status, ATTN_STATUS_BAD_SHAPE);
    if (len <= p.keep) {  // the same for the whole cluster
        for (uint32_t j = rank * kSelThreads + tid; j < p.keep; j += kCtas * kSelThreads) kept[j] = j < len ? j : 0xffffffffu;
        if constexpr (kCopy) copy_share(p, kept, b, seg, len);
        return;
    }
    // this CTA's rows: a contiguous slice, cut into one contiguous piece per warp
    const uint32_t per_warp = ((len + kCtas * kSelWarps - 1) / (kCtas * kSelWarps) + 127) / 128 * 128;
    const uint32_t begin = min(len, rank * per_warp * kSelWarps), end = min(len, begin + per_warp * kSelWarps);
    const uint32_t n = end - begin, n_staged = min(n, p.staged);
    const float* scores = p.scores + static_cast<size_t>(seg) * p.score_stride + begin;
    const uint32_t sink = p.sink > begin ? p.sink - begin : 0u;                       // relative to the slice from here on
    const uint32_t tail = len - min(len, p.recent) > begin ? len - min(len, p.recent) - begin : 0u;
    auto make_key = [&](uint32_t i, float x) { return (i < sink || i >= tail) ? kAlways : score_key(x); };
    __syncthreads();  // the histograms are clear
    uint32_t* top = s_hist + (lane & 1) * kBins;
    // ---- keys into shared memory, and the top digit's histogram on the way (four 16-byte loads of a thread in flight)
    const uint32_t n4 = p.scores_aligned ? n_staged / 4 : 0u;
    constexpr int kAhead = 4;
    for (uint32_t i0 = tid; i0 < n4; i0 += kAhead * kSelThreads) {
        float4 x[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint32_t i = i0 + a * kSelThreads;
            x[a] = i < n4 ? reinterpret_cast<const float4*>(scores)[i] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint32_t i = i0 + a * kSelThreads;
            if (i < n4) {
                const uint4 k = make_uint4(make_key(4 * i, x[a].x), make_key(4 * i + 1, x[a].y), make_key(4 * i + 2, x[a].z), make_key(4 * i + 3, x[a].w));
                reinterpret_cast<uint4*>(s_keys)[i] = k;
                atomicAdd(&top[k.x >> 21], 1u);
                atomicAdd(&top[k.y >> 21], 1u);
                atomicAdd(&top[k.z >> 21], 1u);
                atomicAdd(&top[k.w >> 21], 1u);
            }
        }
    }
    for (uint32_t i = 4 * n4 + tid; i < n; i += kSelThreads) {
        const uint32_t key = make_key(i, scores[i]);
        if (i < n_staged) s_keys[i] = key;
        atomicAdd(&top[key >> 21], 1u);
    }
    // four keys from row i (a multiple of four) on; rows behind the slice's end get key 0 and must be left out by their index
    auto keys_at = [&](uint32_t i) {
        if (i + 4 <= n_staged) return *reinterpret_cast<const uint4*>(s_keys + i);
        uint32_t k[4];
#pragma unroll
        for (int a = 0; a < 4; ++a) k[a] = i + a < n_staged ? s_keys[i + a] : i + a < n ? make_key(i + a, scores[i + a]) : 0u;
        return make_uint4(k[0], k[1], k[2], k[3]);
    };

    // ---- the keep-th largest key, a digit at a time from the top
    uint32_t prefix = 0, need = p.keep;  // keys whose upper digits are those of prefix are still candidates for the need-th largest
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digit_mask = pass == 2 ? 1023u : 2047u;
        uint32_t* hist = s_hist + (pass == 0 ? 0 : (pass + 1) * kBins);
        if (pass > 0) {
            const int above = pass == 1 ? 21 : 10;
            const uint32_t want = prefix >> above;
            auto count = [&](uint32_t i, uint32_t key) {
                if (key >> above == want && i < n) atomicAdd(&hist[(key >> shift) & digit_mask], 1u);
            };
            __syncthreads();  // (the keys are other threads')
#pragma unroll 2
            for (uint32_t i = 4 * tid; i < n; i += 4 * kSelThreads) {
                const uint4 k = keys_at(i);
                count(i, k.x);
                count(i + 1, k.y);
                count(i + 2, k.z);
                count(i + 3, k.w);
            }
        }
        __syncthreads();  // the histogram is complete
        uint32_t* group = s_group + pass * kGroups;
        if (tid < kBins / 4) {
            uint4* x = reinterpret_cast<uint4*>(hist) + tid;
            uint4 h = *x;
            if (pass == 0) {  // the two copies into one
                const uint4 y = x[kBins / 4];
                h = make_uint4(h.x + y.x, h.y + y.y, h.z + y.z, h.w + y.w);
                *x = h;
            }
            uint32_t sum = h.x + h.y + h.z + h.w;
#pragma unroll
            for (int d = 1; d < 8; d *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane % 8 == 0) group[tid / 8] = sum;
        }
        meet();
        // One warp finds the bin, from the top: first its group of 32, then the bin in it. So a CTA reads 384 bytes of each other's
        // memory and not 8 KB (which took 2 us a digit).
        if (warp == 0) {
            auto total = [&](const uint32_t* at) {  // over the cluster; each CTA starts with another one
                uint32_t sum = 0;
#pragma unroll
                for (int c = 0; c < kCtas; ++c) sum += kCtas > 1 ? *cluster.map_shared_rank(at, (rank + c) % kCtas) : *at;
                return sum;
            };
            auto scan = [&](uint32_t x) {
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const uint32_t o = __shfl_up_sync(0xffffffffu, x, d);
                    if (lane >= d) x += o;
                }
                return x;
            };
            const uint32_t hi = total(group + kGroups - 1 - 2 * lane), lo = total(group + kGroups - 2 - 2 * lane);
            const uint32_t incl = scan(hi + lo);
            const int at = __ffs(__ballot_sync(0xffffffffu, incl >= need)) - 1;  // there are at least `need` candidates: some lane has it
            const uint32_t upper = __shfl_sync(0xffffffffu, incl - lo, at), above = __shfl_sync(0xffffffffu, incl - lo - hi, at);
            const int picked = kGroups - 1 - 2 * at - (upper >= need ? 0 : 1);
            const uint32_t before = upper >= need ? above : upper;  // keys in the groups above
            const uint32_t mine = total(hist + 32 * picked + 31 - lane);
            const uint32_t upto = before + scan(mine);
            const int bin = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;
            if (lane == bin) {
                s_pick[0] = 32 * picked + 31 - lane;
                s_pick[1] = upto - mine;
            }
        }
        __syncthreads();
        prefix |= s_pick[0] << shift;
        need -= s_pick[1];
        // (the next write of s_pick comes behind another meeting, and each digit has a histogram of its own)
    }
    // every key above `prefix` stays, and the first `need` rows of those equal to it
    // ---- counts per warp, in order: keys above, and equal ones
    const uint32_t wb = min(n, warp * per_warp), we = min(n, wb + per_warp);
    auto tally = [&](uint32_t i, const uint4& k, uint32_t (&gt)[4], uint32_t (&eq)[4]) {
        const uint32_t key[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            gt[a] = i + a < we && key[a] > prefix;
            eq[a] = i + a < we && key[a] == prefix;
        }
    };
    uint32_t n_gt = 0, n_eq = 0;
#pragma unroll 2
    for (uint32_t i = wb + 4 * lane; i < we; i += 128) {
        uint32_t gt[4], eq[4];
        tally(i, keys_at(i), gt, eq);
        n_gt += gt[0] + gt[1] + gt[2] + gt[3];
        n_eq += eq[0] + eq[1] + eq[2] + eq[3];
    }
    n_gt = __reduce_add_sync(0xffffffffu, n_gt);
    n_eq = __reduce_add_sync(0xffffffffu, n_eq);
    if (lane == 0) {
        s_gt[warp] = n_gt;
        s_eq[warp] = n_eq;
    }
    __syncthreads();
    uint32_t gt = __reduce_add_sync(0xffffffffu, lane < warp ? s_gt[lane] : 0u);  // in front of this warp's piece
    uint32_t eq = __reduce_add_sync(0xffffffffu, lane < warp ? s_eq[lane] : 0u);
    if constexpr (kCtas > 1) {
        if (warp == kSelWarps - 1 && lane == 0) {
            s_counts[0] = gt + n_gt;
            s_counts[1] = eq + n_eq;
        }
        cluster.sync();
        uint32_t og = 0, oe = 0;
        if (lane < static_cast<int>(rank)) {
            const uint32_t* other = cluster.map_shared_rank(s_counts, lane);
            og = other[0];
            oe = other[1];
        }
        gt += __reduce_add_sync(0xffffffffu, og);
        eq += __reduce_add_sync(0xffffffffu, oe);
    }
    // ---- the kept rows, in order: row i goes to place (kept rows in front of it). Four keys a lane at a time where none equals the
    // threshold (few do, unless scores repeat), and otherwise a key a lane.
    const uint32_t below = (1u << lane) - 1u;
    auto emit = [&](uint32_t i, bool in, uint32_t key) {
        const bool is_gt = in && key > prefix, is_eq = in && key == prefix;
        const uint32_t m_gt = __ballot_sync(0xffffffffu, is_gt), m_eq = __ballot_sync(0xffffffffu, is_eq);
        uint32_t place = gt + min(eq, need) + __popc(m_gt & below);
        bool stays = is_gt;
        if (m_eq) {
            const uint32_t my_eq = eq + __popc(m_eq & below);
            place += min(my_eq, need) - min(eq, need);
            stays = is_gt || (is_eq && my_eq < need);
        }
        if (stays) kept[place] = begin + i;
        gt += __popc(m_gt);
        eq += __popc(m_eq);
    };
    const uint32_t whole = wb + (min(we, n_staged) > wb ? (min(we, n_staged) - wb) / 128 * 128 : 0u);  // full rounds of staged keys
#pragma unroll 1
    for (uint32_t i0 = wb; i0 < whole; i0 += 128) {
        const uint32_t i = i0 + 4 * lane;
        const uint4 k = *reinterpret_cast<const uint4*>(s_keys + i);
        if (__any_sync(0xffffffffu, k.x == prefix || k.y == prefix || k.z == prefix || k.w == prefix)) {
#pragma unroll
            for (int a = 0; a < 4; ++a) emit(i0 + 32 * a + lane, true, s_keys[i0 + 32 * a + lane]);
            continue;
        }
        const uint32_t mine = (k.x > prefix) + (k.y > prefix) + (k.z > prefix) + (k.w > prefix);
        uint32_t incl = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const uint32_t o = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += o;
        }
        uint32_t* to = kept + (gt + min(eq, need) + incl - mine);
        if (k.x > prefix) *to++ = begin + i;
        if (k.y > prefix) *to++ = begin + i + 1;
        if (k.z > prefix) *to++ = begin + i + 2;
        if (k.w > prefix) *to = begin + i + 3;
        gt += __shfl_sync(0xffffffffu, incl, 31);
    }
    for (uint32_t i0 = whole; i0 < we; i0 += 32) {
        const uint32_t i = i0 + lane;
        emit(i, i < we, i < n_staged ? s_keys[i] : i < we ? make_key(i, scores[i]) : 0u);
    }
    if constexpr (kCtas > 1) cluster.sync();  // no CTA leaves while another reads its counts
    if constexpr (kCopy) copy_share(p, kept, b, seg, len);
}

// ---- (2a) into another cache: grid (tiles of kept rows, sequences)
constexpr int kGatherThreads = 256;
constexpr int kTileRows = 16;
__global__ void __launch_bounds__(kGatherThreads) evict_gather_kernel(const __grid_constant__ EvictParams p) {
    extern __shared__ uint32_t s_from[];  // [n_kv_heads][kTileRows]
    const uint32_t b = blockIdx.y, j0 = blockIdx.x * kTileRows;
    const uint32_t D16 = p.head_dim / 8;  // 16-byte pieces of a head's row
    grid_dep_launch_dependents();
    grid_dep_wait();
    for (uint32_t i = threadIdx.x; i < p.n_kv_heads * kTileRows; i += kGatherThreads) {
        const uint32_t h = i / kTileRows, j = j0 + i % kTileRows;
        const size_t seg = static_cast<size_t>(b) * p.n_kv_heads + h;
        const uint32_t from = j < p.keep ? p.kept[seg * p.keep + j] : 0xffffffffu;
        s_from[i] = from;
        if (j < p.out_rows) p.scores_out[seg * p.score_out_stride + j] = from != 0xffffffffu ? p.scores[seg * p.score_stride + from] : 0.f;
    }
    __syncthreads();
    const uint32_t width = p.n_kv_heads * D16, total = kTileRows * width;
    const uint16_t* k = p.k + b * p.batch_stride;
    const uint16_t* v = p.v + b * p.batch_stride;
    uint16_t* ko = p.k_out + b * p.out_batch_stride;
    uint16_t* vo = p.v_out + b * p.out_batch_stride;
    if (blockIdx.x == 0 && threadIdx.x == 0) p.kv_len_out[b] = min(rows_of(p, b), p.keep);
    constexpr int kAhead = 4;
    for (uint32_t u0 = threadIdx.x; u0 < total; u0 += kGatherThreads * kAhead) {
        uint4 xk[kAhead], xv[kAhead];
        uint64_t to[kAhead];
        bool move[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint32_t u = u0 + a * kGatherThreads;
            const uint32_t r = u / width, c = u - r * width;
            const uint32_t from = u < total ? s_from[(c / D16) * kTileRows + r] : 0xffffffffu;
            move[a] = from != 0xffffffffu;
            to[a] = (j0 + r) * p.out_row_stride + c * 8;
            if (move[a]) {
                xk[a] = __ldcs(reinterpret_cast<const uint4*>(k + from * p.row_stride + c * 8));
                xv[a] = __ldcs(reinterpret_cast<const uint4*>(v + from * p.row_stride + c * 8));
            }
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (move[a]) {
                *reinterpret_cast<uint4*>(ko + to[a]) = xk[a];
                *reinterpret_cast<uint4*>(vo + to[a]) = xv[a];
            }
        }
    }
}

// ---- (2b) in place: grid (slices of a head's row, (sequence, kv head), K | V). Rows in rising order, a batch of them at a time:
// all loads of a batch, a barrier, its stores. A row's place is never behind the row itself and the rows rise, so a store can
// only hit rows whose loads lie in this batch or an earlier one, and the loads of later batches may be under way already.
constexpr int kMoveThreads = 512;
__global__ void __launch_bounds__(kMoveThreads) evict_compact_kernel(const __grid_constant__ EvictParams p) {
    const uint32_t seg = blockIdx.y, b = seg / p.n_kv_heads, h = seg - b * p.n_kv_heads;
    grid_dep_launch_dependents();
    grid_dep_wait();
    const uint32_t after = min(rows_of(p, b), p.keep);
    const uint32_t* kept = p.kept + static_cast<size_t>(seg) * p.keep;
    const uint32_t pieces = p.head_dim / 8 / p.slices;  // 16-byte pieces of a slice
    const uint32_t rows_at_once = kMoveThreads / pieces;
    const uint32_t my_row = threadIdx.x / pieces, my_piece = threadIdx.x - my_row * pieces;
    uint16_t* base = (blockIdx.z ? p.v_out : p.k_out) + b * p.out_batch_stride + static_cast<size_t>(h) * p.head_dim +
                     (blockIdx.x * pieces + my_piece) * 8;
    constexpr int kAhead = 4;
    const uint32_t step = rows_at_once * kAhead;
    for (uint32_t j0 = 0; j0 < after; j0 += step) {
        uint4 x[kAhead];
        bool move[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const uint32_t j = j0 + a * rows_at_once + my_row;
            move[a] = my_row < rows_at_once && j < after;
            if (move[a]) {
                const uint32_t from = kept[j];
                move[a] = from != j;  // rows in front of the first evicted one stay where they are
                if (move[a]) x[a] = *reinterpret_cast<const uint4*>(base + from * p.row_stride);
            }
        }
        __syncthreads();
#pragma unroll
        for (int a = 0; a < kAhead; ++a)
            if (move[a]) *reinterpret_cast<uint4*>(base + (j0 + a * rows_at_once + my_row) * p.out_row_stride) = x[a];
    }
    // the scores of the rows, by one CTA per (sequence, kv head), the same way
    if (blockIdx.x != 0 || blockIdx.z != 0) return;
    if (h == 0 && threadIdx.x == 0) p.kv_len_out[b] = after;
    float* s = p.scores_out + static_cast<size_t>(seg) * p.score_out_stride;
    for (uint32_t j0 = 0; j0 < after; j0 += kMoveThreads) {
        const uint32_t j = j0 + threadIdx.x;
        const float x = j < after ? s[kept[j]] : 0.f;
        __syncthreads();
        if (j < after) s[j] = x;
    }
    __syncthreads();
    for (uint32_t j = after + threadIdx.x; j < p.out_rows; j += kMoveThreads) s[j] = 0.f;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int attn_kv_evict(const AttnKvEvictArgs* a, void* stream_v) {
    if (!a || !a->k || !a->v || !a->k_out || !a->v_out || !a->scores || !a->scores_out || !a->kept || !a->kv_len_out)
        return ATTN_ERR_INVALID_ARG;
    if (a->batch == 0 || a->n_kv_heads == 0 || a->head_dim == 0 || a->rows == 0 || a->keep == 0 || a->out_rows < a->keep)
        return ATTN_ERR_INVALID_ARG;
    if (static_cast<uint64_t>(a->sink) + a->recent > a->keep) return ATTN_ERR_INVALID_ARG;  // the always-kept rows must fit
    if (a->head_dim % 8 != 0 || a->head_dim > 1024) return ATTN_ERR_UNSUPPORTED;
    const uint64_t segments = static_cast<uint64_t>(a->batch) * a->n_kv_heads;
    if (segments > 65535 || a->n_kv_heads > 256 || a->rows > 0x7fffffffu || a->out_rows > 0x7fffffffu) return ATTN_ERR_UNSUPPORTED;
    EvictParams p{};
    const uint64_t width = static_cast<uint64_t>(a->n_kv_heads) * a->head_dim;
    p.row_stride = a->kv_row_stride ? a->kv_row_stride : width;
    p.out_row_stride = a->out_row_stride ? a->out_row_stride : width;
    p.batch_stride = a->kv_batch_stride;
    p.out_batch_stride = a->out_batch_stride;
    p.score_stride = a->score_stride ? a->score_stride : a->rows;
    p.score_out_stride = a->score_out_stride ? a->score_out_stride : a->out_rows;
    if (p.row_stride < width || p.out_row_stride < width || p.score_stride < a->rows || p.score_out_stride < a->out_rows)
        return ATTN_ERR_INVALID_ARG;
    // output sequences must not share memory: one behind the other, or row by row beside each other
    if (a->batch > 1 && (p.batch_stride == 0 || (p.out_batch_stride < (a->out_rows - 1) * p.out_row_stride + width &&
                                                 (p.out_batch_stride < width || p.out_row_stride < (a->batch - 1) * p.out_batch_stride + width))))
        return ATTN_ERR_INVALID_ARG;
    if (!aligned16(a->k) || !aligned16(a->v) || !aligned16(a->k_out) || !aligned16(a->v_out) ||
        (p.row_stride | p.batch_stride | p.out_row_stride | p.out_batch_stride) % 8 != 0)
        return ATTN_ERR_ALIGNMENT;
    // In place means all three: the same caches with the same strides, and the same scores. Anything else that is written must share no
    // memory with what is read or with what else is written, but for new lengths in the place of the old ones: the CTAs run in any order.
    p.in_place = a->k == a->k_out && a->v == a->v_out && a->scores == a->scores_out;
    if (p.in_place) {
        if (p.row_stride != p.out_row_stride || p.batch_stride != p.out_batch_stride || p.score_stride != p.score_out_stride ||
            a->out_rows != a->rows)
            return ATTN_ERR_INVALID_ARG;
    }
    auto in = [&](const void* base) { return Runs{base, a->batch, 2 * p.batch_stride, a->rows, 2 * p.row_stride, 2 * width}; };
    auto out = [&](const void* base) { return Runs{base, a->batch, 2 * p.out_batch_stride, a->out_rows, 2 * p.out_row_stride, 2 * width}; };
    auto dense = [&](const void* base, uint64_t words) { return Runs{base, 1, 0, 1, 0, 4 * words}; };
    const Runs read[] = {in(a->k), in(a->v), {a->scores, segments, 4 * p.score_stride, 1, 0, 4ull * a->rows}, dense(a->kv_len, a->batch)};
    const Runs written[] = {out(a->k_out), out(a->v_out), {a->scores_out, segments, 4 * p.score_out_stride, 1, 0, 4ull * a->out_rows},
                            dense(a->kept, segments * a->keep), dense(a->kv_len_out, a->batch)};
    for (int i = 0; i < 5; ++i) {
        for (int j = 0; j < (a->kv_len ? 4 : 3); ++j) {
            const bool in_its_place = (p.in_place && i == j) || (i == 4 && j == 3 && a->kv_len_out == a->kv_len);
            if (!in_its_place && share_memory(read[j], written[i])) return ATTN_ERR_INVALID_ARG;
        }
        for (int j = 0; j < i; ++j)
            if (share_memory(written[j], written[i])) return ATTN_ERR_INVALID_ARG;
    }
    DeviceInfo dev{};
    const int rc = current_device_info(&dev);
    if (rc != ATTN_OK) return rc;
    if (dev.cc_major != 10) return ATTN_ERR_DEVICE;
    p.k = static_cast<const uint16_t*>(a->k);
    p.v = static_cast<const uint16_t*>(a->v);
    p.k_out = static_cast<uint16_t*>(a->k_out);
    p.v_out = static_cast<uint16_t*>(a->v_out);
    p.scores = a->scores;
    p.scores_out = a->scores_out;
    p.kept = a->kept;
    p.kv_len = a->kv_len;
    p.kv_len_out = a->kv_len_out;
    p.batch = a->batch;
    p.n_kv_heads = a->n_kv_heads;
    p.head_dim = a->head_dim;
    p.rows = a->rows;
    p.out_rows = a->out_rows;
    p.keep = a->keep;
    p.sink = a->sink;
    p.recent = a->recent;
    p.status = a->status;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);

    // ---- which rows: one CTA for up to 8192 rows (meeting another one costs more than 4096 rows do), eight at most
    uint32_t cl = 1;
    while (cl < 8 && a->rows > cl * 8192ull) cl *= 2;
    const uint64_t slice = (a->rows + cl - 1) / cl + 128 * kSelWarps;
    p.scores_aligned = aligned16(a->scores) && p.score_stride % 4 == 0;
    p.staged = static_cast<uint32_t>(slice < 40 * 1024 ? slice : 40 * 1024);
    // Small calls in one launch: CTAs that select for themselves and copy a share, as many as there are SMs. Measured up to 256 KB a CTA to
    // copy, 8 kv heads of 128, for two launches: 1024 rows to 256 6.2 us for 9.3, 2 x 4096 to 2048 11.0 for 15.5, 8000 to 7000 18.8
    // for 22.6. Not where the new lengths are written over the old ones, which another CTA may still have to read.
    const uint64_t shares = std::max<uint64_t>(1, std::min<uint64_t>(dev.sm_count / segments, 16));
    const bool one_launch = !p.in_place && cl == 1 && a->kv_len_out != a->kv_len && segments <= dev.sm_count &&
                            static_cast<uint64_t>(std::min(a->keep, a->rows)) * a->head_dim * 4 <= shares * kOneLaunchBytes &&
                            (kSelWords + p.staged + static_cast<uint64_t>(a->keep)) * sizeof(uint32_t) <= kOneLaunchSmem;
    auto select = [&](auto kernel) -> int {
        B200_CUDA_TRY(allow_max_smem(kernel));
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(one_launch ? static_cast<uint32_t>(shares) : cl, static_cast<uint32_t>(segments));
        cfg.blockDim = dim3(kSelThreads);
        cfg.dynamicSmemBytes = (kSelWords + p.staged + (one_launch ? a->keep : 0)) * sizeof(uint32_t);
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cl;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
        g_launch_count.fetch_add(1, std::memory_order_relaxed);
        return ATTN_OK;
    };
    if (one_launch) return select(evict_select_kernel<1, true>);
    const int selected = cl == 1   ? select(evict_select_kernel<1>)
                         : cl == 2 ? select(evict_select_kernel<2>)
                         : cl == 4 ? select(evict_select_kernel<4>)
                                   : select(evict_select_kernel<8>);
    if (selected != ATTN_OK) return selected;

    // ---- the copy
    if (p.in_place) {
        // slices of a row until the CTAs cover the GPU twice, a slice no narrower than 32 bytes
        p.slices = 1;
        while (segments * 2 * p.slices < 2ull * dev.sm_count && (p.head_dim / 8) % (p.slices * 2) == 0 && p.head_dim / 8 / (p.slices * 2) >= 2)
            p.slices *= 2;
        B200_CUDA_TRY(launch_dependent(evict_compact_kernel, dim3(p.slices, static_cast<uint32_t>(segments), 2), dim3(kMoveThreads), 0, stream, p));
    } else {
        const uint32_t tiles = (a->out_rows + kTileRows - 1) / kTileRows;
        B200_CUDA_TRY(launch_dependent(evict_gather_kernel, dim3(tiles, a->batch), dim3(kGatherThreads),
                                       a->n_kv_heads * kTileRows * sizeof(uint32_t), stream, p));
    }
    g_launch_count.fetch_add(1, std::memory_order_relaxed);
    return ATTN_OK;
}
