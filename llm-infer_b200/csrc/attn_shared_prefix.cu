// The shared prefix of a batch's decode step as a matrix product for each kv head, on the 5th-generation tensor cores
// (tcgen05 + tensor memory): all B * G query rows of a kv head against the prefix's keys, cut over the GPU along the keys.
//
// Mathematics: for every query row the softmax-normalised sum over a run of keys and its log-sum-exp; the merge pass of
// attn_shared.cu joins the runs (and the rows of the sequences' own caches) by weights exp(lse_i - LSE).
//
// One launch for both: the first p.grid CTAs take the prefix, the others two CTAs each of the split pass over the own rows
// (shared_split.cuh), which needs the same registers and half the shared memory. Two launches beside each other would need the second to
// read what earlier launches wrote without having waited for them: a launch may only wait for the one in front of it.
//
// Work: a segment is a kv head and two tiles of 128 query rows that share one K/V stream (a batch of up to 128 rows has one tile);
// a segment has ceil(P / 64) blocks of 64 keys. The blocks of all segments form one list that is dealt to one CTA per SM in equal
// contiguous runs; a CTA's part of a segment is one piece. The CTA's warps work as in the causal prefill: two softmax
// warpgroups (a thread owns a query row, which is a tensor-memory lane), one thread that feeds K and V by TMA through a ring of
// four stages, one thread that issues the MMAs, scores two blocks ahead of the products. Query rows of a kv head are not evenly
// spaced (heads of one group, then the next sequence), so the softmax warps bring them into the swizzled tile.
//
// With fp32 outputs a segment is one tile, whose keys and output columns the two softmax warpgroups share; P enters the second product in
// three parts (bf16: its 24 bits) or two (fp16: 23 bits, or 2^-32 of the row's maximum where p is small), and a block's products start
// from zero and are added up in registers.
// 64 query rows of 128 dimensions x 65536 keys, 8 kv heads: 71 us (fp16) and 79 (bf16), for 58 with outputs of 16 bits, all of it the
// further MMAs (a third block of scores in tensor memory changed nothing); errors 7e-7 and 5e-7 of the output, where sums left in tensor
// memory and two parts were off by 9e-6.
//
// Bound by the K/V stream up to 128 rows: a block takes 0.80 us of a CTA (32 KB, 0.72 us of an SM's share of HBM). With two tiles it
// takes 1.1 us, in which the special-function units are busy for 0.55 and the tensor pipe for 0.6: the chain from scores to
// probabilities of one block. A launch costs 10 us around its blocks (query rows 2, first block 2, piece and exit 4), which is why
// short prefixes stay in the split pass of attn_shared.cu. 256 query rows x 65536 keys, 8 kv heads of 128, fp16: 80 us in all
// (in the split pass: 355); 128 rows: 59 (185); 20 rows: 53 (51).
// Every wait is bounded; on expiry the role records ATTN_STATUS_WAIT_TIMEOUT, stops, and the CTA still runs its common exit.
#include <cuda.h>

#include <algorithm>

#include "shared_split.cuh"

namespace b200 {
namespace {

using namespace tc;

constexpr int BM = 128;  // query rows per tile
constexpr int BN = 64;   // keys per block
constexpr int kThreads = 384;
constexpr uint32_t kSubTileBytes = BM * 64 * 2;     // [128 query rows][64 elements], 128-byte rows, swizzled
constexpr uint32_t kTileBytes = 2 * kSubTileBytes;  // head_dim 128 (64 fills the first half)
constexpr uint32_t kKvSubBytes = BN * 64 * 2;
constexpr uint32_t kKvBytes = 2 * kKvSubBytes;
constexpr int kStages = 4;
constexpr uint32_t kTmemCols = 512;

enum {
    BAR_Q_FULL = 0,  // [tile]
    BAR_K_FULL = 2,  // [kStages]
    BAR_V_FULL = BAR_K_FULL + kStages,
    BAR_K_EMPTY = BAR_V_FULL + kStages,
    BAR_V_EMPTY = BAR_K_EMPTY + kStages,
    BAR_S_FULL = BAR_V_EMPTY + kStages,  // [tile][block parity]: scores, probabilities, products of a block
    BAR_P_FULL = BAR_S_FULL + 4,
    BAR_O_DONE = BAR_P_FULL + 4,
    BAR_O_FREE = BAR_O_DONE + 4,  // fp32 outputs: [block parity] the block's products have been added up
    BAR_COUNT = BAR_O_FREE + 2
};

constexpr uint32_t kSmemQ = 0;
constexpr uint32_t kSmemK = kSmemQ + 2 * kTileBytes;
constexpr uint32_t kSmemV = kSmemK + kStages * kKvBytes;
constexpr uint32_t kSmemStage = kSmemV + kStages * kKvBytes;  // per tile: [128 rows][128 B] output staging
constexpr uint32_t kStageTileBytes = 128 * 128;
constexpr uint32_t kSmemBars = kSmemStage + 2 * kStageTileBytes;
constexpr uint32_t kSmemTmemPtr = kSmemBars + BAR_COUNT * 8;
constexpr uint32_t kSmemAlloc = kSmemTmemPtr + 16 + 1024;  // slack to align the base to 1024 bytes
static_assert(kThreads == 2 * kSplitThreads && 2 * kSplitSmem <= kMaxDynamicSmem && kSmemAlloc <= kMaxDynamicSmem);

__device__ __forceinline__ void report_timeout(uint32_t* status) {
    if (status) atomicOr(status, ATTN_STATUS_WAIT_TIMEOUT);
}

// One CTA's part of a segment.
struct Item {
    uint32_t seg, kvh, m0, block, blocks;  // first query row; first key block and their number
    bool tile[2];
};

template <bool BF16, bool RES, int HD>
__global__ void __launch_bounds__(kThreads, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const __grid_constant__ CUtensorMap tm_o, const __grid_constant__ CUtensorMap tm_own_k, const __grid_constant__ CUtensorMap tm_own_v,
                     const __grid_constant__ SharedPrefixParams p, const __grid_constant__ SharedParams own) {
    extern __shared__ unsigned char smem_raw[];
    if (blockIdx.x >= p.grid) {  // two CTAs of the split pass, six warps each
        const int half = threadIdx.x >= kSplitThreads;
        const uint32_t cta = (blockIdx.x - p.grid) * 2 + half;
        if (cta < own.ctas)
            split_body<HD, BF16, RES>(tm_own_k, tm_own_v, tm_own_k, tm_own_v, own, smem_raw + half * p.own_smem, cta, threadIdx.x - half * kSplitThreads,
                                      2 * half);
        return;
    }
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - raw);
    const uint32_t bars = base + kSmemBars;
    auto bar = [&](int i) { return bars + 8u * i; };
    volatile uint32_t* tmem_ptr_smem = reinterpret_cast<volatile uint32_t*>(smem + kSmemTmemPtr);
    const int tid = threadIdx.x;
    const int warp = uniform_warp();
    const int lane = tid & 31;
    constexpr uint32_t kRows = RES ? BM : 2 * BM;  // query rows of a segment
    constexpr uint32_t kLoadKv = (HD / 64) * kKvSubBytes;  // bytes of a block actually loaded

    // ---- the CTA's run of the block list
    const uint32_t blocks = (p.prefix + BN - 1) / BN;
    const uint32_t query_rows = p.batch * p.group;
    const uint64_t total = static_cast<uint64_t>(p.segments) * blocks;
    uint32_t t0, t1;
    if (p.ctas_per_seg) {  // a run inside one segment
        const uint32_t seg = blockIdx.x / p.ctas_per_seg, i = blockIdx.x - seg * p.ctas_per_seg;
        t0 = seg * blocks + static_cast<uint32_t>(div_mostly_32(static_cast<uint64_t>(i) * blocks, p.ctas_per_seg));
        t1 = seg * blocks + static_cast<uint32_t>(div_mostly_32((i + 1ull) * blocks, p.ctas_per_seg));
    } else {
        t0 = static_cast<uint32_t>(div_mostly_32(blockIdx.x * total, p.grid));
        t1 = static_cast<uint32_t>(div_mostly_32((blockIdx.x + 1) * total, p.grid));
    }
    auto item_at = [&](uint32_t t, Item& w) {  // the item that starts at block t of the list; false behind the run
        if (t >= t1) return false;
        w.seg = t / blocks;
        w.block = t - w.seg * blocks;
        w.blocks = min(blocks - w.block, t1 - t);
        w.kvh = w.seg / p.pairs;
        w.m0 = (w.seg - w.kvh * p.pairs) * kRows;
        w.tile[0] = true;
        w.tile[1] = !RES && w.m0 + BM < query_rows;
        return true;
    };

    // ---- set-up: barriers, tensor memory
    if (tid == 0) {
        mbar_init(bar(BAR_Q_FULL), 128);
        mbar_init(bar(BAR_Q_FULL + 1), 128);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar(BAR_K_FULL + s), 1);
            mbar_init(bar(BAR_V_FULL + s), 1);
            mbar_init(bar(BAR_K_EMPTY + s), 1);
            mbar_init(bar(BAR_V_EMPTY + s), 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(bar(BAR_S_FULL + i), 1);
            mbar_init(bar(BAR_P_FULL + i), RES ? 256 : 128);
            mbar_init(bar(BAR_O_DONE + i), 1);
        }
        mbar_init(bar(BAR_O_FREE), 256);
        mbar_init(bar(BAR_O_FREE + 1), 256);
        mbar_init_fence();
        prefetch_tensor_map(&tm_k);
        prefetch_tensor_map(&tm_v);
        prefetch_tensor_map(&tm_o);
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_ptr_smem)), kTmemCols);
        tmem_relinquish();
    }
    grid_dep_wait();
    grid_dep_launch_dependents();
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem_base = *tmem_ptr_smem;
    auto tmem_s = [&](int t, uint32_t buf) { return tmem_base + static_cast<uint32_t>(t) * 128u + buf * 64u; };
    auto tmem_o = [&](int t) { return tmem_base + 256u + static_cast<uint32_t>(t) * 128u; };  // of a tile; fp32 outputs: of a block parity
    auto tmem_third = [&](uint32_t buf) { return tmem_base + 128u + buf * 32u; };  // fp32 outputs of bf16: the third part of P

    if (warp < 8) {
        // =============================== softmax warpgroups ===============================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");  // 256 * 208 + 128 * 88 = 384 * 168
        const int t = warp >> 2;                 // tile
        const int r = ((warp & 3) << 5) | lane;  // row inside the tile = tensor-memory lane
        const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) << 5) << 16;
        // which CTAs share each segment, for the merge pass
        for (uint32_t s = blockIdx.x * 256 + tid; s < p.segments; s += p.grid * 256)
            p.seg_ctas[s] = p.ctas_per_seg ? (s * p.ctas_per_seg) | p.ctas_per_seg << 16
                                           : segment_ctas(static_cast<uint64_t>(s) * blocks, (s + 1ull) * blocks, total, p.grid);
        const bool leader = (warp & 3) == 0 && lane == 0;
        bool ok = true;
        uint32_t g0 = 0;  // key blocks of this tile before the current item: buffer and barrier phases run on over the items
        bool staged = false;
        Item w{};
        // A warp brings its 32 query rows of an item, neighbouring lanes neighbouring 16-byte chunks (a row per thread took 2 us to
        // request); rows that are not there are zeros.
        constexpr int kRowChunks = HD / 8;
        auto chunk_at = [&](int i) {  // where chunk i of this lane goes
            const int idx = i * 32 + lane, row = ((warp & 3) << 5) + idx / kRowChunks, c = idx % kRowChunks;
            return base + kSmemQ + t * kTileBytes + row * 128 + (c >> 3) * kSubTileBytes + (((c & 7) ^ (row & 7)) << 4);
        };
        auto bring_rows = [&]() {
            uint32_t m = w.m0 + t * BM + ((warp & 3) << 5) + lane / kRowChunks;
            uint32_t b = fast_div(m, p.div_group), g = m - b * p.group;
#pragma unroll 1  // (run once or twice: every 128 bytes of straight code are a miss of the instruction cache)
            for (int i = 0; i < kRowChunks; ++i) {
                if (m < query_rows) {
                    cp_async16(chunk_at(i), static_cast<const uint16_t*>(p.q) + (static_cast<size_t>(b) * p.n_heads + w.kvh * p.group + g) * HD +
                                                lane % kRowChunks * 8);
                } else {
                    st_shared_zero16(chunk_at(i));
                }
                m += 32 / kRowChunks;
                g += 32 / kRowChunks;
                while (g >= p.group) g -= p.group, ++b;
            }
        };
        auto rows_there = [&]() {
            cp_async_wait_all();
            if (p.q_sign) {
#pragma unroll 1
                for (int i = 0; i < kRowChunks; ++i) xor_shared16(chunk_at(i), p.q_sign);
            }
            fence_async_smem();
            mbar_arrive(bar(BAR_Q_FULL + t));
        };
        // The first item's query rows are requested ahead of the tiles: behind them they came 3 us later.
        bool brought = false;
        if (item_at(t0, w) && w.tile[t]) {
            bring_rows();
            brought = true;
        }
        block_arrive(3, 288);
        if constexpr (RES) {
            // ---- fp32 outputs: the warpgroups share a tile, each takes half of a block's keys and half of O's columns. A block's products start
            // from zero and are added up here: the tensor cores cut their sums off instead of rounding them, which over hundreds of
            // instructions makes the result small by 8e-6 of it.
            constexpr int kKeys = BN / 2, kCols = HD / 2;
            const uint32_t xch = base + kSmemStage + kStageTileBytes + r * 4;  // [block parity][warpgroup][row]: the other half's maximum, or sum
            auto exchange = [&](uint32_t slot, float x) {
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(xch + (slot * 2 + t) * (BM * 4)), "f"(x) : "memory");
                named_bar_sync(4, 256);
                float y;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(y) : "r"(xch + (slot * 2 + (t ^ 1)) * (BM * 4)) : "memory");
                return y;
            };
            // (a thread that has given up waits no more but meets the others all the same: the barriers count on everybody)
            auto wait = [&](uint32_t b, uint32_t parity) {
                if (ok && !mbar_wait(b, parity)) {
                    report_timeout(p.status);
                    ok = false;
                }
            };
            for (uint32_t at = t0; item_at(at, w); at += w.blocks) {
                if (staged) {  // the memory that the last result left through is free again
                    if (leader) tma_store_wait_read();
                    named_bar_sync(4, 256);
                }
                if (t == 0) {
                    if (!brought) bring_rows();
                    brought = false;
                    rows_there();
                }
                float o[kCols];
#pragma unroll
                for (int c = 0; c < kCols; ++c) o[c] = 0.f;
                auto add_products = [&](uint32_t g, float factor) {  // of block g, which the maximum's growth makes `factor` of o
                    wait(bar(BAR_O_DONE + (g & 1)), (g >> 1) & 1);
                    fence_after();
#pragma unroll
                    for (int c = 0; c < kCols / 32; ++c) {
                        float x[32];
                        tmem_ld32(tmem_o(static_cast<int>(g & 1)) + lane_addr + t * kCols + c * 32, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[c * 32 + i] = fmaf(o[c * 32 + i], factor, x[i]);
                    }
                    fence_before();
                    mbar_arrive(bar(BAR_O_FREE + (g & 1)));
                };
                float m_used = -INFINITY, l = 0.f, last = 1.f;
#pragma unroll 1
                for (uint32_t j = 0; j < w.blocks; ++j) {
                    const uint32_t g = g0 + j, buf = g & 1;
                    const uint32_t s_tmem = tmem_s(0, buf) + lane_addr;
                    wait(bar(BAR_S_FULL + buf), (g >> 1) & 1);
                    fence_after();
                    float s[kKeys];
                    tmem_ld32(s_tmem + t * kKeys, s);
                    tmem_wait_ld();
                    const uint32_t left = p.prefix - (w.block + j) * BN;  // keys from this block on
                    if (left < BN) {
#pragma unroll
                        for (int c = 0; c < kKeys; ++c) {
                            if (t * kKeys + c >= left) s[c] = -INFINITY;
                        }
                    }
                    float mx4[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx4[i] = max3(s[i], s[4 + i], s[8 + i]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx4[i] = max3(mx4[i], s[12 + i], s[16 + i]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx4[i] = max3(mx4[i], s[20 + i], max3(s[24 + i], s[28 + i], -INFINITY));
                    float mx = max3(fmaxf(mx4[0], mx4[1]), mx4[2], mx4[3]);
                    fence_before();
                    mx = fmaxf(mx, exchange(buf, mx)) * p.scale_log2;
                    fence_after();  // both halves have been read: P may overwrite them
                    float factor = 1.f;
                    if (mx > m_used + (8.f + kLift<BF16>)) {
                        factor = fast_exp2(m_used - (mx - kLift<BF16>));
                        m_used = mx - kLift<BF16>;
                    }
                    const float m_safe = m_used == -INFINITY ? 0.f : m_used;
                    const f32x2 scale2 = pack_f32x2(p.scale_log2, p.scale_log2), m2 = pack_f32x2(-m_safe, -m_safe);
                    f32x2 sum2[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
                    uint32_t hi[16], lo[16];
                    [[maybe_unused]] uint32_t third[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float p0, p1;
                        unpack_f32x2(fma_f32x2(pack_f32x2(s[2 * i], s[2 * i + 1]), scale2, m2), p0, p1);
                        p0 = fast_exp2(p0);
                        p1 = fast_exp2(p1);
                        const f32x2 pp = pack_f32x2(p0, p1);
                        sum2[i & 1] = add_f32x2(sum2[i & 1], pp);
                        if constexpr (BF16) {  // 8 bits at a time, cut off
                            const float r0 = p0 - upper16(p0), r1 = p1 - upper16(p1);
                            hi[i] = pack_upper16(p0, p1);
                            lo[i] = pack_upper16(r0, r1);
                            third[i] = pack_upper16(r0 - upper16(r0), r1 - upper16(r1));
                        } else {
                            float h0, h1;
                            hi[i] = pack2<BF16>(p0, p1);
                            unpack2<BF16>(hi[i], h0, h1);
                            lo[i] = pack2<BF16>(p0 - h0, p1 - h1);
                        }
                    }
                    // 32 keys -> 16 packed columns of each part
                    tmem_st16(s_tmem + t * 16, hi);
                    tmem_st16(s_tmem + BN / 2 + t * 16, lo);
                    if constexpr (BF16) tmem_st16(tmem_third(buf) + lane_addr + t * 16, third);
                    float s0, s1;
                    unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
                    l = l * factor + (s0 + s1);
                    tmem_wait_st();
                    fence_before();
                    mbar_arrive(bar(BAR_P_FULL + buf));
                    if (j > 0) add_products(g - 1, last);
                    last = factor;
                }
                g0 += w.blocks;
                add_products(g0 - 1, last);
                // ---- the piece: O / l and log-sum-exp (log2 units)
                l += exchange(g0 & 1, l);
                named_bar_sync(4, 256);  // (the exchanged values have been read)
                const float inv = l == 0.f ? 0.f : 1.f / l;  // (a sum of NaN stays one)
                const uint32_t rec_row = (blockIdx.x + w.seg) * kRows;
                if (t == 0 && w.m0 + r < query_rows) p.lse[rec_row + r] = l == 0.f ? -INFINITY : (m_used + kLift<BF16>) + __log2f(l * kUnlift<BF16>);
                // through shared memory and the TMA engine, 32 columns at a time: the second query tile and the staging tiles are free
#pragma unroll
                for (int pass = 0; pass < kCols / 32; ++pass) {
                    const uint32_t stage = t == 0 ? base + kSmemQ + kTileBytes + pass * kSubTileBytes : base + kSmemStage + pass * kStageTileBytes;
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(stage + r * 128 + ((c ^ (r & 7)) << 4)),
                                     "r"(__float_as_uint(o[pass * 32 + c * 4] * inv)), "r"(__float_as_uint(o[pass * 32 + c * 4 + 1] * inv)),
                                     "r"(__float_as_uint(o[pass * 32 + c * 4 + 2] * inv)), "r"(__float_as_uint(o[pass * 32 + c * 4 + 3] * inv))
                                     : "memory");
                }
                fence_async_smem();
                named_bar_sync(1 + t, 128);
                if (leader) {
#pragma unroll
                    for (int pass = 0; pass < kCols / 32; ++pass)
                        tma_store_2d(&tm_o, t == 0 ? base + kSmemQ + kTileBytes + pass * kSubTileBytes : base + kSmemStage + pass * kStageTileBytes,
                                     t * kCols + pass * 32, rec_row);
                    tma_store_commit();
                }
                staged = true;
            }
        } else {
            for (uint32_t at = t0; ok && item_at(at, w); at += w.blocks) {
                if (!w.tile[t]) continue;
                // ---- the query rows into the tile (the previous item's MMAs are over, its result has left)
                const uint32_t m = w.m0 + t * BM + r;
                if (staged) {
                    if (leader) tma_store_wait_read();
                    named_bar_sync(1 + t, 128);
                }
                if (!brought) bring_rows();
                brought = false;
                rows_there();
                float m_used = -INFINITY;  // what the stored probabilities are relative to (log2 units): a maximum less the lift
                float l = 0.f;
                for (uint32_t j = 0; j < w.blocks && ok; ++j) {
                    const uint32_t g = g0 + j, buf = g & 1, par = (g >> 1) & 1;
                    const uint32_t s_tmem = tmem_s(t, buf) + lane_addr;
                    if (!mbar_wait(bar(BAR_S_FULL + 2 * t + buf), par)) { report_timeout(p.status); ok = false; break; }
                    fence_after();
                    float s[BN];
#pragma unroll
                    for (int c = 0; c < BN / 32; ++c) tmem_ld32(s_tmem + c * 32, *reinterpret_cast<float(*)[32]>(&s[c * 32]));
                    tmem_wait_ld();
                    const uint32_t left = p.prefix - (w.block + j) * BN;  // keys from this block on
                    if (left < BN) {
#pragma unroll
                        for (int c = 0; c < BN; ++c) {
                            if (c >= left) s[c] = -INFINITY;
                        }
                    }
                    // four independent chains of three-input maxima
                    float mx4[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) mx4[i] = max3(s[i], s[4 + i], s[8 + i]);
#pragma unroll
                    for (int c = 12; c + 8 <= BN; c += 8) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) mx4[i] = max3(mx4[i], s[c + i], s[c + 4 + i]);
                    }
                    float mx = max3(fmaxf(mx4[0], mx4[1]), mx4[2], mx4[3]);
#pragma unroll
                    for (int c = 12 + (BN - 12) / 8 * 8; c < BN; ++c) mx = fmaxf(mx, s[c]);
                    mx *= p.scale_log2;
                    // Rescale only when the maximum grew by more than 8 (probabilities stay below 2^8, with fp16's lift 2^15).
                    float factor = 1.f;
                    if (mx > m_used + (8.f + kLift<BF16>)) {
                        factor = fast_exp2(m_used - (mx - kLift<BF16>));  // 0 on the first block (m_used = -inf)
                        m_used = mx - kLift<BF16>;
                    }
                    if (g >= 2 && !mbar_wait(bar(BAR_O_DONE + 2 * t + buf), par ^ 1)) { report_timeout(p.status); ok = false; break; }
                    if (j > 0 && __any_sync(0xffffffffu, factor != 1.f)) {
                        if (!mbar_wait(bar(BAR_O_DONE + 2 * t + (buf ^ 1)), ((g - 1) >> 1) & 1)) { report_timeout(p.status); ok = false; break; }
                        fence_after();
#pragma unroll
                        for (int c = 0; c < HD / 32; ++c) {
                            float o[32];
                            tmem_ld32(tmem_o(t) + lane_addr + c * 32, o);
                            tmem_wait_ld();
                            uint32_t u[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(o[i] * factor);
                            tmem_st32(tmem_o(t) + lane_addr + c * 32, u);
                        }
                    }
                    l *= factor;
                    // probabilities; P overwrites S in place
                    const float m_safe = m_used == -INFINITY ? 0.f : m_used;
                    const f32x2 scale2 = pack_f32x2(p.scale_log2, p.scale_log2), m2 = pack_f32x2(-m_safe, -m_safe);
                    f32x2 sum2[2] = {pack_f32x2(0.f, 0.f), pack_f32x2(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < BN / 32; ++c) {
                        uint32_t hi[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float p0, p1;
                            unpack_f32x2(fma_f32x2(pack_f32x2(s[c * 32 + 2 * i], s[c * 32 + 2 * i + 1]), scale2, m2), p0, p1);
                            p0 = fast_exp2(p0);
                            p1 = fast_exp2(p1);
                            const f32x2 pp = pack_f32x2(p0, p1);
                            sum2[i & 1] = add_f32x2(sum2[i & 1], pp);
                            hi[i] = pack2<BF16>(p0, p1);
                        }
                        tmem_st16(s_tmem + c * 16, hi);  // 32 keys -> 16 packed columns
                    }
                    float s0, s1;
                    unpack_f32x2(add_f32x2(sum2[0], sum2[1]), s0, s1);
                    l += s0 + s1;
                    tmem_wait_st();
                    fence_before();
                    mbar_arrive(bar(BAR_P_FULL + 2 * t + buf));
                }
                g0 += w.blocks;
                if (!ok) break;
                // ---- the piece: O / l and log-sum-exp (log2 units)
                if (!mbar_wait(bar(BAR_O_DONE + 2 * t + ((g0 - 1) & 1)), ((g0 - 1) >> 1) & 1)) {
                    report_timeout(p.status);
                    ok = false;
                    break;
                }
                fence_after();
                const float inv = l == 0.f ? 0.f : 1.f / l;  // (a sum of NaN stays one)
                const uint32_t rec_row = (blockIdx.x + w.seg) * kRows + t * BM;
                if (m < query_rows) p.lse[rec_row + r] = l == 0.f ? -INFINITY : (m_used + kLift<BF16>) + __log2f(l * kUnlift<BF16>);
                // The tile leaves through shared memory and the TMA engine, 128 bytes of every row at a time: the query tile, which nothing
                // reads any more, holds the first two passes, the staging tile the third, so that only the fourth waits for a store. (Each pass
                // behind the previous one's store in a single staging tile: 3 us more per piece.)
                auto put = [&](int pass, uint32_t stage) {
                    float o[32];
                    tmem_ld32(tmem_o(t) + lane_addr + pass * 32, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(stage + r * 128 + ((c ^ (r & 7)) << 4)),
                                     "r"(__float_as_uint(o[c * 4] * inv)), "r"(__float_as_uint(o[c * 4 + 1] * inv)),
                                     "r"(__float_as_uint(o[c * 4 + 2] * inv)), "r"(__float_as_uint(o[c * 4 + 3] * inv))
                                     : "memory");
                };
                constexpr int kPasses = HD / 32;
#pragma unroll 1
                for (int pass = 0; pass < kPasses; ++pass) {
                    const uint32_t stage = pass == 2   ? base + kSmemStage + t * kStageTileBytes
                                           : pass == 1 ? base + kSmemQ + t * kTileBytes + kSubTileBytes
                                                       : base + kSmemQ + t * kTileBytes;
                    if (pass == 3) {  // the first pass's store has been read
                        if (leader) asm volatile("cp.async.bulk.wait_group.read 2;" ::: "memory");
                        named_bar_sync(1 + t, 128);
                    }
                    put(pass, stage);
                    fence_async_smem();
                    named_bar_sync(1 + t, 128);
                    if (leader) {
                        tma_store_2d(&tm_o, stage, pass * 32, rec_row);
                        tma_store_commit();
                    }
                }
                staged = true;
                fence_before();  // the next item's first product overwrites O; its P_FULL arrival orders it behind these loads
            }
        }
        if (leader) tma_store_wait_all();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 8) block_wait(3, 288);
        if (warp == 8 && elect_one()) {
            // =============================== TMA producer ===============================
            uint32_t st = 0, phase = 0, it = 0;
            bool ok = true, key_ahead = false;  // key_ahead: the stage's K is under way, its V is not
            Item w;
            for (uint32_t at = t0; ok && item_at(at, w); at += w.blocks) {
                for (uint32_t j = 0; j < w.blocks; ++j, ++it) {
                    const int row = static_cast<int>((w.block + j) * BN), head = static_cast<int>(w.kvh);
                    if (it >= kStages && !mbar_wait(bar(BAR_K_EMPTY + st), phase ^ 1)) { ok = false; break; }
                    const uint32_t kdst = base + kSmemK + st * kKvBytes;
                    mbar_arrive_expect_tx(bar(BAR_K_FULL + st), kLoadKv);
                    tma_load_3d(kdst, &tm_k, bar(BAR_K_FULL + st), 0, row, head);
                    if (HD > 64) tma_load_3d(kdst + kKvSubBytes, &tm_k, bar(BAR_K_FULL + st), 64, row, head);
                    if (it >= kStages && !mbar_wait(bar(BAR_V_EMPTY + st), phase ^ 1)) { ok = false; key_ahead = true; break; }
                    const uint32_t vdst = base + kSmemV + st * kKvBytes;
                    mbar_arrive_expect_tx(bar(BAR_V_FULL + st), kLoadKv);
                    tma_load_3d(vdst, &tm_v, bar(BAR_V_FULL + st), 0, row, head);
                    if (HD > 64) tma_load_3d(vdst + kKvSubBytes, &tm_v, bar(BAR_V_FULL + st), 64, row, head);
                    if (++st == kStages) st = 0, phase ^= 1;
                }
            }
            if (!ok) {  // report, and leave no copy in flight into this CTA's memory
                report_timeout(p.status);
                for (uint32_t s = 0; s < kStages; ++s) {
                    const uint32_t v_phase = s < st ? phase : phase ^ 1, k_phase = s == st && key_ahead ? phase : v_phase;
                    (void)mbar_wait(bar(BAR_K_FULL + s), k_phase);
                    (void)mbar_wait(bar(BAR_V_FULL + s), v_phase);
                }
            }
        } else if (warp == 9 && elect_one()) {
            // =============================== MMA issuer ===============================
            constexpr uint32_t fmt = BF16 ? 1u : 0u;
            constexpr uint32_t idesc_qk = instr_desc(fmt, fmt, 0, BM, BN);  // S: 128 rows x 64 keys
            constexpr uint32_t idesc_pv = instr_desc(fmt, fmt, 1, BM, HD);  // O: 128 rows x head_dim
            const uint64_t q_desc = smem_desc(base + kSmemQ, 16, 1024), k_desc = smem_desc(base + kSmemK, 16, 1024);
            const uint64_t v_desc = smem_desc(base + kSmemV, kKvSubBytes, 1024);
            uint32_t g0[2] = {0, 0};  // key blocks of each tile before the current item
            uint32_t items[2] = {0, 0};
            auto issue_qk = [&](int t, uint32_t j, uint32_t st) {
                const uint32_t buf = (g0[t] + j) & 1;
                const uint64_t qa = q_desc + t * (kTileBytes / 16), ka = k_desc + st * (kKvBytes / 16);
                const uint32_t d = tmem_s(t, buf);
#pragma unroll
                for (int kc = 0; kc < HD / 16; ++kc)
                    mma_ss(d, qa + (kc >> 2) * (kSubTileBytes / 16) + (kc & 3) * 2, ka + (kc >> 2) * (kKvSubBytes / 16) + (kc & 3) * 2,
                           idesc_qk, kc > 0);
                commit(bar(BAR_S_FULL + 2 * t + buf));
            };
            auto issue_pv = [&](int t, uint32_t j, uint32_t st) {
                const uint32_t buf = (g0[t] + j) & 1;
                const uint64_t va = v_desc + st * (kKvBytes / 16);
                const uint32_t pa = tmem_s(t, buf);
                if constexpr (RES) {  // from zero, the small parts first
                    const uint32_t d = tmem_o(static_cast<int>(buf));
#pragma unroll
                    for (int kc = 0; kc < BN / 16 && BF16; ++kc) mma_ts(d, tmem_third(buf) + kc * 8, va + kc * 128, idesc_pv, kc > 0);
#pragma unroll
                    for (int kc = 0; kc < BN / 16; ++kc) mma_ts(d, pa + BN / 2 + kc * 8, va + kc * 128, idesc_pv, BF16 || kc > 0);
#pragma unroll
                    for (int kc = 0; kc < BN / 16; ++kc) mma_ts(d, pa + kc * 8, va + kc * 128, idesc_pv, 1);
                } else {
#pragma unroll
                    for (int kc = 0; kc < BN / 16; ++kc) mma_ts(tmem_o(t), pa + kc * 8, va + kc * 128, idesc_pv, j > 0 || kc > 0);
                }
                commit(bar(BAR_O_DONE + 2 * t + buf));
            };
            bool ok = true;
            uint32_t st = 0, phase = 0, kst = 0, kphase = 0;  // ring position of the next V block, of the next K block
            auto next_k = [&]() {
                if (++kst == kStages) kst = 0, kphase ^= 1;
            };
            Item w;
            for (uint32_t at = t0; ok && item_at(at, w); at += w.blocks) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (ok && w.tile[t]) {
                        ok = mbar_wait(bar(BAR_Q_FULL + t), items[t] & 1);
                        ++items[t];
                    }
                for (uint32_t j = 0; j < 2 && j < w.blocks && ok; ++j) {
                    ok = mbar_wait(bar(BAR_K_FULL + kst), kphase);
                    if (!ok) break;
                    fence_after();
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        if (w.tile[t]) issue_qk(t, j, kst);
                    commit(bar(BAR_K_EMPTY + kst));
                    next_k();
                }
                for (uint32_t j = 0; j < w.blocks && ok; ++j) {
                    if (!mbar_wait(bar(BAR_V_FULL + st), phase)) { ok = false; break; }
                    const bool more = j + 2 < w.blocks;
                    bool k_ready = false;
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (!ok || !w.tile[t]) continue;
                        const uint32_t g = g0[t] + j;
                        if (!mbar_wait(bar(BAR_P_FULL + 2 * t + (g & 1)), (g >> 1) & 1)) { ok = false; break; }
                        if (RES && g >= 2 && !mbar_wait(bar(BAR_O_FREE + (g & 1)), ((g >> 1) & 1) ^ 1)) { ok = false; break; }
                        fence_after();
                        issue_pv(t, j, st);
                        if (more) {
                            if (!k_ready) {
                                if (!mbar_wait(bar(BAR_K_FULL + kst), kphase)) { ok = false; break; }
                                fence_after();
                                k_ready = true;
                            }
                            issue_qk(t, j + 2, kst);
                        }
                    }
                    if (!ok) break;
                    commit(bar(BAR_V_EMPTY + st));
                    if (++st == kStages) st = 0, phase ^= 1;
                    if (more) {
                        commit(bar(BAR_K_EMPTY + kst));
                        next_k();
                    }
                }
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (w.tile[t]) g0[t] += w.blocks;
            }
            if (!ok) report_timeout(p.status);
        }
    }

    // ---- common exit: everybody meets, then the allocating warp releases tensor memory
    fence_before();
    __syncthreads();
    if (warp == 8) {
        fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

int encode(CUtensorMap* map, CUtensorMapDataType type, uint32_t rank, const void* ptr, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return ATTN_ERR_CUDA;
    const cuuint32_t unit[3] = {1, 1, 1};
    const CUresult r = enc(map, type, rank, const_cast<void*>(ptr), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r == CUDA_SUCCESS) return ATTN_OK;
    g_last_cuda_error = static_cast<int>(r);
    return ATTN_ERR_CUDA;
}

}  // namespace

int launch_shared_prefix(const SharedPrefixParams& prefix, const SharedParams& own, const CUtensorMap& tm_own_k, const CUtensorMap& tm_own_v, size_t own_smem,
                         cudaStream_t stream) {
    SharedPrefixParams p = prefix;
    p.own_smem = static_cast<uint32_t>((own_smem + 15) / 16 * 16);
    const size_t smem = std::max<size_t>(kSmemAlloc, 2 * static_cast<size_t>(p.own_smem));
    const uint32_t grid = p.grid + (own.ctas + 1) / 2;
    const CUtensorMapDataType type = p.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    // K, V [row][kv head][head_dim] as (dim, row, head): blocks of 64 elements x 64 rows of one head; rows behind the end read as zeros
    const cuuint64_t kv_dims[3] = {p.head_dim, p.prefix, p.n_kv_heads};
    const cuuint64_t kv_strides[2] = {p.row_stride * 2, p.head_dim * 2ull};
    const cuuint32_t kv_box[3] = {64, BN, 1};
    // pieces [records * 256 or 128 rows][head_dim] fp32, stored 32 columns x 128 rows at a time
    const cuuint64_t o_dims[2] = {p.head_dim, (static_cast<cuuint64_t>(p.grid) + p.segments) * (p.residual ? BM : 2 * BM)};
    const cuuint64_t o_strides[1] = {p.head_dim * 4ull};
    const cuuint32_t o_box[2] = {32, BM};
    CUtensorMap tm_k, tm_v, tm_o;
    int rc;
    if ((rc = encode(&tm_k, type, 3, p.k, kv_dims, kv_strides, kv_box)) != ATTN_OK) return rc;
    if ((rc = encode(&tm_v, type, 3, p.v, kv_dims, kv_strides, kv_box)) != ATTN_OK) return rc;
    if ((rc = encode(&tm_o, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, p.part, o_dims, o_strides, o_box)) != ATTN_OK) return rc;
    auto launch = [&](auto kernel) -> int {
        B200_CUDA_TRY(allow_max_smem(kernel));
        B200_CUDA_TRY(launch_dependent(kernel, dim3(grid), dim3(kThreads), smem, stream, tm_k, tm_v, tm_o, tm_own_k, tm_own_v, p, own));
        g_launch_count.fetch_add(1, std::memory_order_relaxed);
        return ATTN_OK;
    };
    if (p.head_dim == 128) {
        if (p.bf16) return p.residual ? launch(shared_prefix_kernel<true, true, 128>) : launch(shared_prefix_kernel<true, false, 128>);
        return p.residual ? launch(shared_prefix_kernel<false, true, 128>) : launch(shared_prefix_kernel<false, false, 128>);
    }
    if (p.bf16) return p.residual ? launch(shared_prefix_kernel<true, true, 64>) : launch(shared_prefix_kernel<true, false, 64>);
    return p.residual ? launch(shared_prefix_kernel<false, true, 64>) : launch(shared_prefix_kernel<false, false, 64>);
}

}  // namespace b200
