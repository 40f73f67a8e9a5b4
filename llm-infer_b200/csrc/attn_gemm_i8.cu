// Product of 8-bit integers with a scale per token and per channel, on the 5th-generation tensor cores (kind::i8):
//
//     out[t][j] = a_scale[t] * w_scale[j] * sum_i a[t][i] * w[j][i]        t < m tokens, j < n_out channels, i < k
//
// The sum is exact: products of 8 bits, added in 32 (k up to 131071 keeps any sum below 2^31), so cutting k into slices and adding
// them in any order gives the same bits. Weights are the M side of the MMA: a tensor-memory lane is a channel, which has its scale in
// a register, and a warp stores 32 neighbouring channels of a token at a time.
//
// What bounds it: with few tokens the weights' way from memory (8 x 4096 x 128256 79 us = 6.7 TB/s, 8 x 4096 x 28672 20.4 - 20.9 us = 5.6 - 5.8 TB/s) and, where
// they are few, some 4 us from a launch to its first and from its last tile (1 x 4096 x 6144 7.5 us in a graph for 3.8 of reading);
// with many tokens the tensor cores (9184 x 4096 x 28672 with SwiGLU 634 - 654 us = 3.3 - 3.4 POP/s in a burst, twice the measured bf16
// rate; in a long loop the 1000 W cap holds it at 2.8 - 2.9 POP/s and 1.24 - 1.26 GHz, where the pipe does 93 - 95 % of what it can).
#include <algorithm>
#include <type_traits>

#include "attn_internal.cuh"
#include "operand_memory.cuh"
#include "tcgen05_sm100.cuh"
#include "tma_tile.cuh"

namespace b200 {
namespace {

using namespace tc;

constexpr uint32_t kRowsM = 128;   // channels of a weight tile
constexpr uint32_t kStepK = 128;   // bytes (= elements) of k per stage: a 128-byte swizzle row
constexpr uint32_t kWTile = kRowsM * kStepK;  // 16 KB
constexpr uint32_t kMaxK = 131071;

struct GemmI8Params {
    void* out;
    const float* a_scale;
    const float* w_scale;
    uint64_t ldc;
    uint32_t m, n_out;     // n_out: columns of the result (swiglu: half of the weight rows)
    uint32_t k_steps;
    uint32_t stages;
    int32_t out_dtype;
    uint32_t w_early;
    uint32_t* status;
};

// Instruction descriptor of kind::i8: signed 8-bit A and B, both K-major, 32-bit integer accumulators, M x N = m x n.
__host__ __device__ constexpr uint32_t instr_desc_i8(uint32_t m, uint32_t n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// D(tmem) (+)= A(smem) * B(smem), 32 values of k
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}
// The same over a pair of CTAs: A rows 0-127 and half of B's rows in the leader's shared memory, the others at the same offsets in
// its partner.
__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(acc)
        : "memory");
}
// 16 columns of this thread's tensor-memory lane.
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t (&r)[16]) {
    tmem_ld16(taddr, reinterpret_cast<float(&)[16]>(r));
}
// The wait for this thread's tensor-memory loads, tied to the registers they fill: arithmetic on them stays behind it.
__device__ __forceinline__ void wait_ld(uint32_t (&r)[16]) {
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(r[i]));
}

__device__ __forceinline__ int4 ld_cluster_i4(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}

// x / (1 + e^-x), and x e^x / (1 + e^x) of negative x: the divisor is 1 to 2 whatever x is, so that the quick quotient, which gives 0 where
// it passes 2^126, holds for every gate (for one of -88 too, whose 5e-37 a large up value brings back). expf is good to two units in the
// last place, the quotient to two more; the exact quotient takes a branch, behind which nothing of the next value was begun: 7292 x 256 x
// 1536 30.9 -> 17.9 us. (The product with e and the choice cost that shape 13.6 -> 14.1 us now, a longer k nothing.)
__device__ __forceinline__ float silu(float x) {
    const float e = expf(-fabsf(x));
    return __fdividef(x < 0.f ? x * e : x, 1.0f + e);
}
// the scaled sum; the order of the two products is part of the result's bits
__device__ __forceinline__ float scaled(int32_t sum, float w_scale, float a_scale) {
    return __fmul_rn(__fmul_rn(static_cast<float>(sum), w_scale), a_scale);
}
// The same of a channel's 16 tokens, two at a time; a_scale on a 16-byte boundary.
__device__ __forceinline__ void scaled16(float (&y)[16], const uint32_t (&sum)[16], float w_scale, const float* a_scale) {
    const f32x2 w2 = pack_f32x2(w_scale, w_scale);
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const float4 a = *reinterpret_cast<const float4*>(a_scale + i);
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const f32x2 s = pack_f32x2(static_cast<float>(static_cast<int32_t>(sum[i + e])), static_cast<float>(static_cast<int32_t>(sum[i + e + 1])));
            unpack_f32x2(mul_f32x2(mul_f32x2(s, w2), e ? pack_f32x2(a.z, a.w) : pack_f32x2(a.x, a.y)), y[i + e], y[i + e + 1]);
        }
    }
}
template <typename T>
__device__ __forceinline__ T to_out(float x);
template <>
__device__ __forceinline__ float to_out<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half to_out<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 to_out<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
// A channel's values of N tokens, of which there are `left`. Returns where the next token goes. (An address from the one before: with a
// 64-bit product for each, 7292 x 256 x 1536 took 16.8 us for 12.0.)
template <typename T, int N>
__device__ __forceinline__ T* store_tokens(T* dst, uint64_t ldc, const float (&y)[N], uint32_t left) {
    if (left >= N) {
#pragma unroll
        for (int i = 0; i < N; ++i, dst += ldc) *dst = to_out<T>(y[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i, dst += ldc)
            if (i < left) *dst = to_out<T>(y[i]);
    }
    return dst;
}
// f with a value of the output's type
template <typename F>
__device__ __forceinline__ void with_out_type(int32_t dtype, F f) {
    if (dtype == ATTN_DTYPE_F32) f(float{});
    else if (dtype == ATTN_DTYPE_F16) f(__half{});
    else f(__nv_bfloat16{});
}

// ---- few tokens: the weights pass by once ---------------------------------------------------------------------------
// A cluster of CTAs shares one tile of PARTS x 128 channels x N tokens; each CTA takes a slice of k, and the slices' sums meet in
// shared memory over the cluster. Four warps: warp 0 requests the tiles by TMA, warp 1 issues the MMAs, all of them finish the tile.
enum { S_FULL = 0, kStreamMaxStages = 12, S_EMPTY = S_FULL + kStreamMaxStages, S_ACC = S_EMPTY + kStreamMaxStages, S_BARS };
constexpr int kStreamThreads = 128;
constexpr uint32_t kMaxSlices = 8;  // CTAs of a cluster

template <int PARTS, int N>
constexpr uint32_t stream_stage_bytes() { return PARTS * kWTile + N * kStepK; }
constexpr uint32_t kStreamTail = 1024 + 256 + 512;  // alignment of the base; barriers and tensor-memory address; tokens' scales

template <int PARTS, int N>
__global__ void __launch_bounds__(kStreamThreads)
gemm_i8_stream_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a,
                      const __grid_constant__ GemmI8Params p) {
    constexpr uint32_t kStageBytes = stream_stage_bytes<PARTS, N>();
    constexpr uint32_t kCols = PARTS * N < 32 ? 32 : PARTS * N;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;  // swizzled tiles want 1024-byte alignment
    unsigned char* smem = smem_raw + (base - raw);
    const uint32_t bars = base + p.stages * kStageBytes;
    auto bar = [&](int i) { return bars + 8u * i; };
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(smem + p.stages * kStageBytes + S_BARS * 8);
    float* s_scale = reinterpret_cast<float*>(smem + p.stages * kStageBytes + 256);

    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const uint32_t slices = gridDim.x, slice = blockIdx.x;  // the cluster is the grid's x
    const uint32_t tok0 = blockIdx.y * N, row0 = blockIdx.z * kRowsM;
    const uint32_t ks0 = static_cast<uint32_t>(static_cast<uint64_t>(p.k_steps) * slice / slices);
    const uint32_t ks1 = static_cast<uint32_t>(static_cast<uint64_t>(p.k_steps) * (slice + 1) / slices);

    auto gave_up = [&]() {
        if (p.status) atomicOr(p.status, ATTN_STATUS_WAIT_TIMEOUT);
    };
    // a stage's bytes are announced, its weights requested
    auto load_w = [&](uint32_t ks, uint32_t s) {
        mbar_arrive_expect_tx(bar(S_FULL + s), kStageBytes);
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
            tma_load_2d(base + s * kStageBytes + part * kWTile, &tm_w, bar(S_FULL + s), static_cast<int>(ks * kStepK),
                        static_cast<int>(row0 + part * p.n_out));
    };
    const uint32_t early = p.w_early ? min(ks1 - ks0, p.stages) : 0u;
    if (warp == 0) {
        if (elect_one()) {
            prefetch_tensor_map(&tm_w);
            prefetch_tensor_map(&tm_a);
            for (uint32_t s = 0; s < p.stages; ++s) {
                mbar_init(bar(S_FULL + s), 1);
                mbar_init(bar(S_EMPTY + s), 1);
            }
            mbar_init(bar(S_ACC), 1);
            mbar_init_fence();
            // While the previous kernel of the stream may still be running: the first weights come as far as L2. (What that kernel
            // writes to them still arrives: L2 is where both meet.) With w_early they go into the ring.
            for (uint32_t i = 0; i < min(ks1 - ks0, p.stages); ++i) {
                if (p.w_early) {
                    load_w(ks0 + i, i);
                } else {
#pragma unroll
                    for (int part = 0; part < PARTS; ++part)
                        tma_prefetch_2d(&tm_w, static_cast<int>((ks0 + i) * kStepK), static_cast<int>(row0 + part * p.n_out));
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(s_tmem)), kCols);
        tmem_relinquish();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *s_tmem;

    grid_dep_launch_dependents();
    grid_dep_wait();

    // Channels of this thread: one, its tensor-memory lane; where slices' sums meet, four neighbouring ones.
    const bool meet = slices > 1;
    const uint32_t col = row0 + (meet ? 4 * lane : tid), width = meet ? 4 : 1;
    float ws[PARTS][4];
#pragma unroll
    for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int i = 0; i < 4; ++i) ws[part][i] = i < width && col + i < p.n_out ? p.w_scale[part * p.n_out + col + i] : 0.f;
    if (warp >= 2)  // (warp 0 has tiles to request)
        for (uint32_t t = tid - 64; t < N; t += 64) s_scale[t] = tok0 + t < p.m ? p.a_scale[tok0 + t] : 0.f;

    if (warp == 0) {
        if (elect_one()) {
            uint32_t s = 0, phase = 0, issued = 0;
            for (uint32_t ks = ks0; ks < ks1; ++ks, ++issued) {
                if (issued >= p.stages && !mbar_wait(bar(S_EMPTY + s), phase ^ 1)) {
                    gave_up();
                    break;
                }
                if (issued >= early) load_w(ks, s);
                tma_load_2d(base + s * kStageBytes + PARTS * kWTile, &tm_a, bar(S_FULL + s), static_cast<int>(ks * kStepK), static_cast<int>(tok0));
                if (++s == p.stages) s = 0, phase ^= 1;
            }
            // no copy is in flight when the block ends, whatever became of the MMAs
            for (uint32_t i = issued > p.stages ? issued - p.stages : 0; i < issued; ++i)
                mbar_wait(bar(S_FULL + i % p.stages), i / p.stages & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t idesc = instr_desc_i8(kRowsM, N);
            const uint64_t desc0 = smem_desc(base, 16, 1024);
            uint32_t s = 0, phase = 0;
            for (uint32_t ks = ks0; ks < ks1; ++ks) {
                if (!mbar_wait(bar(S_FULL + s), phase)) {
                    gave_up();
                    break;
                }
                fence_after();
                // K-major operands, 128-byte swizzle: 32 bytes per k-step of 32, 8-row groups 1024 bytes apart
                const uint64_t w = desc0 + s * (kStageBytes / 16), a = w + PARTS * (kWTile / 16);
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
                    for (int part = 0; part < PARTS; ++part)
                        mma_i8(tmem + part * N, w + part * (kWTile / 16) + 2 * kk, a + 2 * kk, idesc, (ks - ks0) | kk);
                }
                commit(bar(S_EMPTY + s));
                if (++s == p.stages) s = 0, phase ^= 1;
            }
            commit(bar(S_ACC));
        }
        __syncwarp();
    }
    // (a vote, so that a warp reads tensor memory as one)
    if (!__all_sync(0xffffffffu, mbar_wait(bar(S_ACC), 0)) && lane == 0) gave_up();
    fence_after();
    __syncthreads();  // the tokens' scales; the copies of a block that gave up

    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const uint32_t tokens = min(static_cast<uint32_t>(N), p.m - tok0);
    auto value = [&](uint32_t t, int i, int32_t s0, int32_t s1) {
        float y = scaled(s0, ws[0][i], s_scale[t]);
        if constexpr (PARTS == 2) y = __fmul_rn(silu(y), scaled(s1, ws[1][i], s_scale[t]));
        return y;
    };
    auto finish_slices = [&](auto type, auto count) {
        using T = decltype(type);
        constexpr uint32_t S = decltype(count)::value, kAtOnce = kMaxSlices / S;
        for (uint32_t t0 = slice + S * kAtOnce * warp; t0 < tokens; t0 += S * kAtOnce * 4) {
            int32_t sum[kAtOnce][PARTS][4];
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                int4 v[kAtOnce][S];
#pragma unroll
                for (uint32_t u = 0; u < kAtOnce; ++u) {
                    const uint32_t t = min(t0 + S * u, N - 1u);
#pragma unroll
                    for (uint32_t r = 0; r < S; ++r) v[u][r] = ld_cluster_i4(cluster_address(base + ((part * N + t) * kRowsM + 4 * lane) * 4, r));
                }
#pragma unroll
                for (uint32_t u = 0; u < kAtOnce; ++u) {
#pragma unroll
                    for (uint32_t r = 1; r < S; ++r)
                        v[u][0].x += v[u][r].x, v[u][0].y += v[u][r].y, v[u][0].z += v[u][r].z, v[u][0].w += v[u][r].w;
                    sum[u][part][0] = v[u][0].x, sum[u][part][1] = v[u][0].y, sum[u][part][2] = v[u][0].z, sum[u][part][3] = v[u][0].w;
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < kAtOnce; ++u) {
                const uint32_t t = t0 + S * u;
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = value(min(t, N - 1u), i, sum[u][0][i], sum[u][PARTS - 1][i]);
                T* dst = static_cast<T*>(p.out) + static_cast<size_t>(tok0 + t) * p.ldc + col;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t < tokens && col + i < p.n_out) dst[i] = to_out<T>(y[i]);
            }
        }
    };
    if (!meet) {
        with_out_type(p.out_dtype, [&](auto type) {
            using T = decltype(type);
            T* dst = static_cast<T*>(p.out) + static_cast<size_t>(tok0) * p.ldc + col;
#pragma unroll 1
            for (uint32_t c = 0; c < tokens; c += 16) {
                uint32_t r[PARTS][16];
#pragma unroll
                for (int part = 0; part < PARTS; ++part) ld16(lane_addr + part * N + c, r[part]);
#pragma unroll
                for (int part = 0; part < PARTS; ++part) wait_ld(r[part]);
                float y[16];
                scaled16(y, r[0], ws[0][0], s_scale + c);
                if constexpr (PARTS == 2) {
                    float up[16];
                    scaled16(up, r[1], ws[1][0], s_scale + c);
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[i] = __fmul_rn(silu(y[i]), up[i]);
                }
                dst = store_tokens(dst, p.ldc, y, col < p.n_out ? tokens - c : 0u);
                __syncwarp();
            }
        });
    } else {
        // this slice's sums, [part][token][channel], where the tiles were
        uint32_t* sums = reinterpret_cast<uint32_t*>(smem);
#pragma unroll 1
        for (uint32_t c = 0; c < tokens; c += 16) {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                uint32_t r[16];
                ld16(lane_addr + part * N + c, r);
                wait_ld(r);
#pragma unroll
                for (int i = 0; i < 16; ++i) sums[(part * N + c + i) * kRowsM + tid] = r[i];
            }
        }
        cluster_sync();
        // Each CTA finishes every slices-th token, a thread four channels of it. Eight reads are on their way at once: the slices' sums of
        // as many tokens.
        with_out_type(p.out_dtype, [&](auto type) {
            if (slices == 2) finish_slices(type, std::integral_constant<int, 2>{});
            else if (slices == 4) finish_slices(type, std::integral_constant<int, 4>{});
            else finish_slices(type, std::integral_constant<int, 8>{});
        });
        __syncwarp();
        cluster_sync();  // (a CTA's sums are read by the others)
    }
    fence_before();
    __syncthreads();
    if (warp == 1) {
        fence_after();
        tmem_dealloc(tmem, kCols);
    }
}

// ---- many tokens: pairs of CTAs -------------------------------------------------------------------------------------
// Persistent. Two CTAs (cta_group::2, M 256) share a tile of 256 weight rows x N tokens: each loads its own 128 weight rows and half
// of the tokens, and its tensor memory receives its own rows of the product. With SwiGLU a CTA's 128 rows are 64 gate rows and the
// matching 64 up rows, 16 and 16 in turn (a box of a three-dimensional map), so that a tile moves no more bytes than without and gate
// and up of a channel lie 16 lanes apart in one warp. Ten warps: warp 0 requests the tiles by TMA, warp 1 issues the
// MMAs into one of two accumulators, warps 2-9 scale, round and store the other one; a warpgroup has half of the tokens.
constexpr int kEpiWarps = 8, kPairThreads = (2 + kEpiWarps) * 32;
constexpr uint32_t kPairMaxStages = 8;
enum { P_FULL = 0, P_EMPTY = P_FULL + kPairMaxStages, P_ACC_FULL = P_EMPTY + kPairMaxStages, P_ACC_EMPTY = P_ACC_FULL + 2,
       P_BARS = P_ACC_EMPTY + 2 };
constexpr uint32_t kHalfRows = kRowsM / 2;  // of a weight tile: gate or up rows with SwiGLU
template <int N>
constexpr uint32_t pair_stage_bytes() { return kWTile + N / 2 * kStepK; }
constexpr uint32_t kPairTail = 1024 + 256 + kEpiWarps * 128 * 4;  // alignment of the base; barriers, tensor-memory address; scales

struct PairTiles {
    uint32_t t_tiles, r_tiles, band;
};
// Tile t of the flat list: bands of `band` token tiles, inside a band the token tile varies fastest.
__device__ __forceinline__ void tile_of(const PairTiles& p, uint32_t t, uint32_t& tt, uint32_t& rt) {
    const uint32_t per_band = p.band * p.r_tiles;
    const uint32_t b = t / per_band, r = t - b * per_band;
    const uint32_t rows = min(p.band, p.t_tiles - b * p.band);
    rt = r / rows;
    tt = b * p.band + (r - rt * rows);
}

template <bool SWIGLU, int N>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_i8_pair_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a,
                    const __grid_constant__ GemmI8Params p, const __grid_constant__ PairTiles tl) {
    constexpr uint32_t kStageBytes = pair_stage_bytes<N>();
    constexpr uint32_t kTok = N / 2;                               // tokens that a CTA loads, and that a warpgroup finishes
    constexpr uint32_t kChannels = SWIGLU ? kHalfRows : kRowsM;    // of a CTA's tile
    extern __shared__ unsigned char smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;  // swizzled tiles want 1024-byte alignment
    unsigned char* smem = smem_raw + (base - raw);
    const uint32_t bars_at = p.stages * kStageBytes;
    auto bar = [&](int i) { return base + bars_at + 8u * i; };
    volatile uint32_t* s_tmem = reinterpret_cast<volatile uint32_t*>(smem + bars_at + P_BARS * 8);
    float* s_scales = reinterpret_cast<float*>(smem + bars_at + 256);

    const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t worker = blockIdx.x / 2, workers = gridDim.x / 2;
    const uint32_t tiles = tl.t_tiles * tl.r_tiles;

    if (tid == 0) {
        prefetch_tensor_map(&tm_w);
        prefetch_tensor_map(&tm_a);
        for (uint32_t s = 0; s < p.stages; ++s) {
            mbar_init(bar(P_FULL + s), 1);
            mbar_init(bar(P_EMPTY + s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar(P_ACC_FULL + a), 1);
            mbar_init(bar(P_ACC_EMPTY + a), kEpiWarps * 2);  // one arrival per finishing warp of the pair
        }
        mbar_init_fence();
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(const_cast<uint32_t*>(s_tmem)), 512);
        tmem_relinquish_pair();
    }
    fence_before();
    __syncthreads();
    cluster_sync();  // the partner's barriers exist before anything is counted on them
    fence_after();
    const uint32_t tmem = *s_tmem;

    grid_dep_launch_dependents();
    grid_dep_wait();

    auto gave_up = [&]() {
        if (p.status) atomicOr(p.status, ATTN_STATUS_WAIT_TIMEOUT);
    };
    if (warp == 0) {
        if (elect_one()) {
            uint32_t s = 0, phase = 0, issued = 0;
            bool ok = true;
            for (uint32_t t = worker; t < tiles && ok; t += workers) {
                uint32_t tt, rt;
                tile_of(tl, t, tt, rt);
                const int row = static_cast<int>((rt * 2 + rank) * kChannels);
                const int tok = static_cast<int>(tt * N + rank * kTok);
                for (uint32_t ks = 0; ks < p.k_steps; ++ks, ++issued) {
                    if (issued >= p.stages && !mbar_wait(bar(P_EMPTY + s), phase ^ 1)) {
                        gave_up();
                        ok = false;
                        break;
                    }
                    const uint32_t dst = base + s * kStageBytes, full = bar(P_FULL + s);
                    const int kc = static_cast<int>(ks * kStepK);
                    if (rank == 0) mbar_arrive_expect_tx(full, 2 * kStageBytes);
                    if constexpr (SWIGLU) {
#pragma unroll
                        for (int g = 0; g < 4; ++g) tma_load_3d_pair(dst + g * (kWTile / 4), &tm_w, full, kc, row + 16 * g, 0);
                    } else {
                        tma_load_2d_pair(dst, &tm_w, full, kc, row);
                    }
                    tma_load_2d_pair(dst + kWTile, &tm_a, full, kc, tok);
                    if (++s == p.stages) s = 0, phase ^= 1;
                }
            }
            // No copy is in flight when the pair ends, whatever became of the MMAs: the leader's barriers count both CTAs' bytes,
            // and the CTAs meet at the end.
            if (rank == 0)
                for (uint32_t i = issued > p.stages ? issued - p.stages : 0; i < issued; ++i)
                    mbar_wait(bar(P_FULL + i % p.stages), i / p.stages & 1);
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            constexpr uint32_t idesc = instr_desc_i8(2 * kRowsM, N);
            const uint64_t desc0 = smem_desc(base, 16, 1024);
            uint32_t s = 0, phase = 0, local = 0;
            bool ok = true;
            for (uint32_t t = worker; t < tiles && ok; t += workers, ++local) {
                const uint32_t buf = local & 1;
                if (local >= 2 && !mbar_wait(bar(P_ACC_EMPTY + buf), (local / 2 - 1) & 1)) {
                    gave_up();
                    break;
                }
                fence_after();
                const uint32_t d = tmem + buf * 256;
                for (uint32_t ks = 0; ks < p.k_steps; ++ks) {
                    if (!mbar_wait(bar(P_FULL + s), phase)) {
                        gave_up();
                        ok = false;
                        break;
                    }
                    fence_after();
                    // K-major operands, 128-byte swizzle: 32 bytes per k-step of 32, 8-row groups 1024 bytes apart
                    const uint64_t w = desc0 + s * (kStageBytes / 16), a = w + kWTile / 16;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) mma_i8_pair(d, w + 2 * kk, a + 2 * kk, idesc, ks | kk);
                    commit_pair(bar(P_EMPTY + s));  // the stage may be refilled once these MMAs have read it
                    if (++s == p.stages) s = 0, phase ^= 1;
                }
                commit_pair(bar(P_ACC_FULL + buf));
            }
        }
    } else {
        const uint32_t quarter = warp & 3;       // the tensor-memory lanes that this warp may read
        const uint32_t group = (warp - 2) >> 2;  // its half of the tokens
        const uint32_t lane_addr = tmem + ((quarter * 32) << 16) + group * kTok;
        float* s_scale = s_scales + (warp - 2) * 128;
        const uint32_t empty0 = cluster_address(bar(P_ACC_EMPTY), 0);  // the leader's, also for its partner
        // SwiGLU: lanes 0-15 hold gate rows, lanes 16-31 the up rows of the same 16 channels
        const bool is_up = SWIGLU && lane >= 16;
        const uint32_t in_tile = SWIGLU ? quarter * 16 + (lane & 15) : quarter * 32 + lane;
        uint32_t local = 0;
        for (uint32_t t = worker; t < tiles; t += workers, ++local) {
            uint32_t tt, rt;
            tile_of(tl, t, tt, rt);
            const uint32_t buf = local & 1, tok0 = tt * N + group * kTok;
            const uint32_t col = (rt * 2 + rank) * kChannels + in_tile;
            const bool live = col < p.n_out;
            const float ws = live ? p.w_scale[is_up ? p.n_out + col : col] : 0.f;
#pragma unroll
            for (uint32_t i = lane; i < kTok; i += 32) s_scale[i] = tok0 + i < p.m ? p.a_scale[tok0 + i] : 0.f;
            __syncwarp();
            const uint32_t tokens = tok0 < p.m ? min(kTok, p.m - tok0) : 0u;
            // (a vote, so that the warp gives up or goes on as one)
            if (!__all_sync(0xffffffffu, mbar_wait(bar(P_ACC_FULL + buf), (local / 2) & 1))) {
                if (lane == 0) gave_up();
                break;
            }
            fence_after();
            const uint32_t acc = lane_addr + buf * 256;
            with_out_type(p.out_dtype, [&](auto type) {
                using T = decltype(type);
                // (SwiGLU: gate lanes finish the first 8 of 16 tokens, up lanes the last 8)
                uint32_t first = is_up ? 8 : 0;
                T* dst = static_cast<T*>(p.out) + static_cast<size_t>(tok0 + first) * p.ldc + col;
#pragma unroll 1
                for (uint32_t c = 0; c < kTok; c += 16, first += 16) {
                    uint32_t r[16];
                    ld16(acc + c, r);
                    wait_ld(r);
                    if (c + 16 == kTok) {  // the accumulator is read: hand it back
                        fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster_relaxed(empty0 + 8 * buf);
                    }
                    float y[16];
                    scaled16(y, r, ws, s_scale + c);
                    const uint32_t left = live && first < tokens ? tokens - first : 0u;
                    if constexpr (SWIGLU) {
                        float z[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float other = __shfl_xor_sync(0xffffffffu, is_up ? y[i] : y[8 + i], 16);
                            z[i] = __fmul_rn(silu(is_up ? other : y[i]), is_up ? y[8 + i] : other);
                        }
                        dst = store_tokens(dst, p.ldc, z, left) + 8 * p.ldc;
                    } else {
                        dst = store_tokens(dst, p.ldc, y, left);
                    }
                    __syncwarp();
                }
            });
        }
    }

    // ---- common exit: everybody (of both CTAs) meets, then the allocating warp releases tensor memory ----
    __syncwarp();
    fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// [rows][k] bytes, rows `stride` apart; box = 128 bytes of k x box_rows rows, 128-byte swizzle. Past k and past the rows: zeros. With
// `parts` > 1 that many such matrices one behind the other, and box_rows rows of each in the box.
int make_map(CUtensorMap* map, const void* ptr, uint64_t rows, uint64_t k, uint64_t stride, uint32_t box_rows, uint32_t parts = 1) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return ATTN_ERR_CUDA;
    const cuuint64_t dims[3] = {k, rows, parts};
    const cuuint64_t strides[2] = {stride, rows * stride};
    const cuuint32_t box[3] = {kStepK, box_rows, parts};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, parts > 1 ? 3 : 2, const_cast<void*>(ptr), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        g_last_cuda_error = static_cast<int>(r);
        return ATTN_ERR_CUDA;
    }
    return ATTN_OK;
}

// Operands as the entry point has checked them.
struct Operands {
    const AttnGemmI8Args* a;
    uint64_t a_stride, w_stride, w_rows;
    GemmI8Params p;
    DeviceInfo dev;
    cudaStream_t stream;
};

// Shared memory of a stream CTA: all of an SM's where there are no more CTAs than SMs (clusters have to fit the groups of 16 SMs and
// more that they are placed in), else half of it, so that one CTA streams while its neighbour starts or ends.
uint32_t stream_smem(uint64_t ctas, uint32_t slices, uint32_t sms) {
    const uint64_t fit = slices == 1 ? sms : slices == 2 ? sms - 4 : slices == 4 ? sms - 20 : 0;
    return ctas <= fit ? kMaxDynamicSmem : kMaxDynamicSmem / 2 - 2048;
}

template <int PARTS, int N>
int launch_stream(Operands& o, uint32_t slices) {
    GemmI8Params& p = o.p;
    constexpr uint32_t stage = stream_stage_bytes<PARTS, N>();
    static_assert(2 * stage >= PARTS * N * kRowsM * 4, "the slices' sums lie where the tiles were");
    const uint32_t row_tiles = (p.n_out + kRowsM - 1) / kRowsM, tok_tiles = (p.m + N - 1) / N;
    const uint64_t tiles = static_cast<uint64_t>(row_tiles) * tok_tiles;
    p.stages = std::min<uint32_t>(kStreamMaxStages, (stream_smem(tiles * slices, slices, o.dev.sm_count) - kStreamTail) / stage);
    const uint32_t smem = p.stages * stage + kStreamTail;
    CUtensorMap tm_w, tm_a;
    int rc;
    if ((rc = make_map(&tm_w, o.a->w, o.w_rows, o.a->k, o.w_stride, kRowsM)) != ATTN_OK) return rc;
    if ((rc = make_map(&tm_a, o.a->a, p.m, o.a->k, o.a_stride, N)) != ATTN_OK) return rc;
    auto kernel = gemm_i8_stream_kernel<PARTS, N>;
    B200_CUDA_TRY(allow_max_smem(kernel));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(slices, tok_tiles, row_tiles);
    cfg.blockDim = dim3(kStreamThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = o.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = slices;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tm_w, tm_a, p));
    g_launch_count.fetch_add(1, std::memory_order_relaxed);
    return ATTN_OK;
}

template <bool SWIGLU, int N>
int launch_pair(Operands& o) {
    GemmI8Params& p = o.p;
    constexpr uint32_t stage = pair_stage_bytes<N>(), span = SWIGLU ? kRowsM : 2 * kRowsM;
    p.stages = std::min<uint32_t>(kPairMaxStages, (kMaxDynamicSmem - kPairTail) / stage);
    PairTiles tl{};
    tl.t_tiles = (p.m + N - 1) / N;
    tl.r_tiles = (p.n_out + span - 1) / span;
    if (static_cast<uint64_t>(tl.t_tiles) * tl.r_tiles > 0x7fffffffu) return ATTN_ERR_UNSUPPORTED;
    // token tiles of a band: a wave of 74 tiles is then about as many tokens as channels, the least to read (9184 x 4096 x 28672 with
    // SwiGLU: bands of 4, 8, 16, 36 tiles 749, 708, 786, 784 us; 9184 x 14336 x 4096 326, 322, 331, 354)
    tl.band = std::min<uint32_t>(tl.t_tiles, 8);
    CUtensorMap tm_w, tm_a;
    int rc;
    if (SWIGLU) rc = make_map(&tm_w, o.a->w, p.n_out, o.a->k, o.w_stride, 16, 2);
    else rc = make_map(&tm_w, o.a->w, o.w_rows, o.a->k, o.w_stride, kRowsM);
    if (rc != ATTN_OK) return rc;
    if ((rc = make_map(&tm_a, o.a->a, p.m, o.a->k, o.a_stride, N / 2)) != ATTN_OK) return rc;
    auto kernel = gemm_i8_pair_kernel<SWIGLU, N>;
    B200_CUDA_TRY(allow_max_smem(kernel));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(2 * std::min(tl.t_tiles * tl.r_tiles, static_cast<uint32_t>(o.dev.sm_count) / 2));
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = p.stages * stage + kPairTail;
    cfg.stream = o.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    B200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tm_w, tm_a, p, tl));
    g_launch_count.fetch_add(1, std::memory_order_relaxed);
    return ATTN_OK;
}

template <int PARTS>
int launch_gemm(Operands& o) {
    constexpr bool kSwiglu = PARTS == 2;
    const uint64_t m = o.p.m, sms = o.dev.sm_count, r128 = (o.p.n_out + kRowsM - 1) / kRowsM;
    const uint32_t n = m <= 16 ? 16 : m <= 32 ? 32 : 64;
    const uint64_t tiles = (m + n - 1) / n * r128;
    // Single CTAs for up to 64 tokens (a whole vocabulary of channels is left to pairs, which are persistent: 61 x 4096 x 128256 88.4 and 83.4
    // us, 8 tokens 79.0 and 82.0), and for more where the tiles are half as many as SMs at most and slices of k make up for it:
    // 105 x 12608 x 896 9.1 us in 8 slices, pairs 20.2; 400 x 14336 x 512 10.4 and 21; 128 x 4096 x 4096 8.9 and 9.5; but 256 x 4096 x 6144 13.8 and
    // 10.8. With SwiGLU pairs lose against four slices of a long k only: 299 x 4728 x 864 8.7 and 10.1, 522 x 1712 x 1664 10.4 and 7.9.
    const bool few = tiles <= sms / 2 && (!kSwiglu || (tiles <= 32 && o.p.k_steps >= 32));
    if (m <= 64 ? r128 <= (m <= 32 ? 65535 : 4 * sms) : few) {
        // Slices until they are 256 (of 64 tokens with SwiGLU, whose stages are large, 128), none shorter than its sums' way to their place is
        // worth: a stage with up to 16 tokens (14 x 1744 x 1004 in 1, 2, 4, 8 slices 7.6, 6.3, 5.3, 4.8 us), eight with 64 (100 x 2000 x 2000 6.9,
        // 6.3, 6.3, 6.8; 40 x 1024 x 1024 3.8, 4.0, 3.9, 4.1; 170 x 11328 x 1024 18.0, 12.1, 9.8, 9.6).
        const uint32_t shortest = n == 16 ? 1 : n == 32 ? 3 : 8, most = PARTS * n > 64 ? 128 : 256;
        uint32_t slices = 1;
        while (2 * slices <= (PARTS * n > 64 ? 4 : kMaxSlices) && tiles <= sms / 2 && tiles * 2 * slices <= most && o.p.k_steps >= shortest * 2 * slices)
            slices *= 2;
        return n == 16 ? launch_stream<PARTS, 16>(o, slices) : n == 32 ? launch_stream<PARTS, 32>(o, slices) : launch_stream<PARTS, 64>(o, slices);
    }
    if (m <= 64) return launch_pair<kSwiglu, 64>(o);
    // Tiles of 256 tokens or of 128: the fewer waves of pairs, one of the smaller ones being a little more than half as long. 1003 x 4096 x 4096
    // 15.7 us in one wave of the larger, 16.8 in two; 9184 x 14336 x 4096 322 and 361; but 512 x 4096 x 4096, one wave either way, 14.8 and 10.6.
    const uint64_t pairs = sms / 2, span = kSwiglu ? kRowsM : 2 * kRowsM, r_tiles = (o.p.n_out + span - 1) / span;
    auto waves = [&](uint32_t tokens) { return ((m + tokens - 1) / tokens * r_tiles + pairs - 1) / pairs; };
    return waves(256) * 10 <= waves(128) * 6 ? launch_pair<kSwiglu, 256>(o) : launch_pair<kSwiglu, 128>(o);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int attn_gemm_i8(const AttnGemmI8Args* a, void* stream_v) {
    if (!a || !a->out || !a->a || !a->a_scale || !a->w || !a->w_scale || a->m == 0 || a->n_out == 0 || a->k == 0) return ATTN_ERR_INVALID_ARG;
    if (a->out_dtype != ATTN_DTYPE_F32 && a->out_dtype != ATTN_DTYPE_F16 && a->out_dtype != ATTN_DTYPE_BF16) return ATTN_ERR_INVALID_ARG;
    if (a->k > kMaxK || a->m > 0x7fffff00u || a->n_out > 0x3fffff00u) return ATTN_ERR_UNSUPPORTED;
    Operands o{};
    o.a = a;
    const uint64_t packed = (static_cast<uint64_t>(a->k) + 15) & ~15ull;
    o.a_stride = a->a_stride ? a->a_stride : packed;
    o.w_stride = a->w_stride ? a->w_stride : packed;
    o.w_rows = static_cast<uint64_t>(a->n_out) * (a->swiglu ? 2 : 1);
    GemmI8Params& p = o.p;
    p.ldc = a->ldc ? a->ldc : a->n_out;
    if (o.a_stride < a->k || o.w_stride < a->k || p.ldc < a->n_out) return ATTN_ERR_INVALID_ARG;
    const uint32_t size = a->out_dtype == ATTN_DTYPE_F32 ? 4 : 2;
    auto at = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr); };
    if ((at(a->a) | at(a->w) | o.a_stride | o.w_stride) % 16 || (at(a->a_scale) | at(a->w_scale)) % 4 || at(a->out) % size)
        return ATTN_ERR_ALIGNMENT;
    // a tensor map's limits
    if (o.a_stride >= 1ull << 40 || o.w_stride >= 1ull << 40 || (a->swiglu && o.w_stride >= (1ull << 40) / a->n_out)) return ATTN_ERR_UNSUPPORTED;
    const Runs out(a->out, 1, 0, a->m, size * p.ldc, static_cast<uint64_t>(size) * a->n_out);
    if (share_memory(out, Runs(a->a, 1, 0, a->m, o.a_stride, a->k)) || share_memory(out, Runs(a->w, 1, 0, o.w_rows, o.w_stride, a->k)) ||
        share_memory(out, Runs(a->a_scale, 1, 0, 1, 0, 4ull * a->m)) || share_memory(out, Runs(a->w_scale, 1, 0, 1, 0, 4 * o.w_rows)))
        return ATTN_ERR_INVALID_ARG;
    int rc = current_device_info(&o.dev);
    if (rc != ATTN_OK) return rc;
    if (o.dev.cc_major != 10) return ATTN_ERR_DEVICE;
    p.out = a->out;
    p.a_scale = a->a_scale;
    p.w_scale = a->w_scale;
    p.m = a->m;
    p.n_out = a->n_out;
    p.k_steps = (a->k + kStepK - 1) / kStepK;
    p.out_dtype = a->out_dtype;
    p.w_early = a->w_early ? 1u : 0u;
    p.status = a->status;
    o.stream = static_cast<cudaStream_t>(stream_v);
    return a->swiglu ? launch_gemm<2>(o) : launch_gemm<1>(o);
}
