// Product of 8-bit integers with a scale per token and per channel, on the 5th-generation tensor cores (kind::i8):
//
//     out[t][j] = a_scale[t] * w_scale[j] * sum_i a[t][i] * w[j][i]        t < m tokens, j < n_out channels, i < k
//
// The sum is exact: products of 8 bits, added in 32 (k up to 131071 keeps any sum below 2^31), so cutting k into slices and adding
// them in any order gives the same bits. Weights are the M side of the MMA: a tensor-memory lane is a channel, which has its scale in
// a register, and a warp stores 32 neighbouring channels of a token at a time.
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

__device__ __forceinline__ float silu(float x) { return __fdiv_rn(x, 1.0f + expf(-x)); }
// the scaled sum; the order of the two products is part of the result's bits
__device__ __forceinline__ float scaled(int32_t sum, float w_scale, float a_scale) {
    return __fmul_rn(__fmul_rn(static_cast<float>(sum), w_scale), a_scale);
}
template <typename T>
__device__ __forceinline__ T to_out(float x);
template <>
__device__ __forceinline__ float to_out<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half to_out<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 to_out<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
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
enum { S_FULL = 0, kStreamMaxStages = 8, S_EMPTY = S_FULL + kStreamMaxStages, S_ACC = S_EMPTY + kStreamMaxStages, S_BARS };
constexpr int kStreamThreads = 128;

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

    if (tid == 0) {
        for (uint32_t s = 0; s < p.stages; ++s) {
            mbar_init(bar(S_FULL + s), 1);
            mbar_init(bar(S_EMPTY + s), 1);
        }
        mbar_init(bar(S_ACC), 1);
        mbar_init_fence();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(const_cast<uint32_t*>(s_tmem)), kCols);
        tmem_relinquish();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *s_tmem;

    grid_dep_launch_dependents();
    grid_dep_wait();
    if (tid < N) s_scale[tid] = tok0 + tid < p.m ? p.a_scale[tok0 + tid] : 0.f;

    auto gave_up = [&]() {
        if (p.status) atomicOr(p.status, ATTN_STATUS_WAIT_TIMEOUT);
    };
    if (warp == 0) {
        if (elect_one()) {
            uint32_t s = 0, phase = 0, issued = 0;
            for (uint32_t ks = ks0; ks < ks1; ++ks, ++issued) {
                if (issued >= p.stages && !mbar_wait(bar(S_EMPTY + s), phase ^ 1)) {
                    gave_up();
                    break;
                }
                const uint32_t dst = base + s * kStageBytes, full = bar(S_FULL + s);
                const int kc = static_cast<int>(ks * kStepK);
                mbar_arrive_expect_tx(full, kStageBytes);
#pragma unroll
                for (int part = 0; part < PARTS; ++part)
                    tma_load_2d(dst + part * kWTile, &tm_w, full, kc, static_cast<int>(row0 + part * p.n_out));
                tma_load_2d(dst + PARTS * kWTile, &tm_a, full, kc, static_cast<int>(tok0));
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
    __syncthreads();  // s_scale

    const uint32_t lane_addr = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const uint32_t col = row0 + tid;  // channel of this thread
    const uint32_t tokens = min(static_cast<uint32_t>(N), p.m - tok0);
    const bool live = col < p.n_out;
    const float w0 = live ? p.w_scale[col] : 0.f;
    const float w1 = PARTS == 2 && live ? p.w_scale[p.n_out + col] : 0.f;
    auto finish = [&](auto type, uint32_t t, int32_t s0, int32_t s1) {
        using T = decltype(type);
        float y = scaled(s0, w0, s_scale[t]);
        if constexpr (PARTS == 2) y = __fmul_rn(silu(y), scaled(s1, w1, s_scale[t]));
        static_cast<T*>(p.out)[(tok0 + t) * p.ldc + col] = to_out<T>(y);
    };
    if (slices == 1) {
#pragma unroll 1
        for (uint32_t c = 0; c < N; c += 16) {
            uint32_t r[PARTS][16];
#pragma unroll
            for (int part = 0; part < PARTS; ++part) ld16(lane_addr + part * N + c, r[part]);
#pragma unroll
            for (int part = 0; part < PARTS; ++part) wait_ld(r[part]);
            with_out_type(p.out_dtype, [&](auto type) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (live && c + i < tokens) finish(type, c + i, r[0][i], r[PARTS - 1][i]);
            });
        }
    } else {
        // this slice's sums, [part][token][channel], where the tiles were
        uint32_t* sums = reinterpret_cast<uint32_t*>(smem);
#pragma unroll 1
        for (uint32_t c = 0; c < N; c += 16) {
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
                uint32_t r[16];
                ld16(lane_addr + part * N + c, r);
                wait_ld(r);
#pragma unroll
                for (int i = 0; i < 16; ++i) sums[(part * N + c + i) * kRowsM + tid] = r[i];
            }
        }
        __syncwarp();
        cluster_sync();
        with_out_type(p.out_dtype, [&](auto type) {
            for (uint32_t t = slice; t < tokens; t += slices) {
                int32_t s[2] = {0, 0};
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const uint32_t at = base + ((part * N + t) * kRowsM + tid) * 4;
                    for (uint32_t r = 0; r < slices; ++r) s[part] += static_cast<int32_t>(ld_cluster_u32(cluster_address(at, r)));
                }
                if (live) finish(type, t, s[0], s[PARTS - 1]);
            }
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

// [rows][k] bytes, rows `stride` apart; box = 128 bytes of k x box_rows rows, 128-byte swizzle. Past k and past the rows: zeros.
int make_map(CUtensorMap* map, const void* ptr, uint64_t rows, uint64_t k, uint64_t stride, uint32_t box_rows) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return ATTN_ERR_CUDA;
    const cuuint64_t dims[2] = {k, rows};
    const cuuint64_t strides[1] = {stride};
    const cuuint32_t box[2] = {kStepK, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
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

template <int PARTS, int N>
int launch_stream(Operands& o) {
    GemmI8Params& p = o.p;
    constexpr uint32_t stage = stream_stage_bytes<PARTS, N>();
    const uint32_t row_tiles = (p.n_out + kRowsM - 1) / kRowsM, tok_tiles = (p.m + N - 1) / N;
    if (row_tiles > 65535 || tok_tiles > 65535) return ATTN_ERR_UNSUPPORTED;
    // two CTAs on an SM, so that one of them streams while the other starts or ends
    p.stages = std::min<uint32_t>(kStreamMaxStages, (kMaxDynamicSmem / 2 - 2048 - kStreamTail) / stage);
    const uint64_t tiles = static_cast<uint64_t>(row_tiles) * tok_tiles;
    uint32_t slices = 1;
    while (slices < 8 && slices < p.k_steps && tiles * (slices + 1) <= 2ull * o.dev.sm_count) ++slices;
    if (slices > 1 && p.stages * stage < PARTS * N * kRowsM * 4) slices = 1;  // (the slices' sums lie where the tiles were)
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

template <int PARTS>
int launch_gemm(Operands& o) {
    return o.p.m <= 16 ? launch_stream<PARTS, 16>(o) : o.p.m <= 32 ? launch_stream<PARTS, 32>(o) : o.p.m <= 64 ? launch_stream<PARTS, 64>(o) : launch_stream<PARTS, 128>(o);
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
    if (o.a_stride >= 1ull << 40 || o.w_stride >= 1ull << 40) return ATTN_ERR_UNSUPPORTED;  // a tensor map's limit
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
    p.status = a->status;
    o.stream = static_cast<cudaStream_t>(stream_v);
    return a->swiglu ? launch_gemm<2>(o) : launch_gemm<1>(o);
}
