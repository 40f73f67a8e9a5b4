// Rows of activations (or a matrix's channels) as 8-bit whole numbers with an fp32 scale each, the operand of attn_gemm_i8: plain
// (attn_quantize_i8), or behind the residual's addition and RMSNorm (attn_rmsnorm_i8).
//
// Mathematics: h = x + delta, z = h * weight, A = max|z|, r = 1 / sqrt(mean(h^2) + eps). The norm is y = r z, and the symmetric
// 8-bit form has scale max|y| / 127 = r A / 127 and q = round(y / scale) = round(z * (127 / A)): r cancels. So one pass over the row
// yields both reductions, and q, made of single fp32 operations on single elements, does not depend on the order of any sum. The largest
// |z| is found on the bits without their sign, which order as the numbers do and put infinity and NaN on top.
//
// Bound by memory: every value is read once and written once. A row stays in the registers of its threads between the reductions and
// the rounding (CHUNKS runs of VEC values a thread; CHUNKS 0, for rows longer than that: read twice, the second time from L2).
#include <algorithm>

#include "attn_internal.cuh"
#include "operand_memory.cuh"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

struct RowsParams {
    int8_t* q;
    float* scale;
    void* x_out;
    const void* x;
    const void* delta;
    const float* weight;
    uint64_t q_stride, x_stride, delta_stride, x_out_stride;
    uint32_t rows, dim;
    uint32_t row_threads;  // of a row: 32 (a block serves several rows) or the whole block
    float eps;
    int32_t delta_dtype;
};

constexpr uint32_t kMaxThreads = 1024, kWarpRows = 4;  // threads of a block, rows of one whose rows are a warp's
constexpr uint32_t kInf = 0x7f800000u;
// (four runs of eight values of x, delta and weight beside each other do not fit the 64 registers that 1024 threads have each)
constexpr uint32_t max_threads(bool norm, int vec, uint32_t chunks) { return norm && vec == 8 && chunks == 4 ? 512 : kMaxThreads; }

// VEC values as they lie in memory: fp32 words, or pairs of 16-bit values in the first half of them.
template <int VEC>
struct Raw {
    uint32_t w[VEC];
};
// `n` of the VEC values from element i on; ALIGNED: p + i may be read in runs of VEC values.
template <int VEC, bool ALIGNED>
__device__ __forceinline__ void load(Raw<VEC>& r, const void* p, size_t i, bool wide32, uint32_t n) {
    if (wide32) {
        const uint32_t* s = static_cast<const uint32_t*>(p) + i;
        if (ALIGNED && n >= VEC) {
#pragma unroll
            for (int k = 0; k < VEC; k += 4) *reinterpret_cast<uint4*>(&r.w[k]) = *reinterpret_cast<const uint4*>(s + k);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) r.w[k] = k < n ? s[k] : 0u;
        }
    } else {
        const unsigned short* s = static_cast<const unsigned short*>(p) + i;
        if (ALIGNED && n >= VEC) {
            if constexpr (VEC == 8) *reinterpret_cast<uint4*>(&r.w[0]) = *reinterpret_cast<const uint4*>(s);
            else *reinterpret_cast<uint2*>(&r.w[0]) = *reinterpret_cast<const uint2*>(s);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; k += 2)
                r.w[k / 2] = (k < n ? s[k] : 0u) | (k + 1 < n ? static_cast<uint32_t>(s[k + 1]) << 16 : 0u);
        }
    }
}
template <int VEC>
__device__ __forceinline__ void widen(float (&v)[VEC], const Raw<VEC>& r, int32_t dtype) {
    if (dtype == ATTN_DTYPE_F32) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = __uint_as_float(r.w[k]);
    } else if (dtype == ATTN_DTYPE_F16) {
#pragma unroll
        for (int k = 0; k < VEC; k += 2) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[k / 2]));
            v[k] = f.x, v[k + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < VEC; k += 2) {
            v[k] = __uint_as_float(r.w[k / 2] << 16);
            v[k + 1] = __uint_as_float(r.w[k / 2] & 0xffff0000u);
        }
    }
}
template <int VEC, int DT, bool ALIGNED>
__device__ __forceinline__ void store(void* p, size_t i, const float (&v)[VEC], uint32_t n) {
    if constexpr (DT == ATTN_DTYPE_F32) {
        float* d = static_cast<float*>(p) + i;
        if (ALIGNED && n >= VEC) {
#pragma unroll
            for (int k = 0; k < VEC; k += 4) *reinterpret_cast<float4*>(d + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (k < n) d[k] = v[k];
        }
    } else {
        unsigned short* d = static_cast<unsigned short*>(p) + i;
        uint32_t u[VEC / 2];
#pragma unroll
        for (int k = 0; k < VEC; k += 2) u[k / 2] = pack2<DT == ATTN_DTYPE_BF16>(v[k], v[k + 1]);
        if (ALIGNED && n >= VEC) {
            if constexpr (VEC == 8) *reinterpret_cast<uint4*>(d) = make_uint4(u[0], u[1], u[2], u[3]);
            else *reinterpret_cast<uint2*>(d) = make_uint2(u[0], u[1]);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (k < n) d[k] = static_cast<unsigned short>(u[k / 2] >> (16 * (k & 1)));
        }
    }
}

// A row's reductions, the same in all its threads: the largest bits and the sum.
__device__ __forceinline__ void reduce_row(uint32_t& top, float& sum, bool whole_block) {
    top = __reduce_max_sync(0xffffffffu, top);
#pragma unroll
    for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (!whole_block) return;
    __shared__ uint32_t s_top[kMaxThreads / 32];
    __shared__ float s_sum[kMaxThreads / 32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) s_top[warp] = top, s_sum[warp] = sum;
    __syncthreads();
    const bool there = lane < blockDim.x / 32;
    top = __reduce_max_sync(0xffffffffu, there ? s_top[lane] : 0u);
    sum = there ? s_sum[lane] : 0.f;
#pragma unroll
    for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
}

// DT: type of x. NORM: weight, and the norm's factor in the scale. ALIGNED: rows may be read and written in runs of VEC values.
template <int DT, bool NORM, bool DELTA, int VEC, int CHUNKS, bool ALIGNED>
__global__ void __launch_bounds__(max_threads(NORM, VEC, CHUNKS)) rows_i8_kernel(const __grid_constant__ RowsParams p) {
    grid_dep_launch_dependents();
    grid_dep_wait();
    const bool whole_block = p.row_threads != 32;
    const uint32_t row = whole_block ? blockIdx.x : blockIdx.x * kWarpRows + (threadIdx.x >> 5);
    const uint32_t t = whole_block ? threadIdx.x : threadIdx.x & 31;
    if (row >= p.rows) return;
    const size_t x_row = row * p.x_stride, d_row = row * p.delta_stride, o_row = row * p.x_out_stride;
    const bool wide_delta = p.delta_dtype == ATTN_DTYPE_F32;
    int8_t* q = p.q + row * p.q_stride;

    auto fetch = [&](uint32_t i, Raw<VEC>& rx, Raw<VEC>& rd, Raw<VEC>& rw) {
        const uint32_t n = p.dim - i;
        load<VEC, ALIGNED>(rx, p.x, x_row + i, DT == ATTN_DTYPE_F32, n);
        if constexpr (DELTA) load<VEC, ALIGNED>(rd, p.delta, d_row + i, wide_delta, n);
        if constexpr (NORM) load<VEC, ALIGNED>(rw, p.weight, i, true, n);
    };
    auto combine = [&](const Raw<VEC>& rx, const Raw<VEC>& rd, const Raw<VEC>& rw, float (&h)[VEC], float (&z)[VEC]) {
        widen<VEC>(h, rx, DT);
        if constexpr (DELTA) {
            float d[VEC];
            widen<VEC>(d, rd, p.delta_dtype);
#pragma unroll
            for (int k = 0; k < VEC; ++k) h[k] = __fadd_rn(h[k], d[k]);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) z[k] = NORM ? __fmul_rn(h[k], __uint_as_float(rw.w[k])) : h[k];
    };
    auto count = [&](const float (&h)[VEC], const float (&z)[VEC], uint32_t& top, float& sum) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            top = max(top, __float_as_uint(z[k]) & 0x7fffffffu);
            if constexpr (NORM) sum = fmaf(h[k], h[k], sum);
        }
    };
    float inverse, lift;
    auto scale_of = [&](uint32_t top, float sum) {
        const float a = __uint_as_float(top);
        // (127 / A leaves fp32's range below 2^-121: such rows are lifted first, which is exact)
        lift = top < 0x03000000u ? 18446744073709551616.f : 1.f;
        inverse = top == 0 ? 0.f : __fdiv_rn(127.f, __fmul_rn(a, lift));
        float scale = a;
        if constexpr (NORM) scale *= __frcp_rn(sqrtf(sum / static_cast<float>(p.dim) + p.eps));
        scale = __fdiv_rn(scale, 127.f);
        const bool bad = top >= kInf || (NORM && !(sum < __uint_as_float(kInf)));
        if (bad) inverse = 0.f, scale = __uint_as_float(0x7fc00000u);
        if (t == 0) p.scale[row] = scale;
        return bad;
    };
    auto put = [&](uint32_t i, const float (&z)[VEC], bool bad) {
        const uint32_t n = p.dim - i;
        uint32_t u[VEC / 4];
#pragma unroll
        for (int k = 0; k < VEC; k += 4) {
            uint32_t b[4];
#pragma unroll
            // 1.5 * 2^23 puts the whole number next to a value of at most 2^22 (ties to the even one) into the low bits of the sum
            for (int e = 0; e < 4; ++e)
                b[e] = __float_as_uint(__fadd_rn(__fmul_rn(__fmul_rn(z[k + e], lift), inverse), 12582912.f));
            u[k / 4] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            if (bad) u[k / 4] = 0u;
        }
        if (n >= VEC) {
            if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q + i) = make_uint2(u[0], u[1]);
            else *reinterpret_cast<uint32_t*>(q + i) = u[0];
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (k < n) q[i + k] = static_cast<int8_t>(u[k / 4] >> (8 * (k & 3)));
        }
    };

    uint32_t top = 0;
    float sum = 0.f;
    if constexpr (CHUNKS > 0) {
        Raw<VEC> rx[CHUNKS], rd[CHUNKS], rw[CHUNKS];
        float z[CHUNKS][VEC];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t i = (c * p.row_threads + t) * VEC;
            if (i < p.dim) fetch(i, rx[c], rd[c], rw[c]);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t i = (c * p.row_threads + t) * VEC;
            if (i < p.dim) {
                float h[VEC];
                combine(rx[c], rd[c], rw[c], h, z[c]);
                count(h, z[c], top, sum);
                if constexpr (DELTA)
                    if (p.x_out) store<VEC, DT, ALIGNED>(p.x_out, o_row + i, h, p.dim - i);
            }
        }
        reduce_row(top, sum, whole_block);
        const bool bad = scale_of(top, sum);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t i = (c * p.row_threads + t) * VEC;
            if (i < p.dim) put(i, z[c], bad);
        }
    } else {
        Raw<VEC> rx, rd, rw;
        float h[VEC], z[VEC];
        for (uint32_t i = t * VEC; i < p.dim; i += p.row_threads * VEC) {
            fetch(i, rx, rd, rw);
            combine(rx, rd, rw, h, z);
            count(h, z, top, sum);
        }
        reduce_row(top, sum, whole_block);
        const bool bad = scale_of(top, sum);
        for (uint32_t i = t * VEC; i < p.dim; i += p.row_threads * VEC) {  // (x_out may be x: nothing was written before)
            fetch(i, rx, rd, rw);
            combine(rx, rd, rw, h, z);
            if constexpr (DELTA)
                if (p.x_out) store<VEC, DT, ALIGNED>(p.x_out, o_row + i, h, p.dim - i);
            put(i, z, bad);
        }
    }
}

uint32_t size_of(int32_t dtype) { return dtype == ATTN_DTYPE_F32 ? 4 : 2; }
bool is_float(int32_t d) { return d == ATTN_DTYPE_F32 || d == ATTN_DTYPE_F16 || d == ATTN_DTYPE_BF16; }

template <int DT, bool NORM, bool DELTA>
int launch_rows(RowsParams& p, bool aligned, const DeviceInfo& dev, cudaStream_t stream) {
    constexpr int kWide = DT == ATTN_DTYPE_F32 ? 4 : 8;
    const uint32_t vec = aligned ? kWide : 4;
    auto threads = [&](uint32_t chunks) { return ((p.dim + vec * chunks - 1) / (vec * chunks) + 31) / 32 * 32; };
    uint32_t chunks = 4;
    if (aligned)  // few rows: more threads for each
        while (chunks > 1 && static_cast<uint64_t>(p.rows) * threads(chunks) < static_cast<uint64_t>(dev.sm_count) * 1024 &&
               threads(chunks / 2) <= kMaxThreads)
            chunks /= 2;
    p.row_threads = threads(chunks);
    if (p.row_threads > max_threads(NORM, vec, chunks)) p.row_threads = kMaxThreads, chunks = 0;
    const bool warps = p.row_threads == 32;
    const uint32_t block = warps ? 32 * kWarpRows : p.row_threads;
    const uint32_t grid = warps ? (p.rows + kWarpRows - 1) / kWarpRows : p.rows;
    void (*kernel)(RowsParams) = !aligned ? (chunks ? rows_i8_kernel<DT, NORM, DELTA, 4, 4, false> : rows_i8_kernel<DT, NORM, DELTA, 4, 0, false>)
                                 : chunks == 4 ? rows_i8_kernel<DT, NORM, DELTA, kWide, 4, true>
                                 : chunks == 2 ? rows_i8_kernel<DT, NORM, DELTA, kWide, 2, true>
                                 : chunks == 1 ? rows_i8_kernel<DT, NORM, DELTA, kWide, 1, true>
                                               : rows_i8_kernel<DT, NORM, DELTA, kWide, 0, true>;
    B200_CUDA_TRY(launch_dependent(kernel, dim3(grid), dim3(block), 0, stream, p));
    g_launch_count.fetch_add(1, std::memory_order_relaxed);
    return ATTN_OK;
}

template <bool NORM, bool DELTA>
int launch_rows_of(int32_t dtype, RowsParams& p, bool aligned, const DeviceInfo& dev, cudaStream_t stream) {
    return dtype == ATTN_DTYPE_F32   ? launch_rows<ATTN_DTYPE_F32, NORM, DELTA>(p, aligned, dev, stream)
           : dtype == ATTN_DTYPE_F16 ? launch_rows<ATTN_DTYPE_F16, NORM, DELTA>(p, aligned, dev, stream)
                                     : launch_rows<ATTN_DTYPE_BF16, NORM, DELTA>(p, aligned, dev, stream);
}

int rows_i8(const AttnRowsI8Args* a, bool norm, void* stream_v) {
    if (!a || !a->q || !a->scale || !a->x || a->rows == 0 || a->dim == 0 || !is_float(a->x_dtype)) return ATTN_ERR_INVALID_ARG;
    if (norm ? !a->weight || !(a->eps >= 1.17549435e-38f) || a->eps > 3.4e38f : a->weight || a->delta) return ATTN_ERR_INVALID_ARG;
    if (a->delta ? !is_float(a->delta_dtype) : a->x_out != nullptr) return ATTN_ERR_INVALID_ARG;
    if (a->rows > 0x7fffffffu || a->dim > 0x7fffff00u) return ATTN_ERR_UNSUPPORTED;
    RowsParams p{};
    p.q_stride = a->q_stride ? a->q_stride : (static_cast<uint64_t>(a->dim) + 15) & ~15ull;
    p.x_stride = a->x_stride ? a->x_stride : a->dim;
    p.delta_stride = a->delta_stride ? a->delta_stride : a->dim;
    p.x_out_stride = a->x_out_stride ? a->x_out_stride : a->dim;
    if (p.q_stride < a->dim || p.x_stride < a->dim || p.delta_stride < a->dim || p.x_out_stride < a->dim) return ATTN_ERR_INVALID_ARG;
    const uint32_t xs = size_of(a->x_dtype), ds = size_of(a->delta_dtype);
    auto at = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr); };
    if (at(a->q) % 16 || p.q_stride % 16 || at(a->scale) % 4 || at(a->x) % xs || at(a->x_out) % xs || at(a->weight) % 4 ||
        (a->delta && at(a->delta) % ds))
        return ATTN_ERR_ALIGNMENT;
    // What is written shares memory with nothing else, but for x_out in the place of x: a row's threads run in any order.
    const uint64_t n = a->rows, d = a->dim;
    const Runs q(a->q, 1, 0, n, p.q_stride, d), scale(a->scale, 1, 0, 1, 0, 4 * n), x(a->x, 1, 0, n, xs * p.x_stride, xs * d),
        weight(a->weight, 1, 0, 1, 0, 4 * d), delta(a->delta, 1, 0, n, ds * p.delta_stride, ds * d),
        x_out(a->x_out, 1, 0, n, xs * p.x_out_stride, xs * d);
    if (share_memory(q, scale) || share_memory(q, x) || share_memory(scale, x)) return ATTN_ERR_INVALID_ARG;
    if (norm && (share_memory(q, weight) || share_memory(scale, weight))) return ATTN_ERR_INVALID_ARG;
    if (a->delta && (share_memory(q, delta) || share_memory(scale, delta))) return ATTN_ERR_INVALID_ARG;
    if (a->x_out) {
        const bool in_place = a->x_out == a->x && (n == 1 || p.x_out_stride == p.x_stride);
        if (share_memory(x_out, q) || share_memory(x_out, scale) || share_memory(x_out, weight) || share_memory(x_out, delta) ||
            (!in_place && share_memory(x_out, x)))
            return ATTN_ERR_INVALID_ARG;
    }
    DeviceInfo dev{};
    const int rc = current_device_info(&dev);
    if (rc != ATTN_OK) return rc;
    if (dev.cc_major != 10) return ATTN_ERR_DEVICE;
    p.q = a->q;
    p.scale = a->scale;
    p.x_out = a->x_out;
    p.x = a->x;
    p.delta = a->delta;
    p.weight = a->weight;
    p.rows = a->rows;
    p.dim = a->dim;
    p.eps = a->eps;
    p.delta_dtype = a->delta_dtype;
    // runs of VEC values: 16 bytes of 16-bit values, 32 bytes (two accesses of 16) of fp32 beside them
    const uint64_t rows_apart = n > 1 ? ~0ull : 0ull;
    bool aligned = (at(a->x) | ((xs * p.x_stride) & rows_apart) | at(a->x_out) | (a->x_out ? (xs * p.x_out_stride) & rows_apart : 0) |
                    at(a->weight)) % 16 == 0;
    if (a->delta) {
        const uint32_t vec = a->x_dtype == ATTN_DTYPE_F32 ? 4 : 8, run = std::min<uint32_t>(16, vec * ds);
        aligned = aligned && (at(a->delta) | ((ds * p.delta_stride) & rows_apart)) % run == 0;
    }
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    if (!norm) return launch_rows_of<false, false>(a->x_dtype, p, aligned, dev, stream);
    return a->delta ? launch_rows_of<true, true>(a->x_dtype, p, aligned, dev, stream)
                    : launch_rows_of<true, false>(a->x_dtype, p, aligned, dev, stream);
}

}  // namespace
}  // namespace b200

extern "C" int attn_rmsnorm_i8(const AttnRowsI8Args* args, void* stream) { return b200::rows_i8(args, true, stream); }
extern "C" int attn_quantize_i8(const AttnRowsI8Args* args, void* stream) { return b200::rows_i8(args, false, stream); }
