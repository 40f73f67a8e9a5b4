// Rows of activations (or a matrix's channels) as 8-bit whole numbers with an fp32 scale each, the operand of attn_gemm_i8: plain
// (attn_quantize_i8), or behind the residual's addition and RMSNorm (attn_rmsnorm_i8).
//
// Mathematics: h = x + delta, z = h * weight, A = max|z|, r = 1 / sqrt(mean(h^2) + eps). The norm is y = r z, and the symmetric
// 8-bit form has scale max|y| / 127 = r A / 127 and q = round(y / scale) = round(z * (127 / A)): r cancels. So one pass over the row
// yields both reductions, and q, made of single fp32 operations on single elements, does not depend on the order of any sum. The maxima
// keep NaN, and a row's largest bits say whether it holds one or an infinity.
//
// Bound by memory: every value is read once and written once (norm of 9184 x 4096 fp32 with its delta 74.1 us = 6.6 TB/s, quantisation of
// 9184 x 4096 fp32 28.3 us = 6.6 TB/s, of 9184 x 14336 bf16 65 - 67 us = 5.9 - 6.1 TB/s; one row 1.8 - 2.1 us in a graph). A row stays in the
// registers of its threads between the reductions and the rounding. Close behind memory come the instructions, ~ 10 a value: sums,
// products and maxima take two values at a time, whole numbers come out of the low bits of a sum, 16-bit rows are searched without
// widening them (bf16, 14336 wide: 87 -> 66 us).
#include <algorithm>

#include "attn_internal.cuh"
#include "operand_memory.cuh"
#include "ptx_sm100.cuh"
#include "rows_ring.cuh"
#include "tcgen05_sm100.cuh"

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
    uint32_t whole16;      // rows are a multiple of 16 bytes long
    float eps;
    int32_t delta_dtype;
    uint32_t* status;
};

constexpr uint32_t kMaxThreads = 1024, kWarpRows = 4;  // threads of a block, rows of one whose rows are a warp's
constexpr uint32_t kInf = 0x7f800000u;
constexpr uint32_t kLost = 0xffffffffu;  // among rows' largest bits: a row that did not arrive
constexpr float kLiftTiny = 18446744073709551616.f;  // 2^64
// (four runs of eight values of x, delta and weight beside each other do not fit the 64 registers that 1024 threads have each)
constexpr uint32_t max_threads(bool norm, int vec, uint32_t chunks) { return norm && vec == 8 && chunks == 4 ? 512 : kMaxThreads; }

// VEC values as they lie in memory: fp32 words, or pairs of 16-bit values in the first half of them.
template <int VEC>
struct Raw {
    uint32_t w[VEC];
};
// VEC values from element i on. ALIGNED: all of them, in one run; otherwise one by one, n of them.
template <int VEC, bool ALIGNED>
__device__ __forceinline__ void load(Raw<VEC>& r, const void* p, size_t i, bool wide32, uint32_t n) {
    if (wide32) {
        const uint32_t* s = static_cast<const uint32_t*>(p) + i;
        if constexpr (ALIGNED) {
#pragma unroll
            for (int k = 0; k < VEC; k += 4) *reinterpret_cast<uint4*>(&r.w[k]) = *reinterpret_cast<const uint4*>(s + k);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < VEC; ++k) r.w[k] = k < n ? s[k] : 0u;
        }
    } else {
        const unsigned short* s = static_cast<const unsigned short*>(p) + i;
        if constexpr (ALIGNED) {
            if constexpr (VEC == 8) *reinterpret_cast<uint4*>(&r.w[0]) = *reinterpret_cast<const uint4*>(s);
            else *reinterpret_cast<uint2*>(&r.w[0]) = *reinterpret_cast<const uint2*>(s);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < VEC; k += 2)
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
        if constexpr (ALIGNED) {
#pragma unroll
            for (int k = 0; k < VEC; k += 4) *reinterpret_cast<float4*>(d + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < VEC; ++k)
                if (k < n) d[k] = v[k];
        }
    } else {
        unsigned short* d = static_cast<unsigned short*>(p) + i;
        uint32_t u[VEC / 2];
#pragma unroll
        for (int k = 0; k < VEC; k += 2) u[k / 2] = pack2<DT == ATTN_DTYPE_BF16>(v[k], v[k + 1]);
        if constexpr (ALIGNED) {
            if constexpr (VEC == 8) *reinterpret_cast<uint4*>(d) = make_uint4(u[0], u[1], u[2], u[3]);
            else *reinterpret_cast<uint2*>(d) = make_uint2(u[0], u[1]);
        } else {
#pragma unroll
            for (uint32_t k = 0; k < VEC; ++k)
                if (k < n) d[k] = static_cast<unsigned short>(u[k / 2] >> (16 * (k & 1)));
        }
    }
}

using tc::f32x2;

// h and z of VEC values as they were read, two at a time; the weight is the same for every row, and comes from L1.
template <int DT, bool NORM, bool DELTA, int VEC, bool ALIGNED>
__device__ __forceinline__ void combine(const RowsParams& p, uint32_t i, const Raw<VEC>& rx, const Raw<VEC>& rd, float (&h)[VEC], float (&z)[VEC]) {
    Raw<VEC> rw;
    if constexpr (NORM) load<VEC, ALIGNED>(rw, p.weight, i, true, p.dim - i);
    widen<VEC>(h, rx, DT);
    float d[VEC];
    if constexpr (DELTA) widen<VEC>(d, rd, p.delta_dtype);
#pragma unroll
    for (int k = 0; k < VEC; k += 2) {
        f32x2 v = tc::pack_f32x2(h[k], h[k + 1]);
        if constexpr (DELTA) {
            v = tc::add_f32x2(v, tc::pack_f32x2(d[k], d[k + 1]));
            tc::unpack_f32x2(v, h[k], h[k + 1]);
        }
        if constexpr (NORM) v = tc::mul_f32x2(v, tc::pack_f32x2(__uint_as_float(rw.w[k]), __uint_as_float(rw.w[k + 1])));
        tc::unpack_f32x2(v, z[k], z[k + 1]);
    }
}

// The largest |z| so far and two sums of h^2. NaN counts as more than any number.
struct Found {
    float top = 0.f;
    f32x2 sum = 0;  // (two zeros)
    uint32_t top16 = 0;  // of 16-bit rows as they are: two largest ones, side by side
};
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <bool NORM, int VEC>
__device__ __forceinline__ void count(const float (&h)[VEC], const float (&z)[VEC], Found& f) {
#pragma unroll
    for (int k = 0; k < VEC; k += 2) {
        f.top = max_abs(f.top, z[k], z[k + 1]);
        if constexpr (NORM) {
            const f32x2 v = tc::pack_f32x2(h[k], h[k + 1]);
            f.sum = tc::fma_f32x2(v, v, f.sum);
        }
    }
}
// The same of 16-bit values that nothing is done to, without widening them.
template <int DT, int VEC>
__device__ __forceinline__ void count16(const Raw<VEC>& r, Found& f) {
#pragma unroll
    for (int k = 0; k < VEC / 2; ++k) {
        const uint32_t v = r.w[k] & 0x7fff7fffu;
        if constexpr (DT == ATTN_DTYPE_BF16) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(f.top16) : "r"(v));
        else asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(f.top16) : "r"(v));
    }
}

// A row's reductions, the same in all its threads: the largest bits, among them a thread's `floor`, and the sum. s_top, s_sum: a value per
// warp, in other places for the block's next row.
template <int DT, bool NORM>
__device__ __forceinline__ void reduce_row(const Found& f, uint32_t floor, uint32_t& top, float& sum, bool whole_block, uint32_t* s_top,
                                           float* s_sum) {
    top = max(__float_as_uint(f.top), floor);
    if constexpr (!NORM && DT != ATTN_DTYPE_F32) {
        float lo, hi;
        tc::unpack2<DT == ATTN_DTYPE_BF16>(f.top16, lo, hi);
        top = max(top, max(__float_as_uint(lo), __float_as_uint(hi)));
    }
    float odd;
    tc::unpack_f32x2(f.sum, sum, odd);
    sum += odd;
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (NORM) {
#pragma unroll
        for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    }
    if (!whole_block) return;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) s_top[warp] = top, s_sum[warp] = sum;
    __syncthreads();
    const bool there = lane < blockDim.x / 32;
    top = __reduce_max_sync(0xffffffffu, there ? s_top[lane] : 0u);
    if constexpr (NORM) {
        sum = there ? s_sum[lane] : 0.f;
#pragma unroll
        for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    }
}

// What turns a row's z into whole numbers.
struct Rounding {
    float inverse;  // 127 / A, A lifted where tiny
    bool tiny;      // 127 / A leaves fp32's range below 2^-121: such rows are lifted first, which is exact
    bool bad;
};
// ... and its scale, which thread `first` writes.
template <bool NORM>
__device__ __forceinline__ Rounding finish_row(const RowsParams& p, uint32_t row, uint32_t top, float sum, bool first) {
    Rounding r;
    const float a = __uint_as_float(top);
    r.tiny = top < 0x03000000u;
    r.bad = top >= kInf || (NORM && !(sum < __uint_as_float(kInf)));
    r.inverse = top == 0 || r.bad ? 0.f : __fdiv_rn(127.f, r.tiny ? a * kLiftTiny : a);
    if (first) {
        float scale = a;
        if constexpr (NORM) scale *= __frcp_rn(sqrtf(sum / static_cast<float>(p.dim) + p.eps));
        p.scale[row] = r.bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(scale, 127.f);
    }
    return r;
}
// VEC whole numbers, `n` of which there are.
template <int VEC, bool ALIGNED>
__device__ __forceinline__ void put(int8_t* q, const float (&z)[VEC], const Rounding& r, uint32_t n) {
    uint32_t u[VEC / 4];
    // 1.5 * 2^23 puts the whole number next to a value of at most 2^22 (ties to the even one) into the low bits of the sum
    const f32x2 magic = tc::pack_f32x2(12582912.f, 12582912.f);
    const bool special = r.tiny || r.bad;
#pragma unroll
    for (int k = 0; k < VEC; k += 4) {
        float b[4];
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            float v0 = z[k + e], v1 = z[k + e + 1];
            if (special) v0 = r.bad ? 0.f : v0 * kLiftTiny, v1 = r.bad ? 0.f : v1 * kLiftTiny;
            // (the products one by one: a packed product and the packed sum behind it came out as if fused, rounded once)
            tc::unpack_f32x2(tc::add_f32x2(tc::pack_f32x2(__fmul_rn(v0, r.inverse), __fmul_rn(v1, r.inverse)), magic), b[e], b[e + 1]);
        }
        u[k / 4] = __byte_perm(__byte_perm(__float_as_uint(b[0]), __float_as_uint(b[1]), 0x0040),
                               __byte_perm(__float_as_uint(b[2]), __float_as_uint(b[3]), 0x0040), 0x5410);
    }
    if (ALIGNED || n >= VEC) {
        if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q) = make_uint2(u[0], u[1]);
        else *reinterpret_cast<uint32_t*>(q) = u[0];
    } else {
#pragma unroll
        for (uint32_t k = 0; k < VEC; ++k)
            if (k < n) q[k] = static_cast<int8_t>(u[k / 4] >> (8 * (k & 3)));
    }
}

// A row between its reductions and its rounding: z, or 16-bit values that nothing is done to as they are, in half the registers.
template <int DT, bool NORM, int VEC, int CHUNKS>
struct Kept {
    static constexpr bool kRaw = !NORM && DT != ATTN_DTYPE_F32;
    uint32_t raw[kRaw ? CHUNKS : 1][VEC / 2];
    float z[kRaw ? 1 : CHUNKS][VEC];
    __device__ __forceinline__ void keep(int c, const Raw<VEC>& r) {
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) raw[c][k] = r.w[k];
    }
    __device__ __forceinline__ const float (&values(int c))[VEC] {
        if constexpr (kRaw) {
            Raw<VEC> r;
#pragma unroll
            for (int k = 0; k < VEC / 2; ++k) r.w[k] = raw[c][k];
            widen<VEC>(z[0], r, DT);
            return z[0];
        } else {
            return z[c];
        }
    }
};

// A row per block, or per warp (narrow ones: no barrier). DT: type of x. NORM: weight, and the norm's factor in the scale. ALIGNED: rows may be read and written
// in runs of VEC values. CHUNKS runs a thread, or 0: a row longer than that, read twice.
template <int DT, bool NORM, bool DELTA, int VEC, int CHUNKS, bool ALIGNED>
__global__ void __launch_bounds__(max_threads(NORM, VEC, CHUNKS)) rows_i8_kernel(const __grid_constant__ RowsParams p) {
    grid_dep_launch_dependents();
    grid_dep_wait();
    __shared__ uint32_t s_top[kMaxThreads / 32];
    __shared__ float s_sum[kMaxThreads / 32];
    const bool whole_block = p.row_threads != 32;
    const uint32_t row = whole_block ? blockIdx.x : blockIdx.x * kWarpRows + (threadIdx.x >> 5);
    const uint32_t t = whole_block ? threadIdx.x : threadIdx.x & 31;
    if (row >= p.rows) return;
    const size_t x_row = row * p.x_stride, d_row = row * p.delta_stride, o_row = row * p.x_out_stride;
    const bool wide_delta = p.delta_dtype == ATTN_DTYPE_F32;
    int8_t* q = p.q + row * p.q_stride;
    // Without a branch, so that a thread's loads are requested one behind the other: past the row's end its last values again, or none.
    // (Branches around them had the compiler wait for one run before it asked for the next: 9184 x 4096 fp32 31 -> 49 us.)
    auto fetch = [&](uint32_t i, Raw<VEC>& rx, Raw<VEC>& rd) {
        const uint32_t n = i < p.dim ? p.dim - i : 0u;
        if constexpr (ALIGNED) i = min(i, p.dim - VEC);
        load<VEC, ALIGNED>(rx, p.x, x_row + i, DT == ATTN_DTYPE_F32, n);
        if constexpr (DELTA) load<VEC, ALIGNED>(rd, p.delta, d_row + i, wide_delta, n);
    };
    auto index = [&](uint32_t c) { return (c * p.row_threads + t) * VEC; };  // of run c
    Found found;
    uint32_t top;
    float sum;
    if constexpr (CHUNKS > 0) {
        Raw<VEC> rx[CHUNKS], rd[CHUNKS];
        Kept<DT, NORM, VEC, CHUNKS> kept;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) fetch(index(c), rx[c], rd[c]);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t i = index(c);
            if (i < p.dim) {
                if constexpr (kept.kRaw) {
                    count16<DT, VEC>(rx[c], found);
                    kept.keep(c, rx[c]);
                } else {
                    float h[VEC];
                    combine<DT, NORM, DELTA, VEC, ALIGNED>(p, i, rx[c], rd[c], h, kept.z[c]);
                    count<NORM, VEC>(h, kept.z[c], found);
                    if constexpr (DELTA)
                        if (p.x_out) store<VEC, DT, ALIGNED>(p.x_out, o_row + i, h, p.dim - i);
                }
            }
        }
        reduce_row<DT, NORM>(found, 0u, top, sum, whole_block, s_top, s_sum);
        const Rounding r = finish_row<NORM>(p, row, top, sum, t == 0);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t i = index(c);
            if (i < p.dim) put<VEC, ALIGNED>(q + i, kept.values(c), r, p.dim - i);
        }
    } else {
        Raw<VEC> rx, rd;
        float h[VEC], z[VEC];
        for (uint32_t i = index(0); i < p.dim; i += p.row_threads * VEC) {
            fetch(i, rx, rd);
            combine<DT, NORM, DELTA, VEC, ALIGNED>(p, i, rx, rd, h, z);
            count<NORM, VEC>(h, z, found);
        }
        reduce_row<DT, NORM>(found, 0u, top, sum, whole_block, s_top, s_sum);
        const Rounding r = finish_row<NORM>(p, row, top, sum, t == 0);
        for (uint32_t i = index(0); i < p.dim; i += p.row_threads * VEC) {  // (x_out may be x: nothing of the row was written before)
            fetch(i, rx, rd);
            combine<DT, NORM, DELTA, VEC, ALIGNED>(p, i, rx, rd, h, z);
            if constexpr (DELTA)
                if (p.x_out) store<VEC, DT, ALIGNED>(p.x_out, o_row + i, h, p.dim - i);
            put<VEC, ALIGNED>(q + i, z, r, p.dim - i);
        }
    }
}

// Many rows: a block takes every grid-th one, through a ring of whole rows in shared memory that bulk copies fill, so that reads go on
// while rows are reduced, rounded and stored. Rows lie on 16-byte boundaries and are a multiple of 16 bytes long.
constexpr uint32_t kSlots = 2;
constexpr uint32_t kRingTail = 16 * kMaxThreads / 32 + 64, kRingBytes = kMaxDynamicSmem - kRingTail;  // two turns' reductions, barriers; the rest
template <int DT, bool NORM, bool DELTA, int VEC, int CHUNKS>
__global__ void __launch_bounds__(kMaxThreads) rows_i8_ring_kernel(const __grid_constant__ RowsParams p) {
    extern __shared__ __align__(16) unsigned char smem[];
    uint32_t* s_top = reinterpret_cast<uint32_t*>(smem);  // [2][warps]: a thread is past the barrier of the row between before it
                                                          // writes where another may still have read
    float* s_sum = reinterpret_cast<float*>(s_top + 2 * (kMaxThreads / 32));
    const uint32_t full = smem_u32(smem) + 16 * (kMaxThreads / 32);
    unsigned char* ring = smem + kRingTail;  // [kSlots]{x, delta}
    const uint32_t x_bytes = p.dim * (DT == ATTN_DTYPE_F32 ? 4 : 2), d_bytes = DELTA ? p.dim * (p.delta_dtype == ATTN_DTYPE_F32 ? 4 : 2) : 0;
    const uint32_t slot_bytes = x_bytes + d_bytes;
    const uint32_t t = threadIdx.x;
    if (t == 0) {
        for (uint32_t s = 0; s < kSlots; ++s) mbar_init(full + 8 * s, 1);
        mbar_init_fence();
    }
    __syncthreads();
    grid_dep_launch_dependents();
    grid_dep_wait();
    const uint64_t policy = l2_policy_evict_first();
    auto request = [&](uint32_t n, uint32_t slot) {  // row n of this block
        if (t != 0) return;
        const uint32_t row = blockIdx.x + n * gridDim.x, dst = smem_u32(ring) + slot * slot_bytes, bar = full + 8 * slot;
        mbar_arrive_expect_tx(bar, slot_bytes);
        bulk_g2s(dst, static_cast<const unsigned char*>(p.x) + row * p.x_stride * (DT == ATTN_DTYPE_F32 ? 4 : 2), x_bytes, bar, policy);
        if constexpr (DELTA)
            bulk_g2s(dst + x_bytes, static_cast<const unsigned char*>(p.delta) + row * p.delta_stride * (p.delta_dtype == ATTN_DTYPE_F32 ? 4 : 2),
                     d_bytes, bar, policy);
    };
    auto wait = [&](uint32_t slot, uint32_t phase) { return mbar_wait(full + 8 * slot, phase); };
    const uint32_t mine = (p.rows - blockIdx.x + gridDim.x - 1) / gridDim.x;  // rows of this block
    Kept<DT, NORM, VEC, CHUNKS> kept;
    uint32_t top;
    float sum;
    auto reduce = [&](uint32_t n, uint32_t slot, bool there) {
        const uint32_t row = blockIdx.x + n * gridDim.x;
        const unsigned char* x = ring + slot * slot_bytes;
        Found found;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t i = (c * blockDim.x + t) * VEC;
            if (i < p.dim) {
                Raw<VEC> rx, rd;
                load<VEC, true>(rx, x, i, DT == ATTN_DTYPE_F32, VEC);
                if constexpr (kept.kRaw) {
                    count16<DT, VEC>(rx, found);
                    kept.keep(c, rx);
                } else {
                    float h[VEC];
                    if constexpr (DELTA) load<VEC, true>(rd, x + x_bytes, i, p.delta_dtype == ATTN_DTYPE_F32, VEC);
                    combine<DT, NORM, DELTA, VEC, true>(p, i, rx, rd, h, kept.z[c]);
                    count<NORM, VEC>(h, kept.z[c], found);
                    if constexpr (DELTA)
                        if (p.x_out && there) store<VEC, DT, true>(p.x_out, row * p.x_out_stride + i, h, VEC);
                }
            }
        }
        reduce_row<DT, NORM>(found, there ? 0u : kLost, top, sum, true, s_top + (n & 1) * (kMaxThreads / 32), s_sum + (n & 1) * (kMaxThreads / 32));
        return top != kLost;
    };
    auto finish = [&](uint32_t n) {
        const uint32_t row = blockIdx.x + n * gridDim.x;
        const Rounding r = finish_row<NORM>(p, row, top, sum, t == 0);
        int8_t* q = p.q + row * p.q_stride;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const uint32_t i = (c * blockDim.x + t) * VEC;
            if (i < p.dim) put<VEC, true>(q + i, kept.values(c), r, VEC);
        }
    };
    // A copy that did not arrive within the limit: the block's rows from there on become rows of NaN.
    auto lose = [&](uint32_t n) {
        if (t == 0 && p.status) atomicOr(p.status, ATTN_STATUS_WAIT_TIMEOUT);
        const float none[VEC] = {};
        for (; n < mine; ++n) {
            const uint32_t row = blockIdx.x + n * gridDim.x;
            const Rounding r = finish_row<NORM>(p, row, kLost, 0.f, t == 0);
#pragma unroll 1
            for (uint32_t i = t * VEC; i < p.dim; i += blockDim.x * VEC) put<VEC, true>(p.q + row * p.q_stride + i, none, r, VEC);
        }
    };
    run_ring<kSlots>(mine, request, wait, reduce, finish, lose);
}

uint32_t size_of(int32_t dtype) { return dtype == ATTN_DTYPE_F32 ? 4 : 2; }
bool is_float(int32_t d) { return d == ATTN_DTYPE_F32 || d == ATTN_DTYPE_F16 || d == ATTN_DTYPE_BF16; }

template <int DT, bool NORM, bool DELTA>
int launch_rows(RowsParams& p, uint32_t run, const DeviceInfo& dev, cudaStream_t stream) {
    constexpr int kWide = DT == ATTN_DTYPE_F32 ? 4 : 8;
    const bool aligned = run == kWide;
    const uint32_t vec = aligned ? kWide : 4;
    auto threads = [&](uint32_t chunks) { return ((p.dim + vec * chunks - 1) / (vec * chunks) + 31) / 32 * 32; };
    // Long rows in number: where few blocks of a row's threads fit an SM, the ring keeps the reads going. Quantisation of 9184 x 14336 bf16
    // 78.7 -> 65.7 us, 5500 x 14336 fp32 87 -> 62, 4000 x 28672 fp16 77 -> 56, the norm of 2000 x 16384 bf16 with an fp32 delta 57 -> 53. Blocks
    // of fewer threads do better without (quantisation of 9184 x 8192 bf16 36.6 for 51.3, of 4000 x 11008 25.1 for 30.5, the norm of 4096 x
    // 8192 fp32 67.0 for 79.1, bf16 40.6 for 42.4).
    constexpr uint32_t kRingFrom = !NORM ? 416 : DT == ATTN_DTYPE_F32 ? 544 : 512;
    constexpr uint32_t kRingChunks = NORM && DT != ATTN_DTYPE_F32 ? 2 : 4;
    const uint64_t slot = static_cast<uint64_t>(p.dim) * size_of(DT) + (DELTA ? static_cast<uint64_t>(p.dim) * size_of(p.delta_dtype) : 0);
    if (aligned && p.whole16 && threads(4) >= kRingFrom && threads(kRingChunks) <= kMaxThreads && 2 * slot <= kRingBytes &&
        p.rows > 2u * dev.sm_count) {
        p.row_threads = threads(kRingChunks);
        const uint32_t blocks = p.row_threads <= kMaxThreads / 2 && 2 * (kRingTail + kSlots * slot + 1024) <= 228 * 1024 ? 2 : 1;
        auto kernel = rows_i8_ring_kernel<DT, NORM, DELTA, kWide, kRingChunks>;
        B200_CUDA_TRY(allow_max_smem(kernel));
        B200_CUDA_TRY(launch_dependent(kernel, dim3(blocks * dev.sm_count), dim3(p.row_threads), kRingTail + kSlots * slot, stream, p));
        g_launch_count.fetch_add(1, std::memory_order_relaxed);
        return ATTN_OK;
    }
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
    void (*kernel)(RowsParams) = run == 1 ? (chunks ? rows_i8_kernel<DT, NORM, DELTA, 4, 4, false> : rows_i8_kernel<DT, NORM, DELTA, 4, 0, false>)
                                 : !aligned ? (chunks ? rows_i8_kernel<DT, NORM, DELTA, 4, 4, true> : rows_i8_kernel<DT, NORM, DELTA, 4, 0, true>)
                                 : chunks == 4 ? rows_i8_kernel<DT, NORM, DELTA, kWide, 4, true>
                                 : chunks == 2 ? rows_i8_kernel<DT, NORM, DELTA, kWide, 2, true>
                                 : chunks == 1 ? rows_i8_kernel<DT, NORM, DELTA, kWide, 1, true>
                                               : rows_i8_kernel<DT, NORM, DELTA, kWide, 0, true>;
    B200_CUDA_TRY(launch_dependent(kernel, dim3(grid), dim3(block), 0, stream, p));
    g_launch_count.fetch_add(1, std::memory_order_relaxed);
    return ATTN_OK;
}

template <bool NORM, bool DELTA>
int launch_rows_of(int32_t dtype, RowsParams& p, uint32_t run, const DeviceInfo& dev, cudaStream_t stream) {
    return dtype == ATTN_DTYPE_F32   ? launch_rows<ATTN_DTYPE_F32, NORM, DELTA>(p, run, dev, stream)
           : dtype == ATTN_DTYPE_F16 ? launch_rows<ATTN_DTYPE_F16, NORM, DELTA>(p, run, dev, stream)
                                     : launch_rows<ATTN_DTYPE_BF16, NORM, DELTA>(p, run, dev, stream);
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
    p.status = a->status;
    // Runs that a thread reads and writes at once: 8 values of 16 bits, 4 of any type, or single ones, as the rows' length, places and distances
    // allow. (Quantisation of 9184 x 14336 bf16 65.7 us, of 14335, one by one, 126; neighbouring values to neighbouring threads, whole
    // numbers in single bytes then, 254.)
    const uint64_t apart = n > 1 ? ~0ull : 0ull;
    auto fits = [&](uint64_t ptr, uint64_t stride, uint32_t size, uint32_t values) {
        return (ptr | (stride * size & apart)) % std::min<uint32_t>(16, size * values) == 0;
    };
    auto run_fits = [&](uint32_t values) {
        return d % values == 0 && fits(at(a->x), p.x_stride, xs, values) && at(a->weight) % 16 == 0 &&
               (!a->x_out || fits(at(a->x_out), p.x_out_stride, xs, values)) && (!a->delta || fits(at(a->delta), p.delta_stride, ds, values));
    };
    const uint32_t run = xs == 2 && run_fits(8) ? 8 : run_fits(4) ? 4 : 1;
    // whole rows by bulk copies
    p.whole16 = (xs * d | (a->delta ? ds * d : 0)) % 16 == 0 && (at(a->x) | (xs * p.x_stride & apart)) % 16 == 0 &&
                (!a->delta || (at(a->delta) | (ds * p.delta_stride & apart)) % 16 == 0);
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    if (!norm) return launch_rows_of<false, false>(a->x_dtype, p, run, dev, stream);
    return a->delta ? launch_rows_of<true, true>(a->x_dtype, p, run, dev, stream)
                    : launch_rows_of<true, false>(a->x_dtype, p, run, dev, stream);
}

}  // namespace
}  // namespace b200

extern "C" int attn_rmsnorm_i8(const AttnRowsI8Args* args, void* stream) { return b200::rows_i8(args, true, stream); }
extern "C" int attn_quantize_i8(const AttnRowsI8Args* args, void* stream) { return b200::rows_i8(args, false, stream); }
