// Rotary positions of a batch's tokens, both pair layouts, any table of (scaled) frequencies: q and k of every token are
// rotated, q goes to q_out, k and v into the token's cache row.
//
// Mathematics: pair i of a head's first rotary_dim values, (x[2i], x[2i+1]) interleaved or (x[i], x[i + rotary_dim/2]) in the half
// layout, turns by a = pos * inv_freq[i] and is multiplied by `factor`; the values behind rotary_dim are copied. The angle
// is reduced to a fraction of a turn in 64 bits: a product rounded to 32 bits is off by up to 4e-3 at position 100000. cos
// and sin and the rotation are fp32, each result is rounded once to the output's type.
//
// Bound by memory: every value is read once and written once. A thread owns a unit of two runs of VEC values, so that loads and
// stores are 16 bytes wide in either layout; a block owns a few tokens and makes their cos / sin table in
// shared memory once for all heads. One unit of one value pair (VEC = 1) serves sizes, strides and addresses that 16-byte
// accesses cannot. 9184 tokens of 32 + 8 + 8 heads of 128, bf16 (226 MB): 39.2 us = 5.8 TB/s; a step of eight tokens: 2.0 us in a graph.
// (Requesting the next unit while one turns costs registers and with them blocks: 44.5 us.)
#include "attn_internal.cuh"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

struct RopePosParams {
    void* q_out;
    const void* q;
    const void* k;
    const void* v;
    void* k_cache;
    void* v_cache;
    const float* inv_freq;
    const uint32_t* pos;
    const uint32_t* row;
    const uint32_t* seq;  // null: token i belongs to sequence i
    uint64_t q_stride, k_stride, v_stride, q_out_stride, kv_row_stride, kv_batch_stride;
    uint32_t tokens, n_heads, n_kv_heads, head_dim, rotary_dim, n_seqs, cache_rows;
    uint32_t tokens_per_block, units_per_head, units;  // units of one token: (n_heads + 2 n_kv_heads) * units_per_head
    uint32_t div_units, div_per_head, div_half;  // fast_div multipliers
    uint32_t half_layout;
    float factor;
    uint32_t* status;
};

constexpr int kThreads = 256;
constexpr uint32_t kMaxTokens = 8;  // of a block

// 16-bit and 32-bit floating types <-> fp32, N values at a time (N * size a power of two up to 16 bytes per access)
template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ void widen(float (&x)[N], const Vec<T, N>& t) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = to_f32<T>(t.v[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float (&x)[N]) {
    Vec<T, N> t;
#pragma unroll
    for (int i = 0; i < N; ++i) t.v[i] = from_f32<T>(x[i]);
    *reinterpret_cast<Vec<T, N>*>(p) = t;
}

// A unit as it was read: its values, and where it belongs.
template <typename TIn, int VEC>
struct Unit {
    Vec<TIn, VEC> a, b;
    uint32_t t, head, at0, at1;  // token of the block, head of its kind, offsets of the two runs in the head
    uint32_t kind;               // 0 q, 1 k, 2 v
    bool turn;
};

// grid (token groups, slices of a token's units)
template <typename TIn, typename TQ, typename TC, int VEC>
__global__ void __launch_bounds__(kThreads) rope_positions_kernel(const __grid_constant__ RopePosParams p) {
    extern __shared__ float2 s_cs[];  // [tokens_per_block][rotary_dim / 2] cos, sin (times the factor)
    __shared__ uint64_t s_row[kMaxTokens];  // cache offset of each token's row; kNoRow: there is none
    constexpr uint64_t kNoRow = ~0ull;
    grid_dep_launch_dependents();
    grid_dep_wait();
    const uint32_t t0 = blockIdx.x * p.tokens_per_block;
    const uint32_t nt = min(p.tokens_per_block, p.tokens - t0);
    const uint32_t half = p.rotary_dim / 2;
    const uint32_t q_units = p.n_heads * p.units_per_head, k_units = p.n_kv_heads * p.units_per_head;
    const uint32_t rot_units = half / VEC;  // of a head
    auto read = [&](uint32_t u, Unit<TIn, VEC>& x) {
        x.t = fast_div(u, p.div_units);
        const uint32_t w = u - x.t * p.units;
        x.kind = w < q_units ? 0u : w < q_units + k_units ? 1u : 2u;
        const uint32_t in_kind = x.kind == 0 ? w : x.kind == 1 ? w - q_units : w - q_units - k_units;
        x.head = fast_div(in_kind, p.div_per_head);
        const uint32_t part = in_kind - x.head * p.units_per_head;
        const bool turn = part < rot_units;
        // The two runs lie half of the turned (or of the copied) part of the head apart: partners in the half layout, and in either layout
        // neighbouring lanes read neighbouring runs (runs side by side: 41.9 us where this takes 39.2, 9184 tokens of 32 + 8 + 8 heads of 128).
        if (VEC == 1 && !p.half_layout) {
            x.at0 = part * 2;
            x.at1 = x.at0 + 1;
        } else {
            x.at0 = turn ? part * VEC : p.rotary_dim + (part - rot_units) * VEC;
            x.at1 = x.at0 + (turn ? half : (p.head_dim - p.rotary_dim) / 2);
        }
        x.turn = turn && x.kind != 2;
        const TIn* src = static_cast<const TIn*>(x.kind == 0 ? p.q : x.kind == 1 ? p.k : p.v) +
                         (t0 + x.t) * (x.kind == 0 ? p.q_stride : x.kind == 1 ? p.k_stride : p.v_stride) + static_cast<size_t>(x.head) * p.head_dim;
        x.a = *reinterpret_cast<const Vec<TIn, VEC>*>(src + x.at0);
        x.b = *reinterpret_cast<const Vec<TIn, VEC>*>(src + x.at1);
    };
    for (uint32_t i = threadIdx.x; i < nt * half; i += kThreads) {
        const uint32_t t = fast_div(i, p.div_half), j = i - t * half;
        constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)
        double turns = static_cast<double>(p.pos[t0 + t]) * (static_cast<double>(p.inv_freq[j]) * kTurn);
        turns -= rint(turns);
        float s, c;
        sincospif(2.f * static_cast<float>(turns), &s, &c);
        s_cs[i] = make_float2(c * p.factor, s * p.factor);
    }
    if (threadIdx.x < nt) {
        const uint32_t tok = t0 + threadIdx.x, seq = p.seq ? p.seq[tok] : tok, row = p.row[tok];
        const bool there = seq < p.n_seqs && row < p.cache_rows;
        s_row[threadIdx.x] = there ? seq * p.kv_batch_stride + row * p.kv_row_stride : kNoRow;
        if (!there && p.status) atomicOr(p.status, ATTN_STATUS_BAD_SHAPE);
    }
    __syncthreads();

    const uint32_t step = gridDim.y * kThreads, total = nt * p.units;
    for (uint32_t u = blockIdx.y * kThreads + threadIdx.x; u < total; u += step) {
        Unit<TIn, VEC> x;
        read(u, x);
        float a[VEC], b[VEC];
        widen<TIn, VEC>(a, x.a);
        widen<TIn, VEC>(b, x.b);
        if (x.turn) {
            const float2* cs = s_cs + x.t * half;
            if (p.half_layout || VEC == 1) {
                cs += p.half_layout ? x.at0 : x.at0 / 2;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float y = a[i], z = b[i];
                    a[i] = y * cs[i].x - z * cs[i].y;
                    b[i] = y * cs[i].y + z * cs[i].x;
                }
            } else {
#pragma unroll
                for (int i = 0; i + 1 < VEC; i += 2) {
                    const float y0 = a[i], z0 = a[i + 1], y1 = b[i], z1 = b[i + 1];
                    const float2 c0 = cs[(x.at0 + i) / 2], c1 = cs[(x.at1 + i) / 2];
                    a[i] = y0 * c0.x - z0 * c0.y;
                    a[i + 1] = y0 * c0.y + z0 * c0.x;
                    b[i] = y1 * c1.x - z1 * c1.y;
                    b[i + 1] = y1 * c1.y + z1 * c1.x;
                }
            }
        }
        const size_t in_row = static_cast<size_t>(x.head) * p.head_dim;
        if (x.kind == 0) {
            TQ* dst = static_cast<TQ*>(p.q_out) + (t0 + x.t) * p.q_out_stride + in_row;
            store<TQ, VEC>(dst + x.at0, a);
            store<TQ, VEC>(dst + x.at1, b);
        } else if (s_row[x.t] != kNoRow) {
            TC* dst = static_cast<TC*>(x.kind == 2 ? p.v_cache : p.k_cache) + s_row[x.t] + in_row;
            store<TC, VEC>(dst + x.at0, a);
            store<TC, VEC>(dst + x.at1, b);
        }
    }
}

template <typename TIn, typename TQ, typename TC, int VEC>
int launch(RopePosParams p, const DeviceInfo& dev, cudaStream_t stream) {
    p.units_per_head = p.head_dim / (2 * VEC);
    const uint64_t units = static_cast<uint64_t>(p.n_heads + 2ull * p.n_kv_heads) * p.units_per_head;
    if (units > (1u << 22)) return ATTN_ERR_UNSUPPORTED;
    p.units = static_cast<uint32_t>(units);
    // A block takes up to four tokens when there are enough of them to fill the GPU (one evaluation of a table entry per thread
    // at a rotary dimension of 128); fewer tokens are cut over blocks instead, a unit per thread.
    uint32_t tb = 4;
    while (tb > 1 && (p.tokens + tb - 1) / tb < 4u * dev.sm_count) tb /= 2;
    while (tb > 1 && tb * p.rotary_dim / 2 * sizeof(float2) > 32 * 1024) tb /= 2;
    if (units > 16384) tb = 1;  // (what fast_div divides by units stays below 2^32 / units)
    p.tokens_per_block = tb;
    p.div_units = tb == 1 ? 1u : divider(p.units);  // a multiplier of 1 gives 0: the block's only token
    p.div_per_head = divider(p.units_per_head);
    p.div_half = divider(p.rotary_dim / 2);
    const uint32_t groups = (p.tokens + tb - 1) / tb;
    const uint32_t slices_max = (tb * p.units + kThreads - 1) / kThreads;
    uint32_t slices = 1;
    while (slices < slices_max && static_cast<uint64_t>(groups) * slices < 4ull * dev.sm_count) ++slices;
    const size_t smem = static_cast<size_t>(tb) * (p.rotary_dim / 2) * sizeof(float2);
    auto kernel = rope_positions_kernel<TIn, TQ, TC, VEC>;
    B200_CUDA_TRY(launch_dependent(kernel, dim3(groups, slices), dim3(kThreads), smem, stream, p));
    g_launch_count.fetch_add(1, std::memory_order_relaxed);
    return ATTN_OK;
}

template <typename TIn, typename TQ, typename TC>
int launch_width(const RopePosParams& p, bool wide, const DeviceInfo& dev, cudaStream_t stream) {
    constexpr int kVec = 16 / sizeof(TIn);  // 16-byte loads
    return wide ? launch<TIn, TQ, TC, kVec>(p, dev, stream) : launch<TIn, TQ, TC, 1>(p, dev, stream);
}
template <typename TIn, typename TQ>
int launch_cache(const RopePosParams& p, int32_t kv_dtype, bool wide, const DeviceInfo& dev, cudaStream_t stream) {
    if (kv_dtype == ATTN_DTYPE_F16) return launch_width<TIn, TQ, __half>(p, wide, dev, stream);
    return launch_width<TIn, TQ, __nv_bfloat16>(p, wide, dev, stream);
}
template <typename TIn>
int launch_q(const RopePosParams& p, int32_t q_dtype, int32_t kv_dtype, bool wide, const DeviceInfo& dev, cudaStream_t stream) {
    if (q_dtype == ATTN_DTYPE_F32) return launch_cache<TIn, float>(p, kv_dtype, wide, dev, stream);
    if (q_dtype == ATTN_DTYPE_F16) return launch_cache<TIn, __half>(p, kv_dtype, wide, dev, stream);
    return launch_cache<TIn, __nv_bfloat16>(p, kv_dtype, wide, dev, stream);
}

bool float_dtype(int32_t d) { return d == ATTN_DTYPE_F32 || d == ATTN_DTYPE_F16 || d == ATTN_DTYPE_BF16; }
uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int attn_rope_positions(const AttnRopePositionsArgs* a, void* stream_v) {
    if (!a || !a->q_out || !a->q || !a->k || !a->v || !a->k_cache || !a->v_cache || !a->inv_freq || !a->pos || !a->row)
        return ATTN_ERR_INVALID_ARG;
    if (a->tokens == 0 || a->n_heads == 0 || a->n_kv_heads == 0 || a->head_dim == 0 || a->n_seqs == 0 || a->cache_rows == 0)
        return ATTN_ERR_INVALID_ARG;
    if (a->head_dim % 2 != 0 || a->rotary_dim % 2 != 0 || a->rotary_dim > a->head_dim) return ATTN_ERR_INVALID_ARG;
    if (!float_dtype(a->in_dtype) || !float_dtype(a->q_out_dtype)) return ATTN_ERR_INVALID_ARG;
    if (a->kv_dtype != ATTN_DTYPE_F16 && a->kv_dtype != ATTN_DTYPE_BF16) return ATTN_ERR_UNSUPPORTED;
    if (a->layout != ATTN_ROPE_INTERLEAVED && a->layout != ATTN_ROPE_HALF) return ATTN_ERR_INVALID_ARG;
    if (a->n_seqs > 1 && a->kv_batch_stride == 0) return ATTN_ERR_INVALID_ARG;
    if (!a->seq && a->tokens > a->n_seqs) return ATTN_ERR_INVALID_ARG;
    if (a->head_dim > 1024 || a->n_heads > 65536 || a->n_kv_heads > 65536) return ATTN_ERR_UNSUPPORTED;
    RopePosParams p{};
    p.q_out = a->q_out;
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.inv_freq = a->inv_freq;
    p.pos = a->pos;
    p.row = a->row;
    p.seq = a->seq;
    const uint64_t q_width = static_cast<uint64_t>(a->n_heads) * a->head_dim, kv_width = static_cast<uint64_t>(a->n_kv_heads) * a->head_dim;
    p.q_stride = a->q_stride ? a->q_stride : q_width;
    p.k_stride = a->k_stride ? a->k_stride : kv_width;
    p.v_stride = a->v_stride ? a->v_stride : kv_width;
    p.q_out_stride = a->q_out_stride ? a->q_out_stride : q_width;
    p.kv_row_stride = a->kv_row_stride ? a->kv_row_stride : kv_width;
    p.kv_batch_stride = a->kv_batch_stride;
    if (p.kv_row_stride < kv_width || p.q_out_stride < q_width) return ATTN_ERR_INVALID_ARG;  // outputs would overlap
    p.tokens = a->tokens;
    p.n_heads = a->n_heads;
    p.n_kv_heads = a->n_kv_heads;
    p.head_dim = a->head_dim;
    p.rotary_dim = a->rotary_dim ? a->rotary_dim : a->head_dim;
    p.n_seqs = a->n_seqs;
    p.cache_rows = a->cache_rows;
    p.half_layout = a->layout == ATTN_ROPE_HALF ? 1u : 0u;
    p.factor = a->factor != 0.f ? a->factor : 1.f;
    p.status = a->status;
    const uint32_t in_size = a->in_dtype == ATTN_DTYPE_F32 ? 4 : 2, q_size = a->q_out_dtype == ATTN_DTYPE_F32 ? 4 : 2;
    if ((bits(a->q) | bits(a->k) | bits(a->v)) % in_size || bits(a->q_out) % q_size || (bits(a->k_cache) | bits(a->v_cache)) % 2 ||
        (bits(a->inv_freq) | bits(a->pos) | bits(a->row) | bits(a->seq)) % 4)
        return ATTN_ERR_ALIGNMENT;
    // 16-byte accesses need units of whole vectors, and strides and addresses in 16 bytes (fp32: 4 values, else 8)
    const uint32_t vec = 16 / in_size;
    const bool wide = p.rotary_dim % (2 * vec) == 0 && p.head_dim % (2 * vec) == 0 &&
                      (p.q_stride | p.k_stride | p.v_stride | p.q_out_stride | p.kv_row_stride | p.kv_batch_stride) % 8 == 0 &&
                      (bits(a->q) | bits(a->k) | bits(a->v) | bits(a->q_out) | bits(a->k_cache) | bits(a->v_cache)) % 16 == 0;
    DeviceInfo dev{};
    const int rc = current_device_info(&dev);
    if (rc != ATTN_OK) return rc;
    if (dev.cc_major != 10) return ATTN_ERR_DEVICE;
    cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
    if (a->in_dtype == ATTN_DTYPE_F32) return launch_q<float>(p, a->q_out_dtype, a->kv_dtype, wide, dev, stream);
    if (a->in_dtype == ATTN_DTYPE_F16) return launch_q<__half>(p, a->q_out_dtype, a->kv_dtype, wide, dev, stream);
    return launch_q<__nv_bfloat16>(p, a->q_out_dtype, a->kv_dtype, wide, dev, stream);
}
