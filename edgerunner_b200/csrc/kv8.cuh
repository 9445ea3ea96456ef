// Shared pieces of the 8-bit block-scaled paged cache (er_kv8_*) and of er_qk_norm_rope: activation types, code formats,
// page lookup, rotation tables.
//
// A page holds page_size tokens of every kv head: codes [page][kv head][slot][dim] (one byte each), scales
// [page][kv head][slot / scale_block] (float32).  Element = code * scale, code = an E4M3 float or an int8.
#pragma once

#include <cuda_bf16.h>

#include <atomic>
#include <cmath>

#include "../../include/er_kv.h"
#include "er_common.cuh"

namespace er {

constexpr int kKv8Unit = 16;   // tokens that share one scale at least; every scale_block is a multiple

// ---- activations: 16-byte vectors of T <-> float ----
template <typename T> struct Act;
template <> struct Act<float> {
    static constexpr int kVec = 4;
    static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
        f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <> struct Act<__half> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ void unpack(const uint4& v, float* f) { unpack8(v, f); }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        uint4 v;
        __half2* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        return v;
    }
};
template <> struct Act<__nv_bfloat16> {
    static constexpr int kVec = 8;
    static __device__ __forceinline__ void unpack(const uint4& v, float* f) {   // a bfloat16 is the upper half of a float
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        uint4 v;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        return v;
    }
};
// two neighbouring outputs of one row
__device__ __forceinline__ void store_pair(float* p, float a, float b) { *reinterpret_cast<float2*>(p) = make_float2(a, b); }
__device__ __forceinline__ void store_pair(__half* p, float a, float b) { *reinterpret_cast<__half2*>(p) = __floats2half2_rn(a, b); }
__device__ __forceinline__ void store_pair(__nv_bfloat16* p, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(a, b); }

// Two float32 lanes in one instruction.
struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 pack2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(F2 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
// A lane's pairs (a[i], b[i]) turned by the angles with cosines c[i] and sines s[i].
template <int VEC>
__device__ __forceinline__ void turn2(F2 (&a)[VEC / 2], F2 (&b)[VEC / 2], int i, F2 c, F2 s) {
    const F2 x = a[i], y = b[i], minus = pack2(-1.f, -1.f);
    a[i] = fma2(mul2(y, minus), s, mul2(x, c));
    b[i] = fma2(x, s, mul2(y, c));
}
template <int VEC>
__device__ __forceinline__ float square_sum(const F2 (&a)[VEC / 2], const F2 (&b)[VEC / 2]) {
    F2 x = pack2(0.f, 0.f), y = x;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) { x = fma2(a[i], a[i], x); y = fma2(b[i], b[i], y); }
    float u, v;
    unpack2(add2(x, y), u, v);
    return u + v;
}
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4& v, F2 (&x)[Act<T>::kVec / 2]) {
    float f[Act<T>::kVec];
    Act<T>::unpack(v, f);
#pragma unroll
    for (int i = 0; i < Act<T>::kVec / 2; ++i) x[i] = pack2(f[2 * i], f[2 * i + 1]);
}
template <int N>
__device__ __forceinline__ void floats_of(const F2 (&x)[N], float* f) {
#pragma unroll
    for (int i = 0; i < N; ++i) unpack2(x[i], f[2 * i], f[2 * i + 1]);
}

// ---- codes ----
// Four values (already divided by the scale) -> four codes, the first in the low byte.  Rounded to nearest even, saturating.
template <bool E4M3>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (E4M3) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
        return static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
    } else {
        const int x = max(-128, min(127, __float2int_rn(a))), y = max(-128, min(127, __float2int_rn(b)));
        const int z = max(-128, min(127, __float2int_rn(c))), w = max(-128, min(127, __float2int_rn(d)));
        return (x & 255) | ((y & 255) << 8) | ((z & 255) << 16) | (static_cast<uint32_t>(w) << 24);
    }
}
// Four codes -> two half2 (exact: an E4M3 value and an int8 both fit a half).
template <bool E4M3>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (E4M3) {
        asm("{ .reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b; }" : "=r"(lo), "=r"(hi) : "r"(w));
    } else {   // bytes + 128 as the low mantissa bits of 1024 + u, minus 1152
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
        lo = *reinterpret_cast<const uint32_t*>(&x);
        hi = *reinterpret_cast<const uint32_t*>(&y);
    }
}
template <bool E4M3>
__device__ __forceinline__ void decode4f(uint32_t w, float* f) {
    uint32_t a, b;
    decode4<E4M3>(w, a, b);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
}
// The scale that a block with largest magnitude `amax` needs.  E4M3: the smallest power of two with amax / scale <= 448, so that
// a growing scale moves the exponents of the codes already there and rounds nothing but what falls below the smallest code (E4M3's
// precision does not depend on the scale).  int8: amax / 127.  0 for a block of zeros, NaN for one with an infinity or a NaN.
template <bool E4M3>
__device__ __forceinline__ float needed_scale(float amax) {
    if (!(amax <= 3.402823466e38f)) return __uint_as_float(0x7FC00000u);
    if (amax == 0.f) return 0.f;
    if constexpr (E4M3) {
        const uint32_t b = __float_as_uint(amax);   // 448 = 1.75 * 2^8: one exponent more where the mantissa is above 1.75
        const int e = static_cast<int>(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
        return __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23);   // at least 2^-126: its reciprocal is finite
    } else {
        return fmaxf(__fdiv_rn(amax, 127.f), 1.17549435e-38f);
    }
}

// 1 / scale, 0 for a scale of zero or NaN.  A power of two at or above 2^-126: by its exponent.
template <bool E4M3>
__device__ __forceinline__ float reciprocal_scale(float scale) {
    if (!(scale > 0.f)) return 0.f;
    if constexpr (E4M3) {
        const uint32_t b = __float_as_uint(scale);
        if ((b & 0x7FFFFFu) == 0u && b < 0x7E800000u) return __uint_as_float(0x7F000000u - b);
    }
    return __frcp_rn(scale);
}

// ---- pages ----
struct Kv8Cache {
    uint8_t* codes[2];      // keys, values
    float* scales[2];
    const int32_t* tables;
    const int32_t* lens;
    int* status;
    int num_pages, page_size, scale_block, num_kv_heads, num_seqs, table_width;
    int scale_shift;        // log2(scale_block)
    uint64_t page_magic;    // ceil(2^64 / page_size)
    int64_t table_stride;
};
// tok / page_size by a multiplication (exact below 2^31: the error of tok * ceil(2^64 / d) / 2^64 is under tok / 2^64 < 1 / d)
__device__ __forceinline__ int kv8_page_index(const Kv8Cache& c, int tok) {
    return static_cast<int>(__umul64hi(static_cast<uint64_t>(static_cast<uint32_t>(tok)), c.page_magic));
}
__device__ __forceinline__ int kv8_in_page(const Kv8Cache& c, int tok) { return tok - kv8_page_index(c, tok) * c.page_size; }
// Page of token `tok` of sequence `seq`, or -1.
__device__ __forceinline__ int kv8_page(const Kv8Cache& c, int seq, int tok) {
    const int i = kv8_page_index(c, tok);
    if (i >= c.table_width) return -1;
    const int p = __ldg(c.tables + seq * c.table_stride + i);
    return p >= 0 && p < c.num_pages ? p : -1;
}
// Row of slot `in_page` of (page, head), and the scale of a row.
__device__ __forceinline__ int64_t kv8_row(const Kv8Cache& c, int page, int head, int in_page) {
    return (static_cast<int64_t>(page) * c.num_kv_heads + head) * c.page_size + in_page;
}
__device__ __forceinline__ int64_t kv8_scale_at(const Kv8Cache& c, int64_t row) { return row >> c.scale_shift; }
// Work of a ragged batch is numbered without a prefix sum over it: sequence s owns the numbers from first(starts[s], s) on, `first` growing
// with both and leaving each sequence room enough.  The sequence that owns `slot`, by whole warps: 32 probes at a time, one round of loads for
// up to 32 sequences, two for 1024.
template <typename First>
__device__ __forceinline__ int kv8_find_slot(const int32_t* starts, int num_seqs, int slot, First first) {
    int lo = 0, n = num_seqs;                    // it is one of lo .. lo + n
    while (n > 1) {
        const int step = (n + 31) / 32, s = lo + static_cast<int>(threadIdx.x & 31) * step;
        const bool below = s < lo + n && first(__ldg(starts + min(s, num_seqs - 1)), s) <= slot;
        const int k = max(__popc(__ballot_sync(0xffffffffu, below)) - 1, 0);
        n = min(step, lo + n - (lo + k * step));
        lo += k * step;
    }
    return lo;
}
__device__ __forceinline__ void kv8_report(const Kv8Cache& c, int code) {
    if (c.status != nullptr) atomicExch(c.status, code);
}

// ---- rotation ----
// (cos, sin) of position * theta^(-pair / half) / scaling.  The angle is formed and reduced in 64 bits: in 32 it is off by
// position * 2^-24 radians, 0.06 at a million tokens.
__device__ __forceinline__ double rope_frequency(int pair, int half, double log2_theta, double inv_scaling) {
    return exp2(-static_cast<double>(pair) / static_cast<double>(half) * log2_theta) * inv_scaling;
}
__device__ __forceinline__ float2 rope_turn(int position, double frequency) {
    double u = static_cast<double>(position) * frequency * 0.15915494309189533577;   // whole turns
    u = 2.0 * (u - rint(u));
    const float half_turns = static_cast<float>(u), rest = static_cast<float>(u - half_turns) * 3.14159265f;   // what float32 leaves of the angle: up to 1e-7 radians
    float s, c;
    sincospif(half_turns, &s, &c);
    return make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
}

// ---- host ----
int32_t report_error(int32_t code, const char* message);   // er_kv.cu: records the thread's last-error text
void count_kernel_launch();                                 // er_kv.cu: bumps er_kernel_launch_count()
int32_t kv8_check(const er_kv8_cache* cache, Kv8Cache* out);                // kv8_append.cu: the fields; fills the kernels' form
int32_t kv8_check_device(const void* buffer);                                // it is the current device's
int32_t kv8_launched(cudaError_t e, const char* kernel);                     // status of the launch just made
int kv8_sm_count();                                                          // kv8_decode.cu: SMs of the current device, 0 without one
int32_t kv8_check_attention(const er_kv8_cache* c, const er_kv8_attention_params* u);
int32_t kv8_check_workspace(const er_kv8_attention_params* u, int64_t need);
int64_t kv8_decode_workspace(const er_kv8_cache* c, const er_kv8_attention_params* u, bool ragged);
int32_t kv8_launch_decode(const Kv8Cache& cache, const er_kv8_cache* c, const er_kv8_attention_params* u, bool ragged, int few_rows, cudaStream_t s);
// Dynamic shared memory beyond 48 KB has to be allowed once for each kernel and device.  `most`: the largest size that any call of the kernel asks for.
template <typename Kernel>
inline cudaError_t kv8_allow_smem(Kernel kernel, int most, std::atomic<uint64_t>& devices) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < 64 && (devices.load(std::memory_order_acquire) >> device & 1u) != 0)) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess && device < 64) devices.fetch_or(1ull << device, std::memory_order_release);
    return e;
}
// The window as the kernels take it: 0 (none) where no sequence is longer.  kv8_check_attention keeps position - window, with positions down to -num_tokens
// for queries in front of row 0, inside an int.
inline uint64_t kv8_table_rows(const er_kv8_cache* c) { return static_cast<uint64_t>(c->block_table_width) * c->page_size; }
inline int kv8_window(const er_kv8_cache* c, const er_kv8_attention_params* u) {
    return u->sliding_window >= kv8_table_rows(c) ? 0 : static_cast<int>(u->sliding_window);
}
inline float kv8_scale_log2(float softmax_scale, uint32_t head_dim) {       // scores in units of log2
    return (softmax_scale > 0.f ? softmax_scale : 1.f / std::sqrt(static_cast<float>(head_dim))) * 1.4426950408889634f;
}
// Rows of an output do not overlap (heads beside each other inside a token, or tokens inside a head).
inline bool kv8_rows_apart(int64_t token_stride, int64_t head_stride, int64_t tokens, int64_t heads, int64_t head_dim) {
    if (tokens <= 1 && heads <= 1) return true;
    if (heads <= 1) return token_stride >= head_dim;
    if (tokens <= 1) return head_stride >= head_dim;
    const bool heads_inside = head_stride >= head_dim && token_stride >= head_stride * (heads - 1) + head_dim;
    return heads_inside || (token_stride >= head_dim && head_stride >= token_stride * (tokens - 1) + head_dim);
}
inline bool kv8_aligned(const void* p, uintptr_t bytes = 16) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

}  // namespace er
