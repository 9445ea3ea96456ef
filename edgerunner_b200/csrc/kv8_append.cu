// er_qk_norm_rope and er_kv8_append: head norms, rotation and block quantisation of a ragged batch of rows.
//
// Both are one pass over the rows and bound by memory.  A row (one head of one token) is held by kLanes neighbouring lanes of a warp, each
// with one 16-byte vector of the first half of the row and the vector head_dim / 2 further, so that both members of a rotated pair are in
// one thread, and the sum of squares takes log2(kLanes) shuffles.  The (cos, sin) table of a CTA's tokens is built once in shared memory
// and used by all of their heads: a sincos of a 64-bit angle costs about 60 instructions, and there are 8 to 40 heads to a token.
#include <cmath>
#include <cstdio>

#include "kv8.cuh"

namespace er {

int32_t kv8_launched(cudaError_t e, const char* kernel) {
    count_kernel_launch();
    if (e == cudaSuccess) return ER_OK;
    char msg[200];
    std::snprintf(msg, sizeof(msg), "%s: %s", kernel, cudaGetErrorString(e));
    return report_error(ER_ERR_CUDA, msg);
}

int32_t kv8_check_device(const er_kv8_cache* c) {
    int device = 0;
    cudaPointerAttributes at{};
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaPointerGetAttributes(&at, c->keys);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return report_error(ER_ERR_CUDA, cudaGetErrorString(e));
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) return report_error(ER_ERR_INVALID_ARGUMENT, "keys is not device memory");
    if (at.device != device) return report_error(ER_ERR_INVALID_ARGUMENT, "the cache lives on another device than the current one");
    return ER_OK;
}

int32_t kv8_check(const er_kv8_cache* c, Kv8Cache* out) {
    if (!c->keys || !c->values || !c->key_scales || !c->value_scales || !c->block_tables || !c->kv_lens)
        return report_error(ER_ERR_INVALID_ARGUMENT, "null buffer in er_kv8_cache");
    if (c->format != ER_KV8_E4M3 && c->format != ER_KV8_INT8) return report_error(ER_ERR_INVALID_ARGUMENT, "format must be ER_KV8_E4M3 or ER_KV8_INT8");
    if (c->head_dim != 64 && c->head_dim != 128) return report_error(ER_ERR_UNSUPPORTED, "head_dim of an 8-bit cache must be 64 or 128");
    if (c->scale_block != 16 && c->scale_block != 32 && c->scale_block != 64 && c->scale_block != 128)
        return report_error(ER_ERR_UNSUPPORTED, "scale_block must be 16, 32, 64 or 128");
    if (c->page_size == 0 || c->page_size % c->scale_block != 0 || c->page_size > (1u << 20))
        return report_error(ER_ERR_SHAPE, "page_size must be a multiple of scale_block (up to 2^20)");
    if (c->num_pages == 0 || c->num_pages > 0x7FFFFFFFu || c->num_kv_heads == 0 || c->num_kv_heads > 65535u)
        return report_error(ER_ERR_SHAPE, "num_pages and num_kv_heads must be positive (kv heads up to 65535)");
    if (c->num_seqs > 65536u) return report_error(ER_ERR_UNSUPPORTED, "num_seqs beyond 65536");
    if (c->block_table_width > c->block_table_stride) return report_error(ER_ERR_SHAPE, "block_table_width exceeds block_table_stride");
    if (static_cast<uint64_t>(c->block_table_width) * c->page_size > 0x7FFFFF00ull)
        return report_error(ER_ERR_UNSUPPORTED, "block tables address more than 2^31 rows of a sequence");
    if (static_cast<uint64_t>(c->num_pages) * c->num_kv_heads * c->page_size > 0x7FFFFFFFull)
        return report_error(ER_ERR_UNSUPPORTED, "the cache has more than 2^31 rows (pages * kv heads * page_size)");
    if (!kv8_aligned(c->keys) || !kv8_aligned(c->values)) return report_error(ER_ERR_INVALID_ARGUMENT, "keys and values must be 16-byte aligned");
    out->codes[0] = c->keys; out->codes[1] = c->values;
    out->scales[0] = c->key_scales; out->scales[1] = c->value_scales;
    out->tables = c->block_tables; out->lens = c->kv_lens; out->status = c->status;
    out->num_pages = static_cast<int>(c->num_pages); out->page_size = static_cast<int>(c->page_size);
    out->scale_block = static_cast<int>(c->scale_block); out->num_kv_heads = static_cast<int>(c->num_kv_heads);
    out->num_seqs = static_cast<int>(c->num_seqs); out->table_width = static_cast<int>(c->block_table_width);
    out->table_stride = c->block_table_stride;
    out->scale_shift = c->scale_block == 16 ? 4 : c->scale_block == 32 ? 5 : c->scale_block == 64 ? 6 : 7;
    out->page_magic = ~0ull / c->page_size + 1;   // page_size >= 16
    return ER_OK;
}

namespace {

constexpr int kThreads = 256;

struct NormRope {
    const void* in[2];
    void* out[2];
    int64_t in_token[2], in_head[2], out_token[2], out_head[2];
    const float* weight[2];
    const int32_t* positions;
    int heads[2];
    int num_tokens, head_dim, rotated;   // rotated: pairs
    int tokens_per_cta, lanes;           // lanes per row: a power of two >= head_dim / 2 / vector
    float eps;
    double log2_theta, inv_scaling;
};

// The two vectors of a row in registers -> normed and rotated.  `turns`: the row's token's table, nullptr: no rotation.
template <int VEC>
__device__ __forceinline__ void norm_rotate(float (&a)[VEC], float (&b)[VEC], int first, int half, int rotated, int lanes, const float* weight,
                                            float eps, const float2* turns) {
    if (weight != nullptr) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
        for (int off = lanes >> 1; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
        const float f = rsqrtf(ss / static_cast<float>(2 * half) + eps);
        if (first < half) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                a[i] *= f * __ldg(weight + first + i);
                b[i] *= f * __ldg(weight + half + first + i);
            }
        }
    }
    if (turns != nullptr && first < rotated) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (first + i < rotated) {
                const float2 cs = turns[first + i];
                const float x = a[i], y = b[i];
                a[i] = x * cs.x - y * cs.y;
                b[i] = x * cs.y + y * cs.x;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ NormRope p) {
    extern __shared__ float2 turns[];   // [tokens_per_cta][rotated]
    constexpr int VEC = Act<T>::kVec;
    const int half = p.head_dim >> 1;
    const int t0 = static_cast<int>(blockIdx.x) * p.tokens_per_cta;
    const int nt = min(p.tokens_per_cta, p.num_tokens - t0);
    const int rows_per_warp = 32 / p.lanes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane / p.lanes, first = (lane & (p.lanes - 1)) * VEC;
    const int heads = p.heads[0] + p.heads[1], rows = nt * heads;
    const int step = (kThreads / 32) * rows_per_warp * gridDim.y;
    for (int e = threadIdx.x; e < nt * p.rotated; e += kThreads) {
        const int t = e / p.rotated, pair = e - t * p.rotated;
        turns[e] = rope_turn(__ldg(p.positions + t0 + t), rope_frequency(pair, half, p.log2_theta, p.inv_scaling));
    }
    __syncthreads();
    for (int r0 = (static_cast<int>(blockIdx.y) * (kThreads / 32) + warp) * rows_per_warp; r0 < rows; r0 += step) {
        const int r = r0 + sub;
        const bool on = r < rows && first < half;
        const int t = on ? r / heads : 0;
        int h = on ? r - t * heads : 0;
        const int side = h >= p.heads[0] ? 1 : 0;
        h -= side ? p.heads[0] : 0;
        float a[VEC] = {}, b[VEC] = {};
        if (on) {
            const T* src = static_cast<const T*>(p.in[side]) + (t0 + t) * p.in_token[side] + h * p.in_head[side] + first;
            Act<T>::unpack(*reinterpret_cast<const uint4*>(src), a);
            Act<T>::unpack(*reinterpret_cast<const uint4*>(src + half), b);
        }
        // lanes of one warp may hold a query and a key row: a missing weight is a factor of one
        const bool any_norm = p.weight[0] != nullptr || p.weight[1] != nullptr;
        if (any_norm) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
            for (int off = p.lanes >> 1; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
            const float* w = p.weight[side];
            if (on && w != nullptr) {
                const float f = rsqrtf(ss / static_cast<float>(p.head_dim) + p.eps);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    a[i] *= f * __ldg(w + first + i);
                    b[i] *= f * __ldg(w + half + first + i);
                }
            }
        }
        if (on) {
            norm_rotate<VEC>(a, b, first, half, p.rotated, 1, nullptr, 0.f, p.rotated > 0 ? turns + t * p.rotated : nullptr);
            T* dst = static_cast<T*>(p.out[side]) + (t0 + t) * p.out_token[side] + h * p.out_head[side] + first;
            *reinterpret_cast<uint4*>(dst) = Act<T>::pack(a);
            *reinterpret_cast<uint4*>(dst + half) = Act<T>::pack(b);
        }
    }
}

struct Kv8Append {
    Kv8Cache cache;
    const void* in[2];                 // k, v
    int64_t in_token[2], in_head[2];
    const int32_t* starts;
    const float* weight;
    int num_tokens, rotated;
    float eps;
    double log2_theta, inv_scaling;
};

// CTA = one block of scale_block tokens of one sequence; its warps walk the (side, kv head) pairs, scale_block / 16 warps to a pair, a
// warp holding up to 16 rows of it in registers (16 * D / 32 values a lane) between the maximum and the encoding, so that a row is read
// once.  blockIdx.x numbers the blocks a sequence can touch without a prefix sum over the batch: sequence s owns the numbers from
// starts[s] / scale_block + 2 s on, always enough for a run of tokens that begins and ends inside a block; the rest return at once.
// blockIdx.y spreads the pairs over more CTAs when there are few blocks.
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(kThreads, 2) kv8_append_kernel(const __grid_constant__ Kv8Append p) {
    extern __shared__ float2 turns[];   // [scale_block][rotated]
    __shared__ uint32_t warp_max[kThreads / 32];
    constexpr int VEC = Act<T>::kVec, HALF = D / 2;
    constexpr int kLanes = HALF / VEC, kRowsPerPass = 32 / kLanes, kPasses = 16 / kRowsPerPass;
    const Kv8Cache& c = p.cache;
    const int sb = c.scale_block;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // ---- which sequence, which block ----
    int seq, begin, count, j;
    if (p.starts == nullptr) {
        seq = blockIdx.x;
        begin = seq; count = 1; j = 0;
    } else {
        const int slot = blockIdx.x;
        seq = kv8_find_slot(p.starts, c.num_seqs, slot, [&](int start, int s) { return (start >> c.scale_shift) + 2 * s; });
        begin = __ldg(p.starts + seq);
        count = __ldg(p.starts + seq + 1) - begin;
        j = slot - ((begin >> c.scale_shift) + 2 * seq);
    }
    if (count == 0 || j < 0) return;
    const int len = __ldg(c.lens + seq), first_pos = len - count;
    if (count < 0 || begin < 0 || begin > p.num_tokens - count || first_pos < 0) {
        if (threadIdx.x == 0) kv8_report(c, ER_ERR_SHAPE);
        return;
    }
    const int block_pos = (first_pos / sb + j) * sb;       // first position of the block
    if (block_pos >= len) return;
    const int page = kv8_page(c, seq, block_pos);
    if (page < 0) {
        if (threadIdx.x == 0) kv8_report(c, ER_ERR_OUT_OF_PAGES);
        return;
    }
    const int lead = max(0, first_pos - block_pos);        // rows of the block that were there before
    const int end = min(sb, len - block_pos);              // rows lead .. end are new
    const int in_page = kv8_in_page(c, block_pos);
    const int token0 = begin + block_pos - first_pos;      // the call's token at row 0 of the block (negative below `lead`)
    for (int e = threadIdx.x; e < (end - lead) * p.rotated; e += kThreads) {
        const int t = e / p.rotated, pair = e - t * p.rotated;
        turns[e] = rope_turn(block_pos + lead + t, rope_frequency(pair, HALF, p.log2_theta, p.inv_scaling));
    }
    if (p.rotated > 0) __syncthreads();
    const int wpp = sb / 16, groups = (kThreads / 32) / wpp;           // warps per pair, pairs at a time
    const int pairs = 2 * c.num_kv_heads;
    const int row0 = (warp % wpp) * 16, sub = lane / kLanes, first = (lane % kLanes) * VEC;
    for (int base = static_cast<int>(blockIdx.y) * groups; base < pairs; base += groups * gridDim.y) {   // uniform over the CTA
        const int pr = base + warp / wpp;
        const bool on = pr < pairs;
        const int side = on ? pr & 1 : 0, head = on ? pr >> 1 : 0;
        float a[kPasses][VEC], b[kPasses][VEC];
        uint32_t mx = 0;
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps) {
            const int row = row0 + ps * kRowsPerPass + sub;
#pragma unroll
            for (int i = 0; i < VEC; ++i) a[ps][i] = b[ps][i] = 0.f;
            if (on && row >= lead && row < end) {
                const T* src = static_cast<const T*>(p.in[side]) + (token0 + row) * p.in_token[side] + head * p.in_head[side] + first;
                Act<T>::unpack(__ldg(reinterpret_cast<const uint4*>(src)), a[ps]);
                Act<T>::unpack(__ldg(reinterpret_cast<const uint4*>(src + HALF)), b[ps]);
            }
        }
        const int64_t at = kv8_row(c, page, head, in_page);
        float* scale_at = c.scales[side] + kv8_scale_at(c, at);
        const float old = on && lead > 0 ? *scale_at : 0.f;
        if (side == 0) {                                                // uniform over a warp
#pragma unroll
            for (int ps = 0; ps < kPasses; ++ps) {
                const int row = row0 + ps * kRowsPerPass + sub;
                const int t = min(max(row - lead, 0), end - lead - 1);  // rows of zeros turn by some token's angle
                norm_rotate<VEC>(a[ps], b[ps], first, HALF, p.rotated, kLanes, p.weight, p.eps, p.rotated > 0 ? turns + t * p.rotated : nullptr);
            }
        }
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps)
#pragma unroll
            for (int i = 0; i < VEC; ++i)   // magnitudes compare like integers, infinities and NaN above all others
                mx = max(mx, max(__float_as_uint(a[ps][i]) & 0x7FFFFFFFu, __float_as_uint(b[ps][i]) & 0x7FFFFFFFu));
        mx = __reduce_max_sync(0xffffffffu, mx);
        if (wpp > 1) {
            if (lane == 0) warp_max[warp] = mx;
            __syncthreads();
            for (int w = 0; w < wpp; ++w) mx = max(mx, warp_max[warp / wpp * wpp + w]);
            __syncthreads();                                            // read by all before the next pair's maxima
        }
        if (!on) continue;
        const float need = needed_scale<E4M3>(__uint_as_float(mx));
        const float scale = (old >= need) ? old : (isnan(old) ? old : need);   // a NaN on either side stays
        const float inv = scale > 0.f ? __frcp_rn(scale) : 0.f;         // NaN scale: codes of zeros
        uint8_t* dst = c.codes[side] + at * D;
        const bool grown = lead > 0 && scale > old;
        const float ratio = grown ? __fdiv_rn(old, scale) : 1.f;
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps) {
            const int row = row0 + ps * kRowsPerPass + sub;
            uint8_t* d = dst + row * D + first;
            if (row >= lead && row < end) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    a[ps][i] = inv > 0.f ? a[ps][i] * inv : 0.f;
                    b[ps][i] = inv > 0.f ? b[ps][i] * inv : 0.f;
                }
            } else if (row < lead && grown) {
#pragma unroll
                for (int i = 0; i < VEC; i += 4) {
                    decode4f<E4M3>(*reinterpret_cast<const uint32_t*>(d + i), a[ps] + i);
                    decode4f<E4M3>(*reinterpret_cast<const uint32_t*>(d + HALF + i), b[ps] + i);
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) { a[ps][i] *= ratio; b[ps][i] *= ratio; }
            } else {
                continue;
            }
            uint32_t lo[VEC / 4], hi[VEC / 4];
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                lo[i / 4] = encode4<E4M3>(a[ps][i], a[ps][i + 1], a[ps][i + 2], a[ps][i + 3]);
                hi[i / 4] = encode4<E4M3>(b[ps][i], b[ps][i + 1], b[ps][i + 2], b[ps][i + 3]);
            }
            if constexpr (VEC == 8) {
                *reinterpret_cast<uint2*>(d) = make_uint2(lo[0], lo[1]);
                *reinterpret_cast<uint2*>(d + HALF) = make_uint2(hi[0], hi[1]);
            } else {
                *reinterpret_cast<uint32_t*>(d) = lo[0];
                *reinterpret_cast<uint32_t*>(d + HALF) = hi[0];
            }
        }
        if (row0 == 0 && lane == 0) *scale_at = scale;
    }
}

size_t element_bytes(uint32_t type) { return type == ER_TYPE_FLOAT32 ? 4 : 2; }

bool strides_ok(uint32_t type, const int64_t* s, int n) {
    const int64_t vec = 16 / static_cast<int64_t>(element_bytes(type));
    for (int i = 0; i < n; ++i)
        if (s[i] < 0 || s[i] % vec != 0) return false;
    return true;
}

int32_t check_rope(float theta, float scaling, float partial, float eps) {
    if (!(partial >= 0.f && partial <= 1.f)) return report_error(ER_ERR_INVALID_ARGUMENT, "partial_rotary_factor must be in [0, 1]");
    if (partial > 0.f && !(theta > 0.f && std::isfinite(theta) && scaling > 0.f && std::isfinite(scaling)))
        return report_error(ER_ERR_INVALID_ARGUMENT, "rope_theta and rope_scaling must be positive");
    if (!(eps >= 0.f)) return report_error(ER_ERR_INVALID_ARGUMENT, "rms_eps must not be negative");
    return ER_OK;
}

template <typename T>
int32_t launch_norm_rope(NormRope& p, cudaStream_t s) {
    const int vecs = p.head_dim / 2 / Act<T>::kVec;
    p.lanes = 1;
    while (p.lanes < vecs) p.lanes *= 2;
    // One token to a CTA while that leaves SMs idle, then up to four: the table of four tokens is one sincos a thread.  With fewer tokens
    // than a quarter of the SMs the rows of a token are spread over several CTAs, each with the table of its own.
    p.tokens_per_cta = p.num_tokens <= 2048 ? 1 : 4;
    const int rows_per_pass = kThreads / p.lanes;
    const int rows = p.tokens_per_cta * (p.heads[0] + p.heads[1]);
    const int split = p.num_tokens <= 37 ? (rows + rows_per_pass - 1) / rows_per_pass : 1;
    const dim3 grid((p.num_tokens + p.tokens_per_cta - 1) / p.tokens_per_cta, split);
    qk_norm_rope_kernel<T><<<grid, kThreads, static_cast<size_t>(p.tokens_per_cta) * p.rotated * sizeof(float2), s>>>(p);
    return kv8_launched(cudaGetLastError(), "qk_norm_rope_kernel");
}

template <typename T, int D, bool E4M3>
int32_t launch_append(const Kv8Append& p, cudaStream_t s) {
    const int sb = p.cache.scale_block;
    const unsigned blocks = p.starts == nullptr ? p.cache.num_seqs : p.num_tokens / sb + 2u * p.cache.num_seqs;
    const int groups = (kThreads / 32) / (sb / 16), steps = (2 * p.cache.num_kv_heads + groups - 1) / groups;
    const dim3 grid(blocks, blocks >= 592 ? 1 : steps);   // 592: four CTAs' worth of blocks for each SM
    const size_t smem = static_cast<size_t>(sb) * p.rotated * sizeof(float2);   // up to 64 KB
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kv8_append_kernel<T, D, E4M3>, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
        if (e != cudaSuccess) return kv8_launched(e, "kv8_append_kernel");
    }
    kv8_append_kernel<T, D, E4M3><<<grid, kThreads, smem, s>>>(p);
    return kv8_launched(cudaGetLastError(), "kv8_append_kernel");
}

template <typename T>
int32_t launch_append_shape(const Kv8Append& p, uint32_t head_dim, bool e4m3, cudaStream_t s) {
    if (head_dim == 128) return e4m3 ? launch_append<T, 128, true>(p, s) : launch_append<T, 128, false>(p, s);
    return e4m3 ? launch_append<T, 64, true>(p, s) : launch_append<T, 64, false>(p, s);
}

}  // namespace
}  // namespace er

extern "C" int32_t er_qk_norm_rope(const er_qk_norm_rope_params* u, void* stream) {
    using namespace er;
    if (!u || !u->q || !u->q_out) return report_error(ER_ERR_INVALID_ARGUMENT, "null argument");
    if ((u->k == nullptr) != (u->k_out == nullptr)) return report_error(ER_ERR_INVALID_ARGUMENT, "k and k_out come together");
    if (u->type > ER_TYPE_BFLOAT16) return report_error(ER_ERR_INVALID_ARGUMENT, "type must be one of ER_TYPE_*");
    if (u->head_dim == 0 || u->head_dim % 16 != 0 || u->head_dim > 256) return report_error(ER_ERR_UNSUPPORTED, "head_dim must be a multiple of 16 up to 256");
    if (u->num_heads == 0 || u->num_heads > 65535u || (u->k && (u->num_kv_heads == 0 || u->num_kv_heads > 65535u)))
        return report_error(ER_ERR_SHAPE, "head counts must be between 1 and 65535");
    if (u->num_tokens > 0x7FFFFF00u) return report_error(ER_ERR_UNSUPPORTED, "num_tokens beyond 2^31");
    int32_t rc = check_rope(u->rope_theta, u->rope_scaling, u->partial_rotary_factor, u->rms_eps);
    if (rc != ER_OK) return rc;
    if (!kv8_aligned(u->q) || !kv8_aligned(u->q_out) || !kv8_aligned(u->k) || !kv8_aligned(u->k_out))
        return report_error(ER_ERR_INVALID_ARGUMENT, "q, k and the outputs must be 16-byte aligned");
    const int64_t strides[8] = {u->q_token_stride, u->q_head_stride, u->q_out_token_stride, u->q_out_head_stride,
                                u->k_token_stride, u->k_head_stride, u->k_out_token_stride, u->k_out_head_stride};
    if (!strides_ok(u->type, strides, u->k ? 8 : 4)) return report_error(ER_ERR_INVALID_ARGUMENT, "strides must be multiples of 16 bytes");
    NormRope p{};
    p.in[0] = u->q; p.in[1] = u->k; p.out[0] = u->q_out; p.out[1] = u->k_out;
    p.in_token[0] = u->q_token_stride; p.in_head[0] = u->q_head_stride; p.out_token[0] = u->q_out_token_stride; p.out_head[0] = u->q_out_head_stride;
    p.in_token[1] = u->k_token_stride; p.in_head[1] = u->k_head_stride; p.out_token[1] = u->k_out_token_stride; p.out_head[1] = u->k_out_head_stride;
    p.weight[0] = u->q_norm_weight; p.weight[1] = u->k ? u->k_norm_weight : nullptr;
    p.positions = u->positions;
    p.heads[0] = static_cast<int>(u->num_heads); p.heads[1] = u->k ? static_cast<int>(u->num_kv_heads) : 0;
    p.num_tokens = static_cast<int>(u->num_tokens); p.head_dim = static_cast<int>(u->head_dim);
    p.rotated = static_cast<int>(static_cast<float>(u->head_dim / 2) * u->partial_rotary_factor);
    if (p.rotated > 0 && !u->positions) return report_error(ER_ERR_INVALID_ARGUMENT, "positions are needed for the rotation");
    p.eps = u->rms_eps;
    p.log2_theta = p.rotated > 0 ? std::log2(static_cast<double>(u->rope_theta)) : 0.0;
    p.inv_scaling = p.rotated > 0 ? 1.0 / static_cast<double>(u->rope_scaling) : 0.0;
    if (u->num_tokens == 0) return ER_OK;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (u->type) {
        case ER_TYPE_FLOAT32: return launch_norm_rope<float>(p, s);
        case ER_TYPE_FLOAT16: return launch_norm_rope<__half>(p, s);
        default: return launch_norm_rope<__nv_bfloat16>(p, s);
    }
}

extern "C" int32_t er_kv8_append(const er_kv8_cache* cache, const er_kv8_append_params* u, void* stream) {
    using namespace er;
    if (!cache || !u || !u->k || !u->v) return report_error(ER_ERR_INVALID_ARGUMENT, "null argument");
    if (u->type > ER_TYPE_BFLOAT16) return report_error(ER_ERR_INVALID_ARGUMENT, "type must be one of ER_TYPE_*");
    Kv8Append p{};
    int32_t rc = kv8_check(cache, &p.cache);
    if (rc != ER_OK) return rc;
    rc = check_rope(u->rope_theta, u->rope_scaling, u->partial_rotary_factor, u->rms_eps);
    if (rc != ER_OK) return rc;
    if (!kv8_aligned(u->k) || !kv8_aligned(u->v)) return report_error(ER_ERR_INVALID_ARGUMENT, "k and v must be 16-byte aligned");
    const int64_t strides[4] = {u->k_token_stride, u->k_head_stride, u->v_token_stride, u->v_head_stride};
    if (!strides_ok(u->type, strides, 4)) return report_error(ER_ERR_INVALID_ARGUMENT, "strides must be multiples of 16 bytes");
    if (u->num_tokens > 0x7FFFFF00u) return report_error(ER_ERR_UNSUPPORTED, "num_tokens beyond 2^31");
    if (!u->query_starts && u->num_tokens != cache->num_seqs) return report_error(ER_ERR_SHAPE, "without query_starts num_tokens must be num_seqs");
    rc = kv8_check_device(cache);
    if (rc != ER_OK) return rc;
    if (u->num_tokens == 0 || cache->num_seqs == 0) return ER_OK;
    p.in[0] = u->k; p.in[1] = u->v;
    p.in_token[0] = u->k_token_stride; p.in_head[0] = u->k_head_stride; p.in_token[1] = u->v_token_stride; p.in_head[1] = u->v_head_stride;
    p.starts = u->query_starts;
    p.weight = u->k_norm_weight;
    p.num_tokens = static_cast<int>(u->num_tokens);
    p.rotated = static_cast<int>(static_cast<float>(cache->head_dim / 2) * u->partial_rotary_factor);
    p.eps = u->rms_eps;
    p.log2_theta = p.rotated > 0 ? std::log2(static_cast<double>(u->rope_theta)) : 0.0;
    p.inv_scaling = p.rotated > 0 ? 1.0 / static_cast<double>(u->rope_scaling) : 0.0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = cache->format == ER_KV8_E4M3;
    switch (u->type) {
        case ER_TYPE_FLOAT32: return launch_append_shape<float>(p, cache->head_dim, e4m3, s);
        case ER_TYPE_FLOAT16: return launch_append_shape<__half>(p, cache->head_dim, e4m3, s);
        default: return launch_append_shape<__nv_bfloat16>(p, cache->head_dim, e4m3, s);
    }
}
