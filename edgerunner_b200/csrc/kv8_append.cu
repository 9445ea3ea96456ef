// er_qk_norm_rope and er_kv8_append: head norms, rotation and block quantisation of a ragged batch of rows.
//
// Both are one pass over the rows and bound by memory, if the instructions an element stay under about ten.  A row (one head of one token) is held by
// kLanes neighbouring lanes of a warp, each with one 16-byte vector of the first half of the row and the vector head_dim / 2 further, so that
// both members of a rotated pair are in one thread, and the sum of squares takes log2(kLanes) shuffles.  Angles: the frequencies (a 64-bit exp2 each,
// some 150 instructions of a slow pipe) once a CTA, the (cos, sin) of a token once for all of its heads, in shared memory in the order in which the
// lanes read them: 16 bytes (two pairs) a lane, lane beside lane.
//
// Measured (B200, bfloat16): norm + rotation of 32768 tokens of 32 + 8 heads of 128: 126 us = 5.33 TB/s = 0.81 of the copy bandwidth (157 us with the turns
// read from shared memory for every head); append of 16 x 2048 tokens of 8 kv heads, E4M3, blocks of 32: 61 us = 3.3 TB/s = 0.50: half of its issue
// slots are busy, and without the arithmetic (norm, rotation, maximum, encoding) the same copies take 40 us.
#include <algorithm>
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

int32_t kv8_check_device(const void* buffer) {
    int device = 0;
    cudaPointerAttributes at{};
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaPointerGetAttributes(&at, buffer);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return report_error(ER_ERR_CUDA, cudaGetErrorString(e));
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) return report_error(ER_ERR_INVALID_ARGUMENT, "a buffer is not device memory");
    if (at.device != device) return report_error(ER_ERR_INVALID_ARGUMENT, "the buffers live on another device than the current one");
    return ER_OK;
}

int32_t kv8_check(const er_kv8_cache* c, Kv8Cache* out) {
    if (!c->keys || !c->values || !c->key_scales || !c->value_scales || (!c->block_tables && c->block_table_width > 0) || !c->kv_lens)
        return report_error(ER_ERR_INVALID_ARGUMENT, "null buffer in er_kv8_cache");
    if (c->format != ER_KV8_E4M3 && c->format != ER_KV8_INT8) return report_error(ER_ERR_INVALID_ARGUMENT, "format must be ER_KV8_E4M3 or ER_KV8_INT8");
    if (c->head_dim != 64 && c->head_dim != 128) return report_error(ER_ERR_UNSUPPORTED, "head_dim of an 8-bit cache must be 64 or 128");
    if (c->scale_block != 16 && c->scale_block != 32 && c->scale_block != 64 && c->scale_block != 128)
        return report_error(ER_ERR_UNSUPPORTED, "scale_block must be 16, 32, 64 or 128");
    if (c->page_size == 0 || c->page_size % c->scale_block != 0 || c->page_size > (1u << 20))
        return report_error(ER_ERR_SHAPE, "page_size must be a multiple of scale_block (up to 2^20)");
    if (c->num_pages == 0 || c->num_pages > 0x7FFFFFFFu || c->num_kv_heads == 0 || c->num_kv_heads > 4096u)
        return report_error(ER_ERR_SHAPE, "num_pages and num_kv_heads must be positive (kv heads up to 4096)");
    if (c->num_seqs > 65536u) return report_error(ER_ERR_UNSUPPORTED, "num_seqs beyond 65536");
    if (c->block_table_width > c->block_table_stride) return report_error(ER_ERR_SHAPE, "block_table_width exceeds block_table_stride");
    if (static_cast<uint64_t>(c->block_table_width) * c->page_size > 0x7FFFFF00ull)
        return report_error(ER_ERR_UNSUPPORTED, "block tables address more than 2^31 rows of a sequence");
    if (static_cast<uint64_t>(c->num_pages) * c->num_kv_heads * c->page_size > 0x7FFFFFFFull)
        return report_error(ER_ERR_UNSUPPORTED, "the cache has more than 2^31 rows (pages * kv heads * page_size)");
    if (!kv8_aligned(c->keys) || !kv8_aligned(c->values)) return report_error(ER_ERR_INVALID_ARGUMENT, "keys and values must be 16-byte aligned");
    if (!kv8_aligned(c->key_scales, 4) || !kv8_aligned(c->value_scales, 4) || !kv8_aligned(c->block_tables, 4) || !kv8_aligned(c->kv_lens, 4) || !kv8_aligned(c->status, 4))
        return report_error(ER_ERR_INVALID_ARGUMENT, "scales, block_tables, kv_lens and status must be 4-byte aligned");
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
    int lanes, warps_per_token;          // lanes per row: a power of two >= head_dim / 2 / vector
    float eps;
    double log2_theta, inv_scaling;
};

// A table of turns: the i-th two pairs of all `vectors` lanes of VEC pairs lie side by side, (cos, cos, sin, sin) in 16 bytes.
template <int VEC>
__device__ __forceinline__ void put_turn(float* table, int pair, int vectors, float2 turn) {
    float* at = table + (((pair % VEC) >> 1) * vectors + pair / VEC) * 4 + (pair & 1);
    at[0] = turn.x;
    at[2] = turn.y;
}
// A lane's pairs of a row, turned; `turns`: the token's table at the lane's vector.
template <int VEC>
__device__ __forceinline__ void rotate(F2 (&a)[VEC / 2], F2 (&b)[VEC / 2], int vectors, const float* turns) {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
        const float4 cs = *reinterpret_cast<const float4*>(turns + i * vectors * 4);
        turn2<VEC>(a, b, i, pack2(cs.x, cs.y), pack2(cs.z, cs.w));
    }
}
__device__ __forceinline__ void make_frequencies(double* frequencies, int rotated, int half, double log2_theta, double inv_scaling) {
    for (int i = threadIdx.x; i < rotated; i += blockDim.x) frequencies[i] = rope_frequency(i, half, log2_theta, inv_scaling);
}

// A warp takes the heads of a token (or every warps_per_token-th set of them when there are few tokens), with its lane's turns and weights in
// registers, and kBatch sets of rows at a time, so that the loads of all are in flight together.
template <typename T>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const __grid_constant__ NormRope p) {
    extern __shared__ double shared8[];                            // frequencies [rotated], turns of each warp's token [vectors * VEC]
    constexpr int VEC = Act<T>::kVec, kBatch = 4;
    const float inv_dim = 1.f / static_cast<float>(p.head_dim);
    const int half = p.head_dim >> 1, vectors = half / VEC, table = half;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* turns = reinterpret_cast<float*>(shared8 + ((p.rotated + 1) & ~1)) + warp * 2 * table;
    const int rows_per_warp = 32 / p.lanes, sub = lane / p.lanes, vector = lane & (p.lanes - 1), first = vector * VEC;
    const bool own = first < half;
    make_frequencies(shared8, p.rotated, half, p.log2_theta, p.inv_scaling);
    __syncthreads();
    const int slots = gridDim.x * (kThreads / 32) / p.warps_per_token, share = warp % p.warps_per_token;
    for (int t = (static_cast<int>(blockIdx.x) * (kThreads / 32) + warp) / p.warps_per_token; t < p.num_tokens; t += slots) {
        if (p.rotated > 0) {
            const int position = __ldg(p.positions + t);
            __syncwarp();                                          // the last token's table has been read
            for (int i = lane; i < half; i += 32) put_turn<VEC>(turns, i, vectors, i < p.rotated ? rope_turn(position, shared8[i]) : make_float2(1.f, 0.f));
            __syncwarp();
        }
        F2 c2[VEC / 2], s2[VEC / 2];                               // cos, sin of the lane's pairs
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            float4 cs = make_float4(1.f, 1.f, 0.f, 0.f);
            if (own && p.rotated > 0) cs = *reinterpret_cast<const float4*>(turns + (i * vectors + vector) * 4);
            c2[i] = pack2(cs.x, cs.y);
            s2[i] = pack2(cs.z, cs.w);
        }
#pragma unroll 1
        for (int side = 0; side < 2; ++side) {
            const int heads = side ? p.heads[1] : p.heads[0];
            const float* w = side ? p.weight[1] : p.weight[0];
            F2 ca[VEC / 2], sa[VEC / 2], cb[VEC / 2], sb[VEC / 2];  // ... times the weights of the two members, sb negated
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                F2 wa = pack2(1.f, 1.f), wb = wa;
                if (own && w != nullptr) {
                    const float2 x = __ldg(reinterpret_cast<const float2*>(w + first) + i), y = __ldg(reinterpret_cast<const float2*>(w + half + first) + i);
                    wa = pack2(x.x, x.y);
                    wb = pack2(y.x, y.y);
                }
                ca[i] = mul2(c2[i], wa);
                sa[i] = mul2(s2[i], wa);
                cb[i] = mul2(c2[i], wb);
                sb[i] = mul2(mul2(s2[i], wb), pack2(-1.f, -1.f));
            }
            const int64_t in_head = side ? p.in_head[1] : p.in_head[0], out_head = side ? p.out_head[1] : p.out_head[0];
            const T* src = static_cast<const T*>(side ? p.in[1] : p.in[0]) + t * (side ? p.in_token[1] : p.in_token[0]) + first;
            T* dst = static_cast<T*>(side ? p.out[1] : p.out[0]) + t * (side ? p.out_token[1] : p.out_token[0]) + first;
            const int step = rows_per_warp * p.warps_per_token;
            for (int h0 = share * rows_per_warp + sub; h0 - sub < heads; h0 += kBatch * step) {
                uint4 va[kBatch], vb[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int h = h0 + k * step;
                    va[k] = vb[k] = make_uint4(0, 0, 0, 0);
                    if (own && h < heads) {
                        va[k] = *reinterpret_cast<const uint4*>(src + h * in_head);
                        vb[k] = *reinterpret_cast<const uint4*>(src + h * in_head + half);
                    }
                }
#pragma unroll
                for (int k = 0; k < kBatch; ++k) {
                    const int h = h0 + k * step;
                    F2 a[VEC / 2], b[VEC / 2];
                    unpack_pairs<T>(va[k], a);
                    unpack_pairs<T>(vb[k], b);
                    if (w != nullptr) {
                        float ss = square_sum<VEC>(a, b);
                        for (int off = p.lanes >> 1; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
                        const float f = rsqrtf(ss * inv_dim + p.eps);
                        const F2 f2 = pack2(f, f);
#pragma unroll
                        for (int i = 0; i < VEC / 2; ++i) { a[i] = mul2(a[i], f2); b[i] = mul2(b[i], f2); }
                    }
                    if (own && h < heads) {
                        float x[VEC], y[VEC];
#pragma unroll
                        for (int i = 0; i < VEC / 2; ++i) {
                            const F2 u = a[i];
                            a[i] = fma2(u, ca[i], mul2(b[i], sb[i]));
                            b[i] = fma2(u, sa[i], mul2(b[i], cb[i]));
                        }
                        floats_of(a, x);
                        floats_of(b, y);
                        *reinterpret_cast<uint4*>(dst + h * out_head) = Act<T>::pack(x);
                        *reinterpret_cast<uint4*>(dst + h * out_head + half) = Act<T>::pack(y);
                    }
                }
            }
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

__device__ __forceinline__ float max3_nan(float a, float b, float c) {   // a NaN wins
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// CTA = one block of scale_block tokens of one sequence; its warps walk the (kv head, side) pairs, scale_block / 8 warps to a pair (512
// threads for blocks of 128), a warp holding up to 8 rows of it in registers between the maximum and the encoding, so that a row is read once, while the
// loads of its next pair are in flight.  The norm factor of a row is positive, so it multiplies the row's maximum and the reciprocal of the
// scale, not the elements.  blockIdx.x numbers the blocks a sequence can touch (kv8_find_slot): sequence s owns the numbers from
// starts[s] / scale_block + 2 s on, always enough for a run of tokens that begins and ends inside a block; the rest return at once.  blockIdx.y spreads
// the pairs over more CTAs when there are few blocks.
constexpr int kWarpRows = 8, kAppendSlots = 2;
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <typename T, int D, bool E4M3>
__global__ void __launch_bounds__(512) kv8_append_kernel(const __grid_constant__ Kv8Append p) {
    extern __shared__ double shared8[];        // frequencies [rotated], turns [scale_block][D / 2], rings of the warps
    __shared__ float warp_max[2][16];
    constexpr int VEC = Act<T>::kVec, HALF = D / 2;
    constexpr int kLanes = HALF / VEC, kRowsPerPass = 32 / kLanes, kPasses = kWarpRows / kRowsPerPass;
    float* turns = reinterpret_cast<float*>(shared8 + HALF);
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
    const int block_pos = ((first_pos >> c.scale_shift) + j) << c.scale_shift;       // first position of the block
    if (block_pos >= len || block_pos < 0) return;
    const int page = kv8_page(c, seq, block_pos);
    if (page < 0) {
        if (threadIdx.x == 0) kv8_report(c, ER_ERR_OUT_OF_PAGES);
        return;
    }
    const int lead = max(0, first_pos - block_pos);        // rows of the block that were there before
    const int end = min(sb, len - block_pos);              // rows lead .. end are new
    const int token0 = begin + block_pos - first_pos;      // the call's token at row 0 of the block (negative below `lead`)
    const int64_t block_row = kv8_row(c, page, 0, kv8_in_page(c, block_pos));
    const int wpp = sb / kWarpRows, groups = static_cast<int>(blockDim.x >> 5) / wpp, group = warp / wpp;    // warps per pair, pairs at a time
    const int pairs = 2 * c.num_kv_heads;
    const int row0 = (warp % wpp) * kWarpRows, sub = lane / kLanes, vector = lane % kLanes, first = vector * VEC;
    // Where a warp's side lives.  With several pairs at a time the even groups take keys, the odd ones values, and this is worked out once.
    int side;
    const T* in_rows;              // of head 0: this lane's vector of its first row
    int64_t in_head, in_pass;
    uint8_t* code_rows;
    float* scale_row;
    auto take_side = [&](int s) {
        side = s;
        const int64_t token = s ? p.in_token[1] : p.in_token[0];
        in_head = s ? p.in_head[1] : p.in_head[0];
        in_rows = static_cast<const T*>(s ? p.in[1] : p.in[0]) + (token0 + row0 + sub) * token + first;
        in_pass = kRowsPerPass * token;
        code_rows = (s ? c.codes[1] : c.codes[0]) + (block_row + row0 + sub) * D + first;
        scale_row = (s ? c.scales[1] : c.scales[0]) + kv8_scale_at(c, block_row);
    };
    take_side(group & 1);
    const int scale_head = c.page_size >> c.scale_shift;                 // scales of a head in a page
    const int64_t code_head = static_cast<int64_t>(c.page_size) * D;
    bool is_new[kPasses];
#pragma unroll
    for (int ps = 0; ps < kPasses; ++ps) is_new[ps] = row0 + ps * kRowsPerPass + sub >= lead && row0 + ps * kRowsPerPass + sub < end;
    // A warp's rows come through its own ring in shared memory, the next pair's while this one is worked on (deeper rings measured the same,
    // registers are short); a lane reads what it copied, so no barrier is needed.
    uint4* ring = reinterpret_cast<uint4*>(turns + sb * D) + warp * (kAppendSlots * kPasses * 2 * 32) + lane;
    auto fetch = [&](int it, int slot) {           // one group, empty behind the last pair
        const int pr = it * groups + group;
        if (pr < pairs) {
            if (groups == 1) take_side(pr & 1);
            const T* src = in_rows + (pr >> 1) * in_head;
            const uint32_t to = smem_u32(ring + slot * (kPasses * 2 * 32));
#pragma unroll
            for (int ps = 0; ps < kPasses; ++ps) {                          // rows that are not new: zeros
                const T* from = is_new[ps] ? src + ps * in_pass : static_cast<const T*>(p.in[0]);
                const int bytes = is_new[ps] ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + ps * 1024), "l"(from), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + ps * 1024 + 512), "l"(from + HALF), "r"(bytes) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const int its = (pairs + groups - 1) / groups;
    int it = blockIdx.y;
#pragma unroll
    for (int k = 0; k < kAppendSlots - 1; ++k) fetch(it + k * gridDim.y, k);
    if (p.rotated > 0) {
        make_frequencies(shared8, p.rotated, HALF, p.log2_theta, p.inv_scaling);
        __syncthreads();
        for (int e = threadIdx.x; e < (end - lead) * HALF; e += blockDim.x) {
            const int t = e / HALF, pair = e % HALF;
            put_turn<VEC>(turns + t * D, pair, kLanes, pair < p.rotated ? rope_turn(block_pos + lead + t, shared8[pair]) : make_float2(1.f, 0.f));
        }
    }
    F2 wa[VEC / 2], wb[VEC / 2];
    if (p.weight != nullptr) {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            const float2 x = __ldg(reinterpret_cast<const float2*>(p.weight + first) + i), y = __ldg(reinterpret_cast<const float2*>(p.weight + HALF + first) + i);
            wa[i] = pack2(x.x, x.y);
            wb[i] = pack2(y.x, y.y);
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int turn = 0, slot = 0; it < its; it += gridDim.y, turn ^= 1) {         // uniform over the CTA
        const int pr = it * groups + group, head = pr >> 1;
        if (groups == 1) take_side(pr & 1);
        const int now = side;
        uint8_t* const dst = code_rows + head * code_head;
        float* const scale_at = scale_row + head * scale_head;
        const float before = lead > 0 && pr < pairs ? *scale_at : 0.f;
        F2 a[kPasses][VEC / 2], b[kPasses][VEC / 2];
        asm volatile("cp.async.wait_group %0;" ::"n"(kAppendSlots - 2) : "memory");
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps) {
            unpack_pairs<T>(ring[(slot * kPasses + ps) * 64], a[ps]);
            unpack_pairs<T>(ring[(slot * kPasses + ps) * 64 + 32], b[ps]);
        }
        fetch(it + (kAppendSlots - 1) * gridDim.y, slot == 0 ? kAppendSlots - 1 : slot - 1);
        slot = slot + 1 == kAppendSlots ? 0 : slot + 1;
        // ---- norm, rotation, the largest magnitude ----
        float factor[kPasses], mx = 0.f;
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps) {
            factor[ps] = 1.f;
            if (now == 0) {                                                // uniform over a warp
                if (p.weight != nullptr) {
                    float ss = square_sum<VEC>(a[ps], b[ps]);
#pragma unroll
                    for (int off = kLanes / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
                    factor[ps] = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
                    for (int i = 0; i < VEC / 2; ++i) { a[ps][i] = mul2(a[ps][i], wa[i]); b[ps][i] = mul2(b[ps][i], wb[i]); }
                }
                const int t = min(max(row0 + ps * kRowsPerPass + sub - lead, 0), end - lead - 1);    // rows of zeros turn by some token's angle
                if (p.rotated > 0) rotate<VEC>(a[ps], b[ps], kLanes, turns + t * D + vector * 4);
            }
            float up = 0.f, down = 0.f;
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) {
                float x, y;
                unpack2(a[ps][i], x, y);
                up = max3_nan(up, x, y);
                down = min3_nan(down, x, y);
                unpack2(b[ps][i], x, y);
                up = max3_nan(up, x, y);
                down = min3_nan(down, x, y);
            }
            // rows that are not new have no part in it: without an epsilon the factor of their zeros is infinite
            mx = max3_nan(mx, is_new[ps] ? up * factor[ps] : 0.f, is_new[ps] ? -down * factor[ps] : 0.f);
        }
        mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx) & 0x7FFFFFFFu));   // magnitudes compare like integers, NaN above all
        if (lane == 0) warp_max[turn][warp] = mx;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(wpp * 32) : "memory");      // the warps of the pair; the other half of the array is for the next pair
        for (int w = 0; w < wpp; ++w) mx = max3_nan(mx, warp_max[turn][group * wpp + w], 0.f);
        if (pr < pairs) {
            const float need = needed_scale<E4M3>(mx);
            const float scale = (before >= need) ? before : (isnan(before) ? before : need);  // a NaN on either side stays
            const float inv = reciprocal_scale<E4M3>(scale);
            const bool grown = lead > 0 && scale > before;
            auto store = [&](uint8_t* d, const float* x, const float* y) {
                uint32_t lo[VEC / 4], hi[VEC / 4];
#pragma unroll
                for (int i = 0; i < VEC; i += 4) {
                    lo[i / 4] = encode4<E4M3>(x[i], x[i + 1], x[i + 2], x[i + 3]);
                    hi[i / 4] = encode4<E4M3>(y[i], y[i + 1], y[i + 2], y[i + 3]);
                }
                if constexpr (VEC == 8) {
                    *reinterpret_cast<uint2*>(d) = make_uint2(lo[0], lo[1]);
                    *reinterpret_cast<uint2*>(d + HALF) = make_uint2(hi[0], hi[1]);
                } else {
                    *reinterpret_cast<uint32_t*>(d) = lo[0];
                    *reinterpret_cast<uint32_t*>(d + HALF) = hi[0];
                }
            };
            if (grown && row0 < lead) {                                     // the earlier rows' codes; a loop of its own, since few blocks come here
                const float ratio = __fdiv_rn(before, scale);
#pragma unroll 1
                for (int r = sub; r < min(kWarpRows, lead - row0); r += kRowsPerPass) {
                    uint8_t* d = dst + (r - sub) * D;
                    float x[VEC], y[VEC];
#pragma unroll
                    for (int i = 0; i < VEC; i += 4) {
                        decode4f<E4M3>(*reinterpret_cast<const uint32_t*>(d + i), x + i);
                        decode4f<E4M3>(*reinterpret_cast<const uint32_t*>(d + HALF + i), y + i);
                    }
#pragma unroll
                    for (int i = 0; i < VEC; ++i) { x[i] *= ratio; y[i] *= ratio; }
                    store(d, x, y);
                }
            }
            if (inv > 0.f) {
#pragma unroll
                for (int ps = 0; ps < kPasses; ++ps) {
                    float f = factor[ps] * inv;
                    if (isinf(f)) {                                         // elements below 2^-119: first the norm, then the scale
                        const F2 norm = pack2(factor[ps], factor[ps]);
#pragma unroll
                        for (int i = 0; i < VEC / 2; ++i) { a[ps][i] = mul2(a[ps][i], norm); b[ps][i] = mul2(b[ps][i], norm); }
                        f = inv;
                    }
                    const F2 f2 = pack2(f, f);
                    float x[VEC], y[VEC];
#pragma unroll
                    for (int i = 0; i < VEC / 2; ++i) { a[ps][i] = mul2(a[ps][i], f2); b[ps][i] = mul2(b[ps][i], f2); }
                    floats_of(a[ps], x);
                    floats_of(b[ps], y);
                    if (is_new[ps]) store(dst + ps * kRowsPerPass * D, x, y);
                }
            } else {                                                        // zeros, or a NaN scale: codes of zeros
                const float zeros[VEC] = {};
#pragma unroll 1
                for (int ps = 0; ps < kPasses; ++ps) {
                    const int row = row0 + ps * kRowsPerPass + sub;
                    if (row >= lead && row < end) store(dst + ps * kRowsPerPass * D, zeros, zeros);
                }
            }
            if (row0 == 0 && lane == 0) *scale_at = scale;
        }
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
    // Two CTAs fit an SM by their registers, and each begins with the frequencies: more of them cost a second start (4000 tokens in 500 CTAs 22.0 us, in 296 that
    // walk the tokens 20.6).  Few tokens spread their heads over two, four or eight warps each, as long as the CTAs fit at a time (300 tokens on
    // eight warps each, 300 CTAs: 9.9 us, on four, 150 CTAs: 6.5; on one, 38 CTAs: 7.5).
    const int most = 2 * kv8_sm_count();
    p.warps_per_token = 1;
    while (p.warps_per_token < 8 && static_cast<int64_t>(p.num_tokens) * p.warps_per_token * 2 <= most * (kThreads / 32)) p.warps_per_token *= 2;
    const int tokens_per_cta = (kThreads / 32) / p.warps_per_token;
    const int grid = std::min((p.num_tokens + tokens_per_cta - 1) / tokens_per_cta, std::max(most, 1));
    const size_t smem = ((p.rotated + 1) & ~1) * sizeof(double) + (kThreads / 32) * (p.head_dim / 2) * sizeof(float2);
    qk_norm_rope_kernel<T><<<grid, kThreads, smem, s>>>(p);
    return kv8_launched(cudaGetLastError(), "qk_norm_rope_kernel");
}

template <typename T, int D, bool E4M3>
int32_t launch_append(const Kv8Append& p, cudaStream_t s) {
    const int sb = p.cache.scale_block;
    const unsigned blocks = p.starts == nullptr ? p.cache.num_seqs : p.num_tokens / sb + 2u * p.cache.num_seqs;
    const int threads = sb == 128 ? 512 : 256;
    const int groups = threads / 32 / (sb / kWarpRows), steps = (2 * p.cache.num_kv_heads + groups - 1) / groups;
    // The pairs of a block are spread over as many CTAs as make two an SM with the blocks that have rows: each CTA works out its block's turns, so that more of
    // them cost more than they hide (blocks of 64, one CTA a step against this: 64 single tokens 16.5 / 11.5 us, 16 x 2048 tokens 189 / 65 us; one CTA a
    // block: a single token 22.2 / 4.3 us).
    const int64_t filled = p.starts == nullptr ? p.cache.num_seqs : p.num_tokens / sb + static_cast<int64_t>(p.cache.num_seqs);
    const dim3 grid(blocks, static_cast<unsigned>(std::min<int64_t>(steps, std::max<int64_t>(1, 2 * kv8_sm_count() / filled))));
    const size_t smem = D / 2 * sizeof(double) + static_cast<size_t>(sb) * (D / 2) * sizeof(float2) + threads / 32 * kAppendSlots * kWarpRows * D * sizeof(T);
    if (smem > 48 * 1024) {
        constexpr int kMost = D / 2 * 8 + 128 * (D / 2) * 8 + 16 * kAppendSlots * kWarpRows * D * static_cast<int>(sizeof(T));
        static_assert(kMost <= 232448, "append kernel exceeds the shared memory of an sm_100 CTA");
        static std::atomic<uint64_t> devices{0};
        const cudaError_t e = kv8_allow_smem(kv8_append_kernel<T, D, E4M3>, kMost, devices);
        if (e != cudaSuccess) return kv8_launched(e, "kv8_append_kernel");
    }
    kv8_append_kernel<T, D, E4M3><<<grid, threads, smem, s>>>(p);
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
    if (u->num_tokens > 0x7FFF0000u) return report_error(ER_ERR_UNSUPPORTED, "num_tokens beyond 2^31 - 2^16");   // a warp's next token number stays an int
    int32_t rc = check_rope(u->rope_theta, u->rope_scaling, u->partial_rotary_factor, u->rms_eps);
    if (rc != ER_OK) return rc;
    if (!kv8_aligned(u->q) || !kv8_aligned(u->q_out) || !kv8_aligned(u->k) || !kv8_aligned(u->k_out))
        return report_error(ER_ERR_INVALID_ARGUMENT, "q, k and the outputs must be 16-byte aligned");
    if (!kv8_aligned(u->q_norm_weight, 8) || !kv8_aligned(u->k_norm_weight, 8) || !kv8_aligned(u->positions, 4))      // weights are read in pairs
        return report_error(ER_ERR_INVALID_ARGUMENT, "norm weights must be 8-byte, positions 4-byte aligned");
    const int64_t strides[8] = {u->q_token_stride, u->q_head_stride, u->q_out_token_stride, u->q_out_head_stride,
                                u->k_token_stride, u->k_head_stride, u->k_out_token_stride, u->k_out_head_stride};
    if (!strides_ok(u->type, strides, u->k ? 8 : 4)) return report_error(ER_ERR_INVALID_ARGUMENT, "strides must be multiples of 16 bytes");
    if (!kv8_rows_apart(u->q_out_token_stride, u->q_out_head_stride, u->num_tokens, u->num_heads, u->head_dim) ||
        (u->k && !kv8_rows_apart(u->k_out_token_stride, u->k_out_head_stride, u->num_tokens, u->num_kv_heads, u->head_dim)))
        return report_error(ER_ERR_SHAPE, "rows of an output overlap");
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
    rc = kv8_check_device(u->q);
    if (rc != ER_OK) return rc;
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
    if (!kv8_aligned(u->k_norm_weight, 8) || !kv8_aligned(u->query_starts, 4))
        return report_error(ER_ERR_INVALID_ARGUMENT, "the norm weight must be 8-byte, query_starts 4-byte aligned");
    const int64_t strides[4] = {u->k_token_stride, u->k_head_stride, u->v_token_stride, u->v_head_stride};
    if (!strides_ok(u->type, strides, 4)) return report_error(ER_ERR_INVALID_ARGUMENT, "strides must be multiples of 16 bytes");
    if (u->num_tokens > 0x7FFFFF00u) return report_error(ER_ERR_UNSUPPORTED, "num_tokens beyond 2^31");
    if (!u->query_starts && u->num_tokens != cache->num_seqs) return report_error(ER_ERR_SHAPE, "without query_starts num_tokens must be num_seqs");
    rc = kv8_check_device(cache->keys);
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
