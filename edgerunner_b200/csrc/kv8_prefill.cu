// er_kv8_attention_prefill on the 5th-generation tensor cores: a ragged batch of prompts or prompt chunks, causal by position, over an 8-bit
// block-scaled paged cache.
//
// Mathematics.  s = (q . ck) a scale with a the key scale of 16 or more rows, w = 2^(s log2 e - m) b / R with b the value scale and R a power of two near
// the largest one so far of the blocks that the row sees, o = R sum_i w_i cv_i / sum_i (w_i R / b_i).  Codes are exact in fp16, q and w are rounded to
// it (float16 outputs 3.0e-4 from 64 bits instead of 2.1e-4; a second half of w would lengthen the softmax, which bounds the kernel), sums are float32.  Neither scale costs an operation a score: a multiplies the factor inside exp2's argument, log2(b / R) is part of its offset,
// and the sum of 16 weights is divided by b / R once.
//
// One CTA owns two tiles of 128 query rows of a (sequence, kv head): row r is query r / group, head r % group, any group.  The tensor pipe takes 1024
// clocks for 128 tokens of a tile, exp2 (16 a clock and SM) as long, so the two tiles take turns: while one is in its softmax the products of the other run.
//   warps 0-3, 4-7   softmax of tile 0, 1: a thread is a row.  Reads S from tensor memory twice (maximum, then weights), writes w as fp16 over S.  The
//                    running maximum may lag by 2^8 before the row of O is rescaled in tensor memory, so that this is rare.
//   warps 8-11, 13-15  fetch codes and write them as fp16 into the operand layout: a conversion in the loader reads 1 byte an element from L2
//                    and serves 256 rows.
//   warp 12          one lane issues the products: S_i = Q_i K^T (M128 N128 K16 steps, operands in shared memory), O_i += W_i V (A from tensor memory).
//                    Only products of one shape into one accumulator are ordered by their issue, so S_i of the next tokens, which goes over W_i, waits
//                    until O_i += W_i V has been executed (head size 128; with 64 there is room for W beside S).
// Tensor memory: S_0, S_1 at columns 0, 128; O_0, O_1 from 256 on, D columns each; W_i over S_i, or (head size 64) W_0, W_1 at 384, 448.  Shared
// memory: Q (2 x 128 rows), a ring of K / V tiles of 128 tokens, scales.
// Every wait is bounded (2 s): then the status word is set, the rest of the waits are skipped, the products that have been issued are waited for (3 s), tensor
// memory is freed, the kernel returns.
//
// Measured (B200, 32 query / 8 kv heads of 128): a chunk of 2048 tokens at 32768, int8, float16: 1.29 to 1.31 ms = 810 to 826 TFLOP/s = 0.49 to 0.50 of the library's
// bf16 product; before long sums were folded, without the softmax arithmetic 0.80 ms, without the conversion besides 0.63 ms.  A tile's softmax takes 3400 clocks of a period
// of 4500: 2400 for the weights (1890 alone; 1024 of them exp2), 550 for the maximum.  What changed it on the way: loops over 64 columns instead of
// straight-line code, which had the warps wait for instructions (2.20 -> 1.39 ms); seven loader warps, packed arithmetic, no divisions (1.29); scores of half
// a tile kept in registers between the passes (1.21; 1.26 to 1.29 since products are ordered by commits).  Tried and dropped: part of the exponentials as
// polynomials on the FMA pipe (the same or slower), weights in one pass against the old maximum (registers spill).
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"
#include "prefill_umma.cuh"

namespace er {
namespace {

constexpr int kTok = 128;                  // tokens of a K / V tile
constexpr int kSoftWarps = 8, kLoadWarps = 7, kIssueWarp = 12;   // loaders: warps 8-11 and 13-15
constexpr int kThreads = 512;
constexpr float kLag = 8.f;                // how far (log2) a row's maximum may rise above the one in use
// The tensor cores add into their accumulators with truncation, up to 2^-23 of the sum for each 16 keys, which biases a long chain (keys around 500000, values
// around 1: 3.2e-3 low; 131072 keys: 7.7e-4).  After this many tiles (16384 keys: 1.2e-4 at most, measured 6e-5) a row's O is added to a float32 sum in memory
// and starts again.  A kernel of its own, for tables and windows that reach that far: the code alone, without a fold, costs a short prompt 12.3 -> 13.4 us,
// ragged prompts 148 -> 153.
constexpr int kFold = 128;
constexpr int kMostFoldSlots = 256;
constexpr float kCarry = 5.f;              // weights are carried 2^5 times: w <= 2^(8 + 2 + 5) < 65504
template <int D> __host__ __device__ constexpr int stage_count() { return D == 128 ? 5 : 8; }
// Slots for the scales of a tile's blocks.  The loader of key tile j waits for the ring entry that it fills, not for the scale slot.  With an even number of
// entries that one held the keys of tile j - entries / 2, and those are released by their score product, before the softmax of the same tile reads its scales;
// what is sure to have ended is the softmax of the tile before it.  So a slot may come round after entries / 2 + 1 tiles, no earlier.  (With an odd number the
// entry held values of tile j - entries / 2 - 1, whose product follows that tile's softmax: the same distance.)
template <int D> __host__ __device__ constexpr int scale_slots() { return stage_count<D>() / 2 + 1; }
constexpr int kMostScaleSlots = 5;
template <int D> __host__ __device__ constexpr int tile_bytes() { return kTok * D * 2; }   // also a tile of 128 query rows
// Floats of a CTA's sums: D / 4 groups of columns of 256 rows, then the maximum and the log2 of R that they stand for.
template <int D> __host__ __device__ constexpr int fold_floats() { return 256 * (D + 2); }
template <int D> __host__ __device__ constexpr int prefill_smem() { return (stage_count<D>() + 2) * tile_bytes<D>() + 256 + kMostScaleSlots * 32 * 4 + 1024; }

struct Kv8Prefill {
    Kv8Cache cache;
    const void* q;
    void* out;
    int64_t q_token, q_head, out_token, out_head;
    const int32_t* starts;
    float* partial;             // of the split tiles: [index][256 rows][D + 4]: max, sum, -, -, unnormalised row
    float* fold;                // sums of long contexts: [fold_slots][fold_floats], or nullptr: no CTA has more than kFold tiles
    int fold_slots;             // as many as CTAs can run at a time
    int num_tokens, group, window, min_rows;    // sequences with fewer query rows are somebody else's
    int slots, split_from, parts;               // CTAs [0, split_from) own a tile pair, the others a part of its keys
    float scale_log2;
    uint64_t group_magic;                       // ceil(2^64 / group)
};

// The sequence and the 256 query rows of slot `slot`: sequence s owns the slots from starts[s] * group / 256 + s on.
struct Tile {
    int seq, begin, n, len, row0, rows;        // rows: of the sequence; row0: first of the slot; rows == 0: nothing to do
    int wrong;                                 // what the host could not see: an ER_ERR_* code, or 0
};
__device__ __forceinline__ Tile find_tile(const Kv8Prefill& p, int slot) {
    const int lo = kv8_find_slot(p.starts, p.cache.num_seqs, slot, [&](int start, int s) { return static_cast<int>(static_cast<int64_t>(start) * p.group / 256) + s; });
    Tile t;
    t.seq = lo;
    t.begin = __ldg(p.starts + lo);
    t.n = __ldg(p.starts + lo + 1) - t.begin;
    const int len = __ldg(p.cache.lens + lo);
    t.rows = 0;
    t.row0 = (slot - (static_cast<int>(static_cast<int64_t>(t.begin) * p.group / 256) + lo)) * 256;
    t.len = 0;
    t.wrong = t.begin < 0 || t.n < 0 || t.begin > p.num_tokens - t.n ? ER_ERR_SHAPE : 0;
    if (t.wrong != 0) return t;
    const int rows = t.n * p.group;
    if (rows < p.min_rows || t.row0 < 0 || t.row0 >= rows) return t;
    t.rows = rows;
    t.len = len;
    const int most = p.cache.table_width * p.cache.page_size;     // rows behind the table have no page
    t.wrong = t.len > most ? ER_ERR_OUT_OF_PAGES : t.len < 0 ? ER_ERR_SHAPE : 0;
    t.len = max(0, min(t.len, most));
    return t;
}

// Which of the slots for sums are in use, by the running CTAs of all calls on the device: one fits an SM, so that a slot for each SM is enough, and a call's
// workspace need not hold one for every CTA of its grid.  A slot decides where a CTA keeps its sums, not what they are.
__device__ unsigned int fold_claims[kMostFoldSlots / 32];
__device__ int claim_fold_slot(int slots) {
    for (int k = 0; k < 4 * slots; ++k) {
        const int s = (static_cast<int>(blockIdx.x % static_cast<unsigned>(slots)) + k) % slots;
        if ((atomicOr(&fold_claims[s >> 5], 1u << (s & 31)) >> (s & 31) & 1u) == 0u) return s;
    }
    return -1;      // not with a CTA an SM; the sums would stay in tensor memory
}

// r / group by a multiplication (exact below 2^30)
__device__ __forceinline__ int row_query(const Kv8Prefill& p, int r) {
    return p.group == 1 ? r : static_cast<int>(__umul64hi(static_cast<uint64_t>(static_cast<uint32_t>(r)), p.group_magic));
}

struct Waiter {
    volatile int* abort_flag;
    const Kv8Cache* cache;
    __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity) const {
        if (mbar_try_wait(bar, parity) || *abort_flag) return;
        const uint64_t start = global_timer_ns();
        uint32_t spins = 0;
        while (!mbar_try_wait(bar, parity)) {
            if ((++spins & 0x3FFu) == 0u) {
                if (*abort_flag) return;
                if (global_timer_ns() - start > 2000000000ull) {
                    *abort_flag = 1;
                    kv8_report(*cache, ER_ERR_DEVICE_TIMEOUT);
                    return;
                }
            }
        }
    }
};

// Waits for the loads of tensor memory in flight; names the registers, so that nothing that uses them moves in front.
__device__ __forceinline__ void tmem_wait32(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                   "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
                   "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ bool elect_lane() {
    uint32_t on;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(on));
    return on != 0u;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint32_t half2_word(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int D, bool E4M3, bool Fold>
__global__ void __launch_bounds__(kThreads, 1) kv8_prefill_kernel(const __grid_constant__ Kv8Prefill p) {
    constexpr int kStages = stage_count<D>(), kScaleRing = scale_slots<D>(), kTile = tile_bytes<D>(), kRegion = kTok * 128;   // a region: 128 rows x 64 halves
    constexpr int kBarFull = 0, kBarEmpty = kStages, kBarS = 2 * kStages, kBarP = kBarS + 2, kBarQ = kBarP + 2, kBarO = kBarQ + 1, kBarScale = kBarO + 1,
                  kBarRead = kBarScale + kScaleRing, kNumBars = kBarRead + 2;
    constexpr uint32_t kColO = 256, kColW = D == 128 ? 0 : 384, kStrideW = D == 128 ? 128 : 64;   // tensor-memory columns
    static_assert(kNumBars * 8 + 12 <= 256, "");
    static_assert(kScaleRing > kStages / 2 && kScaleRing <= kMostScaleSlots, "scales would be overwritten while the softmax reads them");
    extern __shared__ uint8_t raw[];
    const Kv8Cache& c = p.cache;
    const uint32_t sbase = (smem_u32(raw) + 1023u) & ~1023u;
    uint8_t* gen = raw + (sbase - smem_u32(raw));
    uint8_t* q_gen = gen + kStages * kTile;                       // two tiles of queries behind the ring
    uint64_t* bars = reinterpret_cast<uint64_t*>(q_gen + 2 * kTile);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* fold_slot = abort_flag + 1;
    float* scale_ring = reinterpret_cast<float*>(q_gen + 2 * kTile + 256);   // [ring][key scale x 8, log2 of the value scale x 8, 1 / it x 8, -]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- which rows, which keys ----
    int unit = blockIdx.x, part = 0, parts = 1;
    if (unit >= p.split_from) {
        part = (unit - p.split_from) % p.parts;
        parts = p.parts;
        unit = p.split_from + (unit - p.split_from) / p.parts;
    }
    const int head = unit % c.num_kv_heads;                       // the last rows, which see most, first
    const Tile tile = find_tile(p, p.slots - 1 - unit / c.num_kv_heads);
    if (tile.wrong != 0 && threadIdx.x == 0) kv8_report(c, tile.wrong);
    if (tile.rows == 0) return;
    const int past = tile.len - tile.n, last_row = min(tile.rows, tile.row0 + 256) - 1;
    const int hi = min(tile.len, past + last_row / p.group + 1);  // keys below it
    const int lo = p.window > 0 ? max(0, past + tile.row0 / p.group - p.window + 1) : 0;
    int t_begin = lo / kTok, tiles = max(0, (hi + kTok - 1) / kTok - t_begin);
    if (parts > 1) {
        const int per = (tiles + parts - 1) / parts, b = min(tiles, part * per);
        tiles = min(tiles, b + per) - b;
        t_begin += b;
    }
    const bool two = tile.row0 + 128 < tile.rows;

    if (tid == 0) {
        for (int i = 0; i < kNumBars; ++i) {
            uint32_t n = 1;
            if (i < kBarEmpty) n = kTok / 16;
            else if (i == kBarP || i == kBarP + 1) n = 4;
            else if (i == kBarQ) n = two ? 8 : 4;
            else if (i >= kBarScale && i < kBarRead) n = kTok / 16;
            mbar_init(bars + i, n);
        }
        *abort_flag = 0;
        if constexpr (Fold) *fold_slot = tiles > kFold ? claim_fold_slot(p.fold_slots) : -1;
        mbar_init_fence();
    }
    if (warp == kIssueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int folding = Fold ? *fold_slot : -1;         // negative: not
    const Waiter wait{abort_flag, &c};
    // Codes -> fp16 operand tiles.  The 16-token units of the half tiles (keys of tile 0, values of tile 0, keys of tile 1, ...; eight to a half
    // tile) go round robin to the loader warps, each with the codes of its next unit on the way in registers and the page of the one behind it looked
    // up.  Lane: 16 codes of the rows lane / 4 and 8 further, two rows of four chunks to eight lanes, which store without bank conflicts.
    auto load_tiles = [&](int w) {
        constexpr int kParts = D / 64, kLoads = 2 * kParts;          // 64 codes of 8 rows at a time
        struct Unit {
            uint4 v[kLoads];
            float kscale, vscale;
            int page;
        };
        const int r8 = lane >> 2, c4 = lane & 3;
        const uint32_t dst_lane = sbase + um_swz(r8, 2 * c4), dst_lane2 = sbase + um_swz(r8, 2 * c4 + 1);
        const int64_t src_lane = static_cast<int64_t>(r8) * D + c4 * 16;
        const int total = 16 * tiles;
        auto token_of = [&](int q) { return (t_begin + (q >> 4)) * kTok + (q & 7) * 16; };
        // blocks in front of the window are not fetched: their pages may be gone or somebody else's
        auto look_up = [&](Unit& x, int q) { x.page = q < total && token_of(q) < tile.len && token_of(q) + kKv8Unit > lo ? kv8_page(c, tile.seq, token_of(q)) : -1; };
        auto fetch = [&](Unit& x, int q) {
            const int side = (q >> 3) & 1, tok = token_of(q), valid = x.page >= 0 ? tile.len - tok : 0;
            const int64_t row = kv8_row(c, max(x.page, 0), head, kv8_in_page(c, tok));
            const uint8_t* src = (side ? c.codes[1] : c.codes[0]) + row * D + src_lane;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                x.v[i] = make_uint4(0, 0, 0, 0);
                if (r8 + 8 * (i / kParts) < valid) x.v[i] = __ldg(reinterpret_cast<const uint4*>(src + (i / kParts) * 8 * D + (i % kParts) * 64));
            }
            if (side == 0 && lane == 0) {
                x.kscale = -1.f;
                x.vscale = 0.f;
                if (valid > 0) {
                    x.kscale = __ldg(c.scales[0] + kv8_scale_at(c, row));
                    x.vscale = __ldg(c.scales[1] + kv8_scale_at(c, row));
                } else if (q < total && tok < tile.len && tok + kKv8Unit > lo) {   // pages in front of the window may be gone
                    kv8_report(c, ER_ERR_OUT_OF_PAGES);
                }
            }
        };
        auto step = [&](Unit& x, int q) {
            if (q >= total) return;
            const int idx = q >> 3, st = idx % kStages, j = idx >> 1, u = q & 7;
            if (idx >= kStages) wait(bars + kBarEmpty + st, ((idx / kStages) - 1) & 1);
            const uint32_t at = st * kTile + u * 16 * 128;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint4 a, b;                                            // codes 0 .. 8, 8 .. 16 of the lane
                decode4<E4M3>(x.v[i].x, a.x, a.y);
                decode4<E4M3>(x.v[i].y, a.z, a.w);
                decode4<E4M3>(x.v[i].z, b.x, b.y);
                decode4<E4M3>(x.v[i].w, b.z, b.w);
                const uint32_t off = at + (i / kParts) * 8 * 128 + (i % kParts) * kRegion;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst_lane + off), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w) : "memory");
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst_lane2 + off), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
            }
            if ((idx & 1) == 0 && lane == 0) {
                float* s = scale_ring + (j % kScaleRing) * 32 + u;
                s[0] = x.kscale;
                s[8] = __log2f(x.vscale);                              // NaN stays NaN; 0 gives -inf
                s[16] = 1.f / x.vscale;
                mbar_arrive(bars + kBarScale + j % kScaleRing);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + kBarFull + st);
            fetch(x, q + kLoadWarps);
            look_up(x, q + 2 * kLoadWarps);
        };
        Unit x;
        look_up(x, w);
        fetch(x, w);
        look_up(x, w + kLoadWarps);
        for (int q = w; q < total; q += kLoadWarps) {
            step(x, q);
        }
    };

    // Registers of the groups of four warps: 512 threads x 128 at launch = 128 x (168 + 168 + 88 + 88).  Each branch moves its own.
    if (warp >= kSoftWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp != kIssueWarp) {
            load_tiles(warp - kSoftWarps - (warp > kIssueWarp ? 1 : 0));
        } else if (tiles > 0) {
            // ================= products: the whole warp walks the loop, so that descriptors stay in uniform registers; one lane issues =================
            const bool leader = elect_lane();
            constexpr uint32_t kHi = umma_desc_hi(1024);
            constexpr uint32_t idesc_qk = umma_idesc(128, kTok, false), idesc_pv = umma_idesc(128, D, true);
            const uint32_t ring_lo = umma_desc_lo(sbase, 16), v_lo = umma_desc_lo(sbase, kRegion), q_lo = umma_desc_lo(sbase + kStages * kTile, 16);
            auto scores = [&](int i, int idx) {                  // S_i = Q_i K^T, K in ring entry idx
                uint32_t kd = ring_lo + static_cast<uint32_t>(idx % kStages) * (kTile >> 4), qd = q_lo + i * (kTile >> 4);
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = ((kk >> 2) * kRegion + (kk & 3) * 32) >> 4;
                        umma_f16(tmem + 128u * i, umma_desc_pack(qd + off, kHi), umma_desc_pack(kd + off, kHi), idesc_qk, kk > 0);
                    }
                    umma_commit(smem_u32(bars + kBarS + i));
                }
                __syncwarp();
            };
            auto outputs = [&](int i, int idx, bool first) {     // O_i += W_i V
                uint32_t vd = v_lo + static_cast<uint32_t>(idx % kStages) * (kTile >> 4), a = tmem + kColW + kStrideW * i;
                if (leader) {
#pragma unroll
                    for (int kt = 0; kt < kTok / 16; ++kt)
                        umma_f16_ts(tmem + kColO + static_cast<uint32_t>(D) * i, a + 8u * kt, umma_desc_pack(vd + ((kt * 2048) >> 4), kHi), idesc_pv, !first || kt > 0);
                }
                __syncwarp();
            };
            auto full = [&](int idx) {
                wait(bars + kBarFull + idx % kStages, (idx / kStages) & 1);
                tc_fence_after();
            };
            auto read = [&](int i, int j) {                       // W_i of tile j has been read
                if constexpr (D == 128) {
                    if (leader) umma_commit(smem_u32(bars + kBarRead + i));
                    __syncwarp();
                    wait(bars + kBarRead + i, j & 1);
                    tc_fence_after();
                }
            };
            auto release = [&](int idx) {
                if (leader) umma_commit(smem_u32(bars + kBarEmpty + idx % kStages));
                __syncwarp();
            };
            wait(bars + kBarQ, 0);
            full(0);
            scores(0, 0);
            if (two) scores(1, 0);
            release(0);
            for (int j = 0; j < tiles; ++j) {
                const int vi = 2 * j + 1, ki = 2 * j + 2;
                const bool more = j + 1 < tiles;
                full(vi);
                wait(bars + kBarP, j & 1);
                tc_fence_after();
                const bool fresh = Fold && folding >= 0 ? j % kFold == 0 : j == 0;
                outputs(0, vi, fresh);
                if (more) {
                    full(ki);
                    read(0, j);
                    scores(0, ki);
                }
                if (two) {
                    wait(bars + kBarP + 1, j & 1);
                    tc_fence_after();
                    outputs(1, vi, fresh);
                }
                release(vi);
                if (more) {
                    if (two) {
                        read(1, j);
                        scores(1, ki);
                    }
                    release(ki);
                }
            }
            if (leader) umma_commit(smem_u32(bars + kBarO));
            __syncwarp();
            // After a wait that ran out nobody else waits for the products, which read this CTA's memory and write the tensor memory that is freed below.
            const uint64_t start = global_timer_ns();
            while (!mbar_try_wait(bars + kBarO, 0) && global_timer_ns() - start < 3000000000ull) {}
        }
    } else {
        // ================= softmax =================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
        if (warp < 4 || two) {
        const int i = warp >> 2, m_row = tid & 127, row = tile.row0 + i * 128 + m_row;
        const int qi = row_query(p, min(row, tile.rows - 1));
        const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t tm_s = tmem + 128u * i + lane_base, tm_o = tmem + kColO + static_cast<uint32_t>(D) * i + lane_base, tm_w = tmem + kColW + kStrideW * i + lane_base;
        // Queries: each warp copies its 32 rows into the operand layout, whole rows at a time (D / 8 lanes a row) and past the L1, most of whose memory
        // is shared memory here: as loads they waited for room there, 5 us a CTA.  float16 rows are operands as they are; a bfloat16 row is divided by
        // a power of two in place, since its range is not fp16's.
        float factor = p.scale_log2;           // log2(e) * scale * that power of two
        {
            constexpr int kLanes = D / 8, kRows = 32 / kLanes;
            const int chunk = lane % kLanes;
            uint8_t* tile_gen = q_gen + i * kTile;
            const uint32_t to = smem_u32(tile_gen) + (chunk >> 3) * kRegion;
            // row r0 of the tile is head `at_head` of query `query`; kRows further is dq queries and dh heads further
            int r0 = (warp & 3) * 32 + lane / kLanes;
            const int r = tile.row0 + i * 128 + r0, query = row_query(p, r), dq = row_query(p, kRows), dh = kRows - dq * p.group;
            int at_head = r - query * p.group;
            const T* src = static_cast<const T*>(p.q) + static_cast<int64_t>(tile.begin + query) * p.q_token + (head * p.group + at_head) * p.q_head + chunk * 8;
            const int64_t on = dq * p.q_token + dh * p.q_head, wrap = p.q_token - p.group * p.q_head;
#pragma unroll 4
            for (int k = 0; k < 32 / kRows; ++k) {
                if (r + k * kRows < tile.rows)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + um_swz(r0, chunk & 7)), "l"(src) : "memory");
                else
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(to + um_swz(r0, chunk & 7)), "r"(0) : "memory");
                r0 += kRows;
                src += on;
                at_head += dh;
                if (at_head >= p.group) { at_head -= p.group; src += wrap; }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
            if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
                uint32_t mx = 0;
#pragma unroll 4
                for (int k = 0; k < D / 8; ++k) {
                    const uint4 v = *reinterpret_cast<const uint4*>(tile_gen + (k >> 3) * kRegion + um_swz(m_row, k & 7));
                    const uint32_t w[4] = {v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu, v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu};
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx = __vmaxu2(mx, w[e]);                  // magnitudes compare like integers
                }
                mx = max(mx >> 16, mx & 0xFFFFu);
                const uint32_t ex = min(max(mx >> 7, 1u), 252u);
                const float down = __uint_as_float((253u - ex) << 23);
                factor *= __uint_as_float((ex + 1u) << 23);
#pragma unroll 4
                for (int k = 0; k < D / 8; ++k) {
                    uint4* at = reinterpret_cast<uint4*>(tile_gen + (k >> 3) * kRegion + um_swz(m_row, k & 7));
                    float f[8];
                    Act<T>::unpack(*at, f);
                    uint4 o;
                    o.x = half2_word(f[0] * down, f[1] * down);
                    o.y = half2_word(f[2] * down, f[3] * down);
                    o.z = half2_word(f[4] * down, f[5] * down);
                    o.w = half2_word(f[6] * down, f[7] * down);
                    *at = o;
                }
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + kBarQ);
        }
        const int limit = min(tile.len - 1, past + qi);
        const int lower = p.window > 0 ? past + qi - p.window + 1 : 0;
        float m = -INFINITY, l = 0.f, LR = -200.f;
        // This thread's row of the sums; what they count now, if they have been begun.
        float* const sums = p.fold + static_cast<int64_t>(max(folding, 0)) * fold_floats<D>();
        float4* const sum_row = reinterpret_cast<float4*>(sums) + i * 128 + m_row;
        float* const sum_max = sums + 256 * D + i * 128 + m_row;
        auto counts = [&]() {
            const float was = __ldcg(sum_max);
            return was == -INFINITY ? 0.f : fast_exp2(was - m) * fast_exp2(__ldcg(sum_max + 256) - LR);
        };
        for (int j = 0; j < tiles; ++j) {
            const int t0 = (t_begin + j) * kTok;
            wait(bars + kBarScale + j % kScaleRing, (j / kScaleRing) & 1);
            const float* sc = scale_ring + (j % kScaleRing) * 32;
            float vm = -INFINITY, kmin = INFINITY;
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                kmin = fminf(kmin, sc[g]);
                vm = fmaxf(vm, sc[8 + g]);
            }
            const bool edge = __any_sync(0xffffffffu, kmin < 0.f || t0 + kTok - 1 > limit || t0 < lower);
            if (edge) {         // only the blocks that this row sees: one that it does not may be of any size
                vm = -INFINITY;
#pragma unroll
                for (int g = 0; g < 8; ++g)
                    if (t0 + 16 * g <= limit && t0 + 16 * g + 15 >= lower) vm = fmaxf(vm, sc[8 + g]);
            }
            // The columns of chunk c0 .. c0 + 32 that this row sees, one bit each.
            auto seen = [&](int c0) {
                const int from = min(max(lower - t0 - c0, 0), 32), to = min(max(limit + 1 - t0 - c0, 0), 32);
                uint32_t bits = static_cast<uint32_t>((1ull << to) - 1ull) & ~static_cast<uint32_t>((1ull << from) - 1ull);
                if (sc[c0 / 16] < 0.f) bits &= 0xFFFF0000u;
                if (sc[c0 / 16 + 1] < 0.f) bits &= 0x0000FFFFu;
                return bits;
            };
            auto hide = [&](uint32_t (&s)[32], uint32_t bits) {
#pragma unroll
                for (int k = 0; k < 32; ++k) s[k] = (bits >> k & 1u) != 0u ? s[k] : 0xFF800000u;
            };
            wait(bars + kBarS + i, j & 1);
            tc_fence_after();
            // ---- the maximum; the columns 0 .. 63 last, they stay in registers ----
            float mx = -INFINITY;
            uint32_t a[32], b[32];
            tmem_ld32_nowait(tm_s + 64, a);
            tmem_ld32_nowait(tm_s + 96, b);
#pragma unroll 1
            for (int c0 = 64; c0 >= 0; c0 -= 64) {
                const float4 ks4 = *reinterpret_cast<const float4*>(sc + c0 / 16);
                const float ks[4] = {ks4.x, ks4.y, ks4.z, ks4.w};
                tmem_wait32(a);
                tmem_wait32(b);
                if (edge) {
                    hide(a, seen(c0));
                    hide(b, seen(c0 + 32));
                }
                auto take = [&](const uint32_t (&s)[32], int g0) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float x = __uint_as_float(s[16 * h]), y = __uint_as_float(s[16 * h + 1]);
#pragma unroll
                        for (int k = 2; k < 14; k += 4) {
                            x = max3(x, __uint_as_float(s[16 * h + k]), __uint_as_float(s[16 * h + k + 1]));
                            y = max3(y, __uint_as_float(s[16 * h + k + 2]), __uint_as_float(s[16 * h + k + 3]));
                        }
                        x = max3(x, __uint_as_float(s[16 * h + 14]), __uint_as_float(s[16 * h + 15]));
                        mx = fmaxf(mx, ks[g0 + h] < 0.f ? -INFINITY : fmaxf(x, y) * ks[g0 + h]);   // scales are not negative but for the mark of a hidden block
                    }
                };
                take(a, 0);
                if (c0 > 0) tmem_ld32_nowait(tm_s, a);
                take(b, 2);
                if (c0 > 0) tmem_ld32_nowait(tm_s + 32, b);
            }
            mx *= factor;
            // ---- after kFold tiles: O joins the sums in memory and begins anew ----
            const bool fold = Fold && folding >= 0 && j > 0 && j % kFold == 0;
            if (fold) {
                const float before = j == kFold ? 0.f : counts();
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t o[32];
                    tmem_ld32_nowait(tm_o + c0, o);
                    tmem_wait32(o);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        float4* at = sum_row + (c0 / 4 + k) * 256;
                        float4 v = make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                        if (j > kFold) {
                            const float4 w = __ldcg(at);
                            v = make_float4(fmaf(w.x, before, v.x), fmaf(w.y, before, v.y), fmaf(w.z, before, v.z), fmaf(w.w, before, v.w));
                        }
                        __stcg(at, v);
                    }
                }
                __stcg(sum_max, m);
                __stcg(sum_max + 256, LR);
            }
            // ---- move to it, if it is far enough above the one in use ----
            const bool grow = vm > LR + 2.f;
            if (__any_sync(0xffffffffu, grow || mx > m + kLag)) {
                const float m_new = fmaxf(m, mx), LR_new = grow ? ceilf(vm) : LR;
                const float corr = m_new == -INFINITY ? 1.f : fast_exp2(m - m_new);
                l *= corr;
                const float oc = corr * fast_exp2(LR - LR_new);
                m = m_new;
                LR = LR_new;
                if (j > 0 && !fold) {
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t o[32];
                        tmem_ld32_nowait(tm_o + c0, o);
                        tmem_wait32(o);
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * oc);
                        tmem_st32_words(tm_o + c0, o);
                    }
                }
            }
            // ---- weights: those of 64 columns go over 32, read by then ----
            const float base = m == -INFINITY ? 0.f : m;
            const float R = fast_exp2(LR - kCarry);
#pragma unroll 1
            for (int c0 = 0; c0 < kTok; c0 += 64) {
                // of the four blocks of 16: the factor of a score, the exponent's offset, what a sum of weights counts
                const float4 k4 = *reinterpret_cast<const float4*>(sc + c0 / 16), e4 = *reinterpret_cast<const float4*>(sc + 8 + c0 / 16),
                             i4 = *reinterpret_cast<const float4*>(sc + 16 + c0 / 16);
                float f[4] = {k4.x, k4.y, k4.z, k4.w}, up[4] = {e4.x, e4.y, e4.z, e4.w}, count[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    up[g] = up[g] - LR + kCarry;
                    up[g] = (up[g] < -60.f ? -60.f : up[g]) - base;   // a NaN stays; below 2^-60 a weight is nothing in fp16, but counts in the sum
                    f[g] *= factor;
                    count[g] = fminf(count[g] * R, 1.152921504606846976e18f);
                }
                if (c0 > 0) {
                    tmem_wait32(a);
                    tmem_wait32(b);
                }
                if (edge) {
                    const uint32_t bits[2] = {seen(c0), seen(c0 + 32)};
                    hide(a, bits[0]);
                    hide(b, bits[1]);
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        if (f[g] == 0.f) f[g] = 1.17549435e-38f;      // a hidden -inf stays one
                        if ((bits[g >> 1] >> (16 * (g & 1)) & 0xFFFFu) == 0u) { f[g] = 1.f; up[g] = 0.f; }   // nothing seen: the scales may be anything
                    }
                }
                uint32_t out[32];
                auto weigh = [&](const uint32_t (&s)[32], int g0) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int g = g0 + h;
                        const F2 f2 = pack2(f[g], f[g]), up2 = pack2(up[g], up[g]);
                        F2 sum = pack2(0.f, 0.f), sum2 = sum;
#pragma unroll
                        for (int k = 0; k < 16; k += 2) {
                            const F2 x2 = fma2(pack2(__uint_as_float(s[16 * h + k]), __uint_as_float(s[16 * h + k + 1])), f2, up2);
                            float u, v;
                            unpack2(x2, u, v);
                            u = fast_exp2(u);
                            v = fast_exp2(v);
                            if (k & 2) sum2 = add2(sum2, pack2(u, v)); else sum = add2(sum, pack2(u, v));
                            out[8 * g + (k >> 1)] = half2_word(u, v);
                        }
                        float x, y;
                        unpack2(add2(sum, sum2), x, y);
                        l = fmaf(x + y, count[g], l);
                    }
                };
                weigh(a, 0);
                if (c0 == 0) tmem_ld32_nowait(tm_s + 64, a);
                weigh(b, 2);
                if (c0 == 0) tmem_ld32_nowait(tm_s + 96, b);
                tmem_st32_words(tm_w + static_cast<uint32_t>(c0 / 2), out);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bars + kBarP + i);      // one arrival a warp: 128 of them would queue at the barrier
        }
        // ---- the rows ----
        if (tiles > 0) {
            wait(bars + kBarO, 0);
            tc_fence_after();
        }
        const float up = fast_exp2(LR - kCarry), f = parts > 1 ? up : (l == 0.f ? 0.f : up / l);
        const float f_sums = Fold && folding >= 0 ? counts() * f : 0.f;
        float* part_row = parts > 1 ? p.partial + (static_cast<int64_t>(static_cast<int>(blockIdx.x) - p.split_from) * 256 + i * 128 + m_row) * (D + 4) : nullptr;
        if (parts > 1) { part_row[0] = m; part_row[1] = l; }
        // Finished rows leave through shared memory, a bulk copy a row: over the ring of K / V tiles, which every product has read.
        constexpr int kOutRow = D * 2 + 16;
        uint8_t* out_row = gen + (i * 128 + m_row) * kOutRow;
        static_assert(256 * kOutRow <= kStages * kTile, "");
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t o[32];
            if (tiles > 0) {
                tmem_ld32_nowait(tm_o + c0, o);
                tmem_wait32(o);
            }
            float x[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = tiles > 0 && (parts > 1 || l != 0.f) ? __uint_as_float(o[k]) * f : 0.f;
            if (Fold && folding >= 0 && (parts > 1 || l != 0.f)) {
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    const float4 w = __ldcg(sum_row + (c0 + k) / 4 * 256);
                    x[k] = fmaf(w.x, f_sums, x[k]);
                    x[k + 1] = fmaf(w.y, f_sums, x[k + 1]);
                    x[k + 2] = fmaf(w.z, f_sums, x[k + 2]);
                    x[k + 3] = fmaf(w.w, f_sums, x[k + 3]);
                }
            }
            if (parts > 1) {
#pragma unroll
                for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4*>(part_row + 4 + c0 + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
            } else {
#pragma unroll
                for (int k = 0; k < 32; k += 8) *reinterpret_cast<uint4*>(out_row + (c0 + k) * 2) = Act<T>::pack(x + k);
            }
        }
        if (parts == 1 && row < tile.rows) {
            fence_async_smem();
            T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(tile.begin + qi) * p.out_token + (head * p.group + row - qi * p.group) * p.out_head;
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(out_row)), "r"(D * 2) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (Fold && tid == 0 && folding >= 0) {
        __threadfence();
        atomicAnd(&fold_claims[folding >> 5], ~(1u << (folding & 31)));
    }
    if (warp == kIssueWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Joins the parts of the split tile pairs: a warp per query row, a lane D / 32 dims.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_prefill_join_kernel(const __grid_constant__ Kv8Prefill p) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    const int unit = p.split_from + static_cast<int>(blockIdx.x) / 32, r = (static_cast<int>(blockIdx.x) % 32) * 8 + (threadIdx.x >> 5);
    const Tile tile = find_tile(p, p.slots - 1 - unit / p.cache.num_kv_heads);
    const int row = tile.row0 + r;
    if (tile.rows == 0 || row >= tile.rows) return;
    const float* base = p.partial + (static_cast<int64_t>(unit - p.split_from) * p.parts * 256 + r) * (D + 4);
    float M = -INFINITY, L = 0.f, acc[V];
    for (int k = 0; k < p.parts; ++k) M = fmaxf(M, base[static_cast<int64_t>(k) * 256 * (D + 4)]);
    const float M0 = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int k = 0; k < p.parts; ++k) {
        const float* src = base + static_cast<int64_t>(k) * 256 * (D + 4);
        const float f = fast_exp2(src[0] - M0);
        L = fmaf(src[1], f, L);
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = fmaf(src[4 + lane * V + i], f, acc[i]);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(tile.begin + row / p.group) * p.out_token + (unit % p.cache.num_kv_heads * p.group + row % p.group) * p.out_head + lane * V;
#pragma unroll
    for (int i = 0; i < V; i += 2) store_pair(dst + i, acc[i] * inv, acc[i + 1] * inv);
}

struct Plan {
    int slots, split_from, parts, grid;
};
// One CTA fits an SM.  With fewer than four rounds of tile pairs the last round counts: its pairs are cut along the keys into the number of parts
// (up to 8, no more CTAs than four rounds, at least four tiles of the longest sequence to a part) that fills whole rounds best; a second launch
// joins them.  With more rounds the pairs that see most run first and the short ones of the prompts' beginnings fill the gaps.
Plan make_plan(const er_kv8_cache* c, const er_kv8_attention_params* u, int sms) {
    Plan pl;
    const int group = static_cast<int>(u->num_heads / c->num_kv_heads), kv_heads = static_cast<int>(c->num_kv_heads);
    pl.slots = static_cast<int>(static_cast<int64_t>(u->num_tokens) * group / 256) + static_cast<int>(c->num_seqs);
    const int64_t units = static_cast<int64_t>(pl.slots) * kv_heads;
    const int64_t most_tiles = (static_cast<int64_t>(c->block_table_width) * c->page_size + kTok - 1) / kTok;
    const int rest = static_cast<int>(units % sms);
    pl.split_from = static_cast<int>(units);
    pl.parts = 1;
    double best = 1.0;
    for (int k = 2; k <= 8 && units < 4 * sms && rest > 0 && rest * k <= 4 * sms && 4 * k <= most_tiles; ++k) {
        const double rounds = static_cast<double>((rest * k + sms - 1) / sms) / k;
        if (rounds < best - 0.02) {
            best = rounds;
            pl.parts = k;
            pl.split_from = static_cast<int>(units) - rest;
        }
    }
    pl.grid = pl.split_from + (static_cast<int>(units) - pl.split_from) * pl.parts;
    return pl;
}

// Bytes of the split pairs' partial rows, and of the sums behind them: none where no CTA can have more than kFold tiles.
int64_t partial_bytes(const er_kv8_cache* c, const Plan& pl) {
    return pl.parts > 1 ? static_cast<int64_t>(pl.grid - pl.split_from) * 256 * (c->head_dim + 4) * 4 : 0;
}
int64_t fold_bytes(const er_kv8_cache* c, const er_kv8_attention_params* u, int sms) {
    uint64_t keys = kv8_table_rows(c);
    if (u->sliding_window > 0) keys = std::min<uint64_t>(keys, static_cast<uint64_t>(u->sliding_window) + 256 + 2 * kTok);   // a pair's queries, both ends of the tiles
    return keys > static_cast<uint64_t>(kFold) * kTok && sms <= kMostFoldSlots ? static_cast<int64_t>(sms) * 256 * (c->head_dim + 2) * 4 : 0;
}

template <typename T, int D, bool E4M3, bool Fold>
int32_t launch_kernel(const Kv8Prefill& p, const Plan& pl, cudaStream_t s) {
    constexpr int kSmem = prefill_smem<D>();
    static_assert(kSmem <= 232448, "prefill kernel exceeds the shared memory of an sm_100 CTA");
    static std::atomic<uint64_t> devices{0};
    const cudaError_t e = kv8_allow_smem(kv8_prefill_kernel<T, D, E4M3, Fold>, kSmem, devices);
    if (e != cudaSuccess) return kv8_launched(e, "kv8_prefill_kernel");
    kv8_prefill_kernel<T, D, E4M3, Fold><<<pl.grid, kThreads, kSmem, s>>>(p);
    return kv8_launched(cudaGetLastError(), "kv8_prefill_kernel");
}
template <typename T, int D, bool E4M3>
int32_t launch(const Kv8Prefill& p, const Plan& pl, cudaStream_t s) {
    const int32_t rc = p.fold != nullptr ? launch_kernel<T, D, E4M3, true>(p, pl, s) : launch_kernel<T, D, E4M3, false>(p, pl, s);
    if (rc != ER_OK || pl.parts == 1) return rc;
    kv8_prefill_join_kernel<T, D><<<(pl.grid - pl.split_from) / pl.parts * 32, 256, 0, s>>>(p);
    return kv8_launched(cudaGetLastError(), "kv8_prefill_join_kernel");
}
template <typename T>
int32_t launch_shape(const Kv8Prefill& p, const Plan& pl, uint32_t head_dim, bool e4m3, cudaStream_t s) {
    if (head_dim == 128) return e4m3 ? launch<T, 128, true>(p, pl, s) : launch<T, 128, false>(p, pl, s);
    return e4m3 ? launch<T, 64, true>(p, pl, s) : launch<T, 64, false>(p, pl, s);
}

// Sequences with up to this many query rows run on the decode kernel, which splits their keys over the GPU: it computes 16 rows
// at a time, the tile pair 256.
constexpr int kFewRows = 32;

struct Split {
    bool few, many;     // which of the two kernels have sequences to work on, as far as the host knows
};
Split split_of(const er_kv8_cache* c, const er_kv8_attention_params* u) {
    const uint64_t group = u->num_heads / c->num_kv_heads;
    const uint64_t most = u->max_query_len > 0 ? std::min(u->max_query_len, u->num_tokens) : u->num_tokens;
    const int64_t least = static_cast<int64_t>(u->num_tokens) - static_cast<int64_t>(most) * (static_cast<int64_t>(c->num_seqs) - 1);   // tokens of the shortest
    if (u->type == ER_TYPE_FLOAT32) return {true, false};
    const bool many = most * group > kFewRows;
    return {!many || least < 0 || static_cast<uint64_t>(least) * group <= kFewRows, many};
}

}  // namespace
}  // namespace er

extern "C" int64_t er_kv8_prefill_workspace_bytes(const er_kv8_cache* cache, const er_kv8_attention_params* u) {
    using namespace er;
    if (!cache || !u || cache->num_kv_heads == 0 || u->num_heads < cache->num_kv_heads) return report_error(ER_ERR_INVALID_ARGUMENT, "null argument, or no heads");
    const int sms = kv8_sm_count();
    if (sms == 0) return report_error(ER_ERR_CUDA, "no CUDA device (no CPU fallback)");
    const Split sp = split_of(cache, u);
    int64_t bytes = sp.few ? kv8_decode_workspace(cache, u, true) : 0;      // the two kernels run one after the other
    if (sp.many) {
        const Plan pl = make_plan(cache, u, sms);
        bytes = std::max(bytes, partial_bytes(cache, pl) + fold_bytes(cache, u, sms));
    }
    return bytes;
}

extern "C" int32_t er_kv8_attention_prefill(const er_kv8_cache* cache, const er_kv8_attention_params* u, void* stream) {
    using namespace er;
    if (!cache || !u) return report_error(ER_ERR_INVALID_ARGUMENT, "null argument");
    Kv8Cache c{};
    int32_t rc = kv8_check(cache, &c);
    if (rc == ER_OK) rc = kv8_check_attention(cache, u);
    if (rc != ER_OK) return rc;
    if (!u->query_starts) return report_error(ER_ERR_INVALID_ARGUMENT, "query_starts is needed for a ragged batch");
    if (!kv8_aligned(u->query_starts, 4)) return report_error(ER_ERR_INVALID_ARGUMENT, "query_starts must be 4-byte aligned");
    if ((static_cast<uint64_t>(u->num_tokens) * (u->num_heads / cache->num_kv_heads) / 256 + cache->num_seqs) * cache->num_kv_heads > (1u << 28))
        return report_error(ER_ERR_UNSUPPORTED, "more than 2^28 tiles of query rows");
    rc = kv8_check_device(cache->keys);
    if (rc == ER_OK) rc = kv8_check_workspace(u, er_kv8_prefill_workspace_bytes(cache, u));
    if (rc != ER_OK || cache->num_seqs == 0 || u->num_tokens == 0) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool e4m3 = cache->format == ER_KV8_E4M3;
    const Split sp = split_of(cache, u);
    if (sp.many) {
        Kv8Prefill p{};
        p.cache = c;
        p.q = u->q; p.out = u->out;
        p.q_token = u->q_token_stride; p.q_head = u->q_head_stride; p.out_token = u->out_token_stride; p.out_head = u->out_head_stride;
        p.starts = u->query_starts;
        p.partial = static_cast<float*>(u->workspace);
        p.num_tokens = static_cast<int>(u->num_tokens);
        p.group = static_cast<int>(u->num_heads) / c.num_kv_heads;
        p.window = kv8_window(cache, u);
        p.min_rows = sp.few ? kFewRows + 1 : 0;      // a hint that is wrong costs time, not rows
        p.group_magic = p.group == 1 ? 0 : ~0ull / static_cast<uint64_t>(p.group) + 1;
        p.scale_log2 = kv8_scale_log2(u->softmax_scale, cache->head_dim);
        const int sms = kv8_sm_count();
        const Plan pl = make_plan(cache, u, sms);
        if (fold_bytes(cache, u, sms) > 0) {
            p.fold = p.partial + partial_bytes(cache, pl) / 4;
            p.fold_slots = sms;
        }
        p.slots = pl.slots; p.split_from = pl.split_from; p.parts = pl.parts;
        rc = u->type == ER_TYPE_FLOAT16 ? launch_shape<__half>(p, pl, cache->head_dim, e4m3, s) : launch_shape<__nv_bfloat16>(p, pl, cache->head_dim, e4m3, s);
        if (rc != ER_OK) return rc;
    }
    return sp.few ? kv8_launch_decode(c, cache, u, true, sp.many ? kFewRows : 0, s) : ER_OK;
}
