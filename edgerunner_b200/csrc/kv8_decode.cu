// er_kv8_attention_decode: attention of one or a few new tokens per sequence over an 8-bit block-scaled paged cache.
//
// Mathematics.  With codes c and block scales a (keys) and b (values), row i of a block:  s_i = (q . ck_i) a scale,  o = sum_i p_i b cv_i /
// sum_i p_i,  p_i = exp(s_i - m).  Codes are exact in fp16, so both contractions run on mma.sync.m16n8k16 with fp16 operands and float32
// accumulators; the key scale multiplies the score, the value scale the probability.  The probabilities that enter the second product are
// w = p * b / R with R the power of two next above the largest value scale that the query has seen so far (so w <= 1 whatever the scales are), carried 4096
// times so that small ones stay normal fp16 numbers; R and m move together and rarely.  bfloat16 rows round w to fp16; float32 and float16 rows carry a second
// half with what that leaves (64 ragged sequences in float16: 226 -> 236 us with up to four query rows a kv head, 193 -> 208 us with 16).
//
// Work.  Bound by memory: 2 D bytes a row for 4 D flops a query head.  A persistent CTA per SM; the list of 32-token units of all (sequence, kv head,
// row tile) items is cut evenly over the CTAs whatever the lengths are, inside a CTA the units of an item go round robin to the warps.  A warp
// streams its units through its own ring of shared-memory stages with TMA (boxes of 16 rows; no barrier between warps, 96 to 130 KB in flight a SM),
// and runs both products of a unit alone: scores as S^T = K q^T (2 x 16 tokens x 8 query rows), outputs as O^T = V^T w^T (16 dims x 8 query
// rows), so eight query rows fill a tile and K is an A operand as it lies in memory.  The warps of a CTA are joined in shared memory at the end of an
// item, the CTAs that share an item by a second small launch that overlaps this one's tail.
//
// Measured (B200, head size 128, 32 query / 8 kv heads): 64 sequences of 1024 .. 16384 rows in 16-row pages, E4M3, bfloat16: 227 to 234 us = 5.0 to 5.1 TB/s = 0.76 to 0.78 of
// the copy bandwidth; one sequence of 131072 int8 rows, float16: 58 to 61 us = 4.4 to 4.6 TB/s.  With the arithmetic taken out the first takes 207 us, with the copies
// taken out 173 us: what is left is their overlap at the ends of items (4.5 a CTA), the start and the joining launch.  32 tokens at a time instead of 16
// brought 312 -> 237 us (the bookkeeping of a unit was half of its instructions); cp.async instead of TMA measured the same.
//
// Lane (g, t) = (lane / 4, lane % 4).  The contraction index of the scores is relabelled so that lane t owns the dims [D/4 t, D/4 (t+1)) of a
// row: two (D = 64: one) 16-byte reads a row.  The dims of the outputs are relabelled so that lane g owns D/8 consecutive ones: 16 (8) bytes of
// four token rows, turned into token pairs by byte permutes.  Stage layout: 16-byte chunks XORed so that both reads are free of bank conflicts.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv8.cuh"
#include "tmap.h"

namespace er {
namespace {

constexpr int kMinUnits = 8;          // units of a CTA, so that short work stays together
constexpr int kUnit = 2 * kKv8Unit;   // tokens that a warp takes at a time: two halves, each with a page and scales of its own
// The tensor cores add into their accumulators with truncation: a product of 16 keys takes up to 2^-23 from the sum, half of that on average, and a warp adds every
// 8th or 12th of a visit (one CTA over 500000 rows: 1.7e-4 low, 4 million rows: 1.4e-3).  float32 rows move their sums to registers every 8 units.  16-bit rows
// have no registers for that: where a query may see more rows than kPlainRows they add them to a float32 sum in memory every kSumUnits units of a warp, that is
// every 196608 rows of a CTA's visit (1.2e-4 at most, measured 7e-5).  A kernel of its own, since the count alone costs the loop (64 ragged sequences: 231 us
// without, 236 with it, 262 with eight warps that keep the sums in registers).
constexpr uint64_t kPlainRows = 1u << 18;
constexpr int kSumUnits = 512;
constexpr float kWeightScale = 4096.f;    // 2^12
constexpr float kLift0 = 8.507059173023462e37f;    // 2^126, while no scale above 2^-114 has been seen

struct Kv8Decode {
    CUtensorMap maps[2];            // codes of the keys, values as [rows][head_dim], boxes of 16 rows
    Kv8Cache cache;
    const void* q;
    void* out;
    int64_t q_token, q_head, out_token, out_head;
    float* partial;
    float4* sums;                   // of long visits: [CTA][warp][NT][D / 16 + 1][lane]: accumulators, then the maxima and lifts that they stand for
    const int32_t* starts;          // tokens of the sequences, or nullptr: query_len each
    int num_tokens, group, query_len, window, tile_rows;
    int few_rows;                   // > 0: sequences with more query rows are somebody else's
    float scale_log2;
};

// ---- the work list ----
// Query row r of a (sequence, kv head) is query r / group, head r % group of the kv head's group; tile_rows of them make an item.
struct SeqRange {
    int len, begin, n;              // rows in the cache, first query token, queries
    int first_unit, units;          // first unit that a query can see, units of an item (at least 1: an empty one writes zeros)
    int row_tiles;                  // 0 for a sequence without queries
};
__device__ __forceinline__ SeqRange seq_range(const Kv8Decode& p, int seq) {
    SeqRange r;
    if (p.starts == nullptr) {
        r.begin = seq * p.query_len;
        r.n = p.query_len;
    } else {
        r.begin = __ldg(p.starts + seq);
        r.n = __ldg(p.starts + seq + 1) - r.begin;
        if (r.begin < 0 || r.n < 0 || r.begin > p.num_tokens - r.n) r.n = 0;
    }
    r.row_tiles = (r.n * p.group + p.tile_rows - 1) / p.tile_rows;
    if (p.few_rows > 0 && r.n * p.group > p.few_rows) r.row_tiles = 0;
    r.len = max(0, min(__ldg(p.cache.lens + seq), p.cache.table_width * p.cache.page_size));   // rows behind the table have no page
    const int lo = p.window > 0 ? max(0, r.len - r.n - p.window + 1) : 0;
    r.first_unit = lo / kUnit;
    r.units = max(1, (r.len + kUnit - 1) / kUnit - r.first_unit);
    return r;
}
struct Place {        // a position in the list
    int seq, item;    // item of the sequence: kv head * row_tiles + row tile
    int unit;         // unit of the item
    SeqRange r;
    __device__ __forceinline__ void next_item(const Kv8Decode& p) {   // only where there is one
        unit = 0;
        if (++item == p.cache.num_kv_heads * r.row_tiles) {
            item = 0;
            do r = seq_range(p, ++seq); while (r.row_tiles == 0);
        }
    }
    // The first and the last row that some query row of the item's tile sees, without regard to the length of the cache.
    __device__ __forceinline__ int first_query(const Kv8Decode& p) const { return item % r.row_tiles * p.tile_rows / p.group; }
    __device__ __forceinline__ int last_query(const Kv8Decode& p) const {
        return (min(r.n * p.group, (item % r.row_tiles + 1) * p.tile_rows) - 1) / p.group;
    }
    // The first row that the tile sees: pages in front of it may be gone.
    __device__ __forceinline__ int lowest(const Kv8Decode& p) const { return p.window > 0 ? max(0, r.len - r.n + first_query(p) - p.window + 1) : 0; }
    // Of the `count` units from `unit` on, those [u0, u1) that the tile sees anything of.
    __device__ __forceinline__ void visible(const Kv8Decode& p, int count, int& u0, int& u1) const {
        const int base = r.first_unit + unit, end = r.len - r.n + last_query(p) + 1;      // rows below `end`
        const int lo = lowest(p) / kUnit;
        u0 = max(0, lo - base);
        u1 = min(count, max(0, end + kUnit - 1) / kUnit - base);
    }
    __device__ __forceinline__ int token(int u) const { return (r.first_unit + unit + u) * kUnit; }   // of the u-th unit from here
};
// The list, by every thread of the CTA.  `pick(total)` names the unit that the CTA looks for, negative: none.  With a thread a sequence the lengths are
// read once for both; longer batches are summed first and then walked 32 sequences at a time.
struct Found {
    int64_t total;
    Place place;
};
struct ListScratch {
    int64_t sums[16];
    Place place;
};
template <typename Pick>
__device__ Found find_in_list(const Kv8Decode& p, ListScratch* scratch, Pick pick) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, seqs = p.cache.num_seqs, heads = p.cache.num_kv_heads;
    auto units_of = [&](const SeqRange& r) { return static_cast<int64_t>(r.units) * r.row_tiles * heads; };
    auto take = [&](int s, const SeqRange& r, int64_t offset) {
        Place pl;
        pl.seq = s;
        pl.r = r;
        pl.item = static_cast<int>(offset / r.units);
        pl.unit = static_cast<int>(offset % r.units);
        scratch->place = pl;
    };
    const bool once = seqs <= static_cast<int>(blockDim.x);
    SeqRange mine{};
    int64_t sum = 0, incl = 0;
    for (int s = threadIdx.x; s < seqs; s += blockDim.x) {
        mine = seq_range(p, s);
        sum += units_of(mine);
    }
    incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += o;
    }
    if (lane == 31) scratch->sums[warp] = incl;
    __syncthreads();
    Found f{};
    int64_t before = 0;
    for (int w = 0; w < warps; ++w) {
        if (w < warp) before += scratch->sums[w];
        f.total += scratch->sums[w];
    }
    const int64_t at = pick(f.total);
    if (once) {
        const int64_t start = before + incl - sum;
        if (at >= start && at < start + sum) take(threadIdx.x, mine, at - start);
    } else if (warp == 0 && at >= 0) {
        before = 0;
        for (int s0 = 0; s0 < seqs; s0 += 32) {
            const int s = s0 + lane;
            SeqRange r{};
            if (s < seqs) r = seq_range(p, s);
            const int64_t n = units_of(r);
            incl = n;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += o;
            }
            const int64_t start = before + incl - n;
            const bool here = at >= start && at < start + n;
            if (here) take(s, r, at - start);
            before += __shfl_sync(0xffffffffu, incl, 31);
            if (__any_sync(0xffffffffu, here)) break;
        }
    }
    __syncthreads();
    f.place = scratch->place;
    return f;
}
// CTA c of n takes the units [total c / n, total (c + 1) / n).
__device__ __forceinline__ int used_ctas(int64_t total, int ctas) { return static_cast<int>(min(static_cast<int64_t>(ctas), (total + kMinUnits - 1) / kMinUnits)); }
__device__ __forceinline__ int64_t cta_begin(int64_t total, int n, int c) { return total * c / n; }
__device__ __forceinline__ int cta_of(int64_t total, int n, int64_t unit) { return static_cast<int>(((unit + 1) * n - 1) / total); }

// ---- instructions ----
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int row, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst), "l"(map), "r"(0), "r"(row),
                 "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void split_half2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = half2_bits(a - f.x, b - f.y);
}

// 2^12 over the power of two next above (or at) a value scale.  Scales from 2^-126 (smaller ones count as 0) to 2^126.
__device__ __forceinline__ float lift_below(float scale) {
    const uint32_t b = __float_as_uint(scale), e = min((b >> 23) + ((b & 0x7FFFFFu) != 0u ? 1u : 0u), 253u);
    return __uint_as_float(min(266u - e, 253u) << 23);
}
__device__ __forceinline__ float inverse_lift(float lift) { return __uint_as_float(0x7F000000u - __float_as_uint(lift)); }

// A stage: keys of the two halves, values of the two halves.
template <int D> struct Stage {
    static constexpr int kHalf = kKv8Unit * D, kSide = 2 * kHalf, kBytes = 2 * kSide;
    // byte offset of 16-byte chunk c of row r inside a half: the 128-byte (64-byte) swizzle of the tensor map
    static __device__ __forceinline__ int at(int r, int c) {
        if constexpr (D == 128) return r * 128 + ((c ^ (r & 7)) << 4);
        else return r * 64 + ((c ^ (r >> 1 & 3)) << 4);
    }
};
template <int NT> __host__ __device__ constexpr int decode_rows() { return 8 * NT; }
// Warps of a CTA.  A unit costs a warp about 570 instructions, most of them in chains: with two warps to a scheduler it waits for itself a
// quarter of the time.  Three fit where 168 registers do: one column tile of 16-bit rows (64 ragged sequences: 237 -> 226 us).
template <typename T, int NT> __host__ __device__ constexpr int decode_warps() { return sizeof(T) == 2 && NT == 1 ? 12 : 8; }
// Warps that meet in shared memory at the end of an item; those beyond hand theirs to a partner first.
template <typename T, int NT> __host__ __device__ constexpr int join_warps() { return decode_warps<T, NT>() / 2; }
template <typename T, int D, int NT> __host__ __device__ constexpr int decode_stages() {
    constexpr int n = decode_warps<T, NT>() == 12 ? 2 : NT == 1 ? 3 : 2;
    return D == 128 ? n : 2 * n;
}
template <typename T, int D, int NT> __host__ __device__ constexpr int join_floats() { return join_warps<T, NT>() * 8 * NT * (D + 4); }
template <typename T, int D, int NT> __host__ __device__ constexpr int decode_smem() {
    return decode_warps<T, NT>() * decode_stages<T, D, NT>() * (Stage<D>::kBytes + 16 + 8) + (join_floats<T, D, NT>() + join_warps<T, NT>() * 8 * NT * 2) * 4 + static_cast<int>(sizeof(ListScratch)) + 16 + 1024;
}
// One partial: max, sum, -, - and the unnormalised row.
template <int D> __host__ __device__ constexpr int partial_stride() { return D + 4; }

// A wait of at most 2 s: then the status word is set, later waits are skipped and the kernel runs to its end.
__device__ __forceinline__ void bounded_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, const Kv8Cache& c) {
    if (mbar_try_wait(bar, parity) || *abort_flag) return;
    const uint64_t start = global_timer_ns();
    uint32_t spins = 0;
    while (!mbar_try_wait(bar, parity)) {
        if ((++spins & 0x3FFu) == 0u) {
            if (*abort_flag) return;
            if (global_timer_ns() - start > 2000000000ull) {
                *abort_flag = 1;
                kv8_report(c, ER_ERR_DEVICE_TIMEOUT);
                return;
            }
        }
    }
}

template <typename T, int D, bool E4M3, int NT, bool Long, bool Pairs>
__global__ void __launch_bounds__(decode_warps<T, NT>() * 32, 1) kv8_decode_kernel(const __grid_constant__ Kv8Decode p) {
    constexpr bool kSplit = sizeof(T) == 4;      // float32: queries as a high and a low half
    // Weights as a high and a low half: one rounding to fp16 is seen beside float16's own (131072 rows: 3.3e-4 from 64 bits instead of 2.2e-4), not beside bfloat16's.
    // The low halves are a second product, or (Pairs: up to four query rows) take the four free columns, whose queries are the first four's over again.
    constexpr bool kSplitW = !std::is_same<T, __nv_bfloat16>::value && !Pairs;
    static_assert(!Pairs || (NT == 1 && std::is_same<T, __half>::value), "");
    constexpr int kColumn = Pairs ? 3 : 7;       // column c of a tile is query row c & kColumn
    static_assert(!kSplit || (NT == 1 && !Long), "");
    constexpr int kRows = decode_rows<NT>(), kStages = decode_stages<T, D, NT>(), kWarps = decode_warps<T, NT>(), kThreads = kWarps * 32, kJoin = join_warps<T, NT>();
    constexpr int KK = D / 16, MT = D / 16, kWords = D / 16;   // k-steps of the scores; m-tiles of the outputs; 4-byte words of a lane's part of a key row
    constexpr int kOwn = D / 8;                                 // dims of a lane g in the outputs
    constexpr int kJoinRow = D + 4;
    extern __shared__ uint8_t raw[];
    uint8_t* stages = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);     // the swizzle goes by the address
    float* stage_scales = reinterpret_cast<float*>(stages + kWarps * kStages * Stage<D>::kBytes);
    float* join = stage_scales + kWarps * kStages * 4;
    float* join_ml = join + join_floats<T, D, NT>();
    uint64_t* bars = reinterpret_cast<uint64_t*>(join_ml + kJoin * kRows * 2);
    ListScratch* scratch = reinterpret_cast<ListScratch*>(bars + kWarps * kStages);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(scratch + 1);
    const Kv8Cache& c = p.cache;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, half = lane >> 4;
    const int odd = D == 64 ? t & 1 : 0;
    const uint32_t pairs_lo = odd ? 0x1504u : 0x5140u, pairs_hi = odd ? 0x3726u : 0x7362u;   // bytes 0, 1 (2, 3) of a row pair, the lower row first
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x < kWarps * kStages) mbar_init(bars + threadIdx.x, 2);    // a lane of each half arrives with the bytes of its copies
    if (threadIdx.x == 0) *abort_flag = 0;
    mbar_init_fence();

    const int cta = blockIdx.x;
    const Found list = find_in_list(p, scratch, [&](int64_t total) {
        const int n = used_ctas(total, gridDim.x);
        return cta < n ? cta_begin(total, n, cta) : -1;
    });
    const int64_t total = list.total;
    const int n = used_ctas(total, gridDim.x);
    if (cta == 0) {                 // what the host cannot see
        for (int s = threadIdx.x; s < c.num_seqs; s += kThreads) {
            if (__ldg(c.lens + s) > c.table_width * c.page_size) kv8_report(c, ER_ERR_OUT_OF_PAGES);
            if (__ldg(c.lens + s) < 0) kv8_report(c, ER_ERR_SHAPE);
            if (p.starts != nullptr && seq_range(p, s).n != __ldg(p.starts + s + 1) - __ldg(p.starts + s)) kv8_report(c, ER_ERR_SHAPE);
        }
    }
    if (cta >= n) return;
    int64_t left = cta_begin(total, n, cta + 1) - cta_begin(total, n, cta);       // units of this CTA not yet walked over
    Place at = list.place;

    // ---- producer: this warp's units, kStages - 1 ahead ----
    uint8_t* my_stages = stages + warp * kStages * Stage<D>::kBytes;
    uint64_t* my_bars = bars + warp * kStages;
    float* my_scales = stage_scales + warp * kStages * 4;   // per stage: key and value scale of half 0, of half 1
    Place pp = at;                  // segment the producer is in
    int64_t pleft = left;           // units from pp.unit on
    int pseg = static_cast<int>(min(static_cast<int64_t>(pp.r.units - pp.unit), pleft));   // units of the segment
    int pu, pend;                   // next unit of the segment for this warp; end of those that are worth a look
    int ppage = -1;                 // page of this lane's half of it
    bool pmore = true;
    pp.visible(p, pseg, pu, pend);
    pu += warp;
    auto settle = [&]() {           // moves on to the segment that holds this warp's next unit and looks its page up
        while (pu >= pend) {
            pleft -= pseg;
            if (pleft <= 0) { pmore = false; return; }
            pp.next_item(p);
            pseg = static_cast<int>(min(static_cast<int64_t>(pp.r.units), pleft));
            pp.visible(p, pseg, pu, pend);
            pu += warp;
        }
        const int tok = pp.token(pu) + half * kKv8Unit;
        // blocks in front of the window are not fetched: their pages may be gone or somebody else's
        ppage = tok < pp.r.len && (p.window == 0 || tok + kKv8Unit > pp.lowest(p)) ? kv8_page(c, pp.seq, tok) : -1;
    };
    int pstage = 0, produced = 0;
    auto produce = [&]() {          // the next unit, if there is one: lanes 0-15 see to half 0, 16-31 to half 1
        if (pmore && !*abort_flag) {
            const int tok = pp.token(pu) + half * kKv8Unit;
            float* sc = my_scales + pstage * 4 + half * 2;
            const int64_t row = kv8_row(c, max(ppage, 0), pp.item / pp.r.row_tiles, kv8_in_page(c, tok));
            if ((lane & 15) == 0) {
                mbar_arrive_expect_tx(my_bars + pstage, ppage >= 0 ? 2 * Stage<D>::kHalf : 0);
                if (ppage >= 0) {
                    const uint32_t dst = smem_u32(my_stages + pstage * Stage<D>::kBytes + half * Stage<D>::kHalf);
                    tma_rows(dst, &p.maps[0], static_cast<int>(row), my_bars + pstage);
                    tma_rows(dst + Stage<D>::kSide, &p.maps[1], static_cast<int>(row), my_bars + pstage);
                } else if (tok < pp.r.len && tok + kKv8Unit > pp.lowest(p)) {
                    kv8_report(c, ER_ERR_OUT_OF_PAGES);
                }
            }
            if ((lane & 15) < 2) {
                if (ppage >= 0) cp_async4(smem_u32(sc + (lane & 15)), ((lane & 15) == 0 ? c.scales[0] : c.scales[1]) + kv8_scale_at(c, row));
                else sc[lane & 15] = -1.f;      // nothing to see: no row yet, or no page
            }
            pu += kWarps;
            ++produced;
            settle();
        }
        cp_async_commit();
        pstage = pstage + 1 == kStages ? 0 : pstage + 1;
    };
    settle();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) produce();

    // the rows of this lane's columns g, dims [D/4 t, D/4 (t+1)): of the next item while the warps of this one are joined
    constexpr int kVecs = D / 4 / Act<T>::kVec;
    uint4 ahead[NT][kVecs];
    auto load_queries = [&]() {
        const int head = at.item / at.r.row_tiles, first_row = at.item % at.r.row_tiles * kRows;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = first_row + nt * 8 + (g & kColumn), qi = r / p.group;
            const T* src = static_cast<const T*>(p.q) + static_cast<int64_t>(at.r.begin + qi) * p.q_token + (head * p.group + r - qi * p.group) * p.q_head + (D / 4) * t;
#pragma unroll
            for (int i = 0; i < kVecs; ++i) ahead[nt][i] = r < at.r.n * p.group ? __ldg(reinterpret_cast<const uint4*>(src) + i) : make_uint4(0, 0, 0, 0);
        }
    };
    load_queries();

    int cstage = 0, cphase = 0;
    bool first_segment = true;
    while (left > 0) {
        const int seg = static_cast<int>(min(static_cast<int64_t>(at.r.units - at.unit), left));
        const int head = at.item / at.r.row_tiles, rt = at.item % at.r.row_tiles, rows = at.r.n * p.group;
        const int past = at.r.len - at.r.n;            // position of query 0
        int u0, u1;
        at.visible(p, seg, u0, u1);
        const int all_see_to = past + at.first_query(p), all_see_from = past + at.last_query(p) - p.window + 1;
        // ---- queries of this lane's column g: dims [D/4 t, D/4 (t+1)), scaled to at most 1 by a power of two ----
        uint32_t qh[NT][KK][2], ql[kSplit ? NT : 1][kSplit ? KK : 1][2];
        float qscale[NT][2];        // of the columns 2t, 2t + 1
        int limit[NT][2];           // last row that they see
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float x[D / 4];
#pragma unroll
            for (int i = 0; i < kVecs; ++i) Act<T>::unpack(ahead[nt][i], x + i * Act<T>::kVec);
            uint32_t mx = 0;
#pragma unroll
            for (int i = 0; i < D / 4; ++i) mx = max(mx, __float_as_uint(x[i]) & 0x7FFFFFFFu);
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const uint32_t ex = min(max(mx >> 23, 1u), 252u);     // an infinity or a NaN goes through as it is
            const float down = __uint_as_float((253u - ex) << 23) , up = __uint_as_float((ex + 1u) << 23);   // 2^(126 - ex), 2^(ex - 126)
#pragma unroll
            for (int k = 0; k < KK; ++k) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float a = x[4 * k + 2 * j] * down, b = x[4 * k + 2 * j + 1] * down;
                    if constexpr (kSplit) split_half2(a, b, qh[nt][k][j], ql[nt][k][j]);
                    else qh[nt][k][j] = half2_bits(a, b);
                }
            }
            const float f = up * p.scale_log2;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                qscale[nt][j] = __shfl_sync(0xffffffffu, f, (2 * t + j) * 4);
                const int rr = rt * kRows + nt * 8 + ((2 * t + j) & kColumn);
                limit[nt][j] = past + min(rr, rows - 1) / p.group;
            }
        }
        float o[NT][MT][4], m[NT][2], l[NT][2], lift[NT][2];    // lift: 4096 / R, powers of two
        float keep[kSplit ? MT : 1][4];     // float32: the tensor cores' sums are moved here every 8 units (their accumulators round towards zero)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < MT; ++i) { o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f; }
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
            lift[nt][0] = lift[nt][1] = kLift0;
        }
#pragma unroll
        for (int i = 0; i < (kSplit ? MT : 1); ++i) keep[i][0] = keep[i][1] = keep[i][2] = keep[i][3] = 0.f;
        int since = 0;
        // Long visits: this lane's sums in memory, once they have been begun, are added to the accumulators, which then go there and start again.
        bool begun = false;
        float4* const sums = Long ? p.sums + static_cast<int64_t>(cta * kWarps + warp) * (NT * (MT + 1) * 32) + lane : nullptr;
        auto add_sums = [&]() {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float4 was = __ldcg(sums + (nt * (MT + 1) + MT) * 32);
                const float was_m[2] = {was.x, was.y}, was_lift[2] = {was.z, was.w};
                float f[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) f[j] = was_m[j] == -INFINITY ? 0.f : fast_exp2(was_m[j] - m[nt][j]) * (lift[nt][j] * inverse_lift(was_lift[j]));
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const float4 v = __ldcg(sums + (nt * (MT + 1) + i) * 32);
                    o[nt][i][0] = fmaf(v.x, f[0], o[nt][i][0]);
                    o[nt][i][1] = fmaf(v.y, f[1], o[nt][i][1]);
                    o[nt][i][2] = fmaf(v.z, f[0], o[nt][i][2]);
                    o[nt][i][3] = fmaf(v.w, f[1], o[nt][i][3]);
                }
            }
        };

        for (int u = u0 + warp; u < u1; u += kWarps) {
            cp_async_wait<kStages - 2>();
            bounded_wait(my_bars + cstage, cphase, abort_flag, c);
            __syncwarp();           // the unit is here for every lane, and every lane has read the one before, whose stage is filled next
            produce();
            const uint8_t* ks = my_stages + cstage * Stage<D>::kBytes;
            const uint8_t* vs = ks + Stage<D>::kSide;
            const float4 sc4 = *reinterpret_cast<const float4*>(my_scales + cstage * 4);
            const float kscale[2] = {sc4.x, sc4.z};
            float vscale[2] = {sc4.y, sc4.w};
            const int tok0 = at.token(u);
            // ---- scores: 2 x 16 tokens x 8 NT query rows ----
            float s[2][NT][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float s2[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[h][nt][0] = s[h][nt][1] = s[h][nt][2] = s[h][nt][3] = s2[nt][0] = s2[nt][1] = s2[nt][2] = s2[nt][3] = 0.f;
#pragma unroll
                for (int c16 = 0; c16 < kWords / 4; ++c16) {
                    const int ch = (kWords / 4) * t + c16;
                    const uint4 r0 = *reinterpret_cast<const uint4*>(ks + h * Stage<D>::kHalf + Stage<D>::at(g, ch));
                    const uint4 r1 = *reinterpret_cast<const uint4*>(ks + h * Stage<D>::kHalf + Stage<D>::at(g + 8, ch));
                    const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = 4 * c16 + i;
                        uint32_t a0, a1, a2, a3;
                        decode4<E4M3>(w0[i], a0, a2);
                        decode4<E4M3>(w1[i], a1, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816(i & 1 ? s2[nt] : s[h][nt], a0, a1, a2, a3, qh[nt][k][0], qh[nt][k][1]);
                            if constexpr (kSplit) mma16816(i & 1 ? s2[nt] : s[h][nt], a0, a1, a2, a3, ql[nt][k][0], ql[nt][k][1]);
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[h][nt][e] = (s[h][nt][e] + s2[nt][e]) * (kscale[h] * qscale[nt][e & 1]);
            }
            // ---- online softmax; lane's scores: tokens g, g + 8 of each half, of the columns 2t, 2t + 1 ----
            const bool edge = fminf(kscale[0], kscale[1]) < 0.f || tok0 + kUnit - 1 > all_see_to || (p.window > 0 && tok0 < all_see_from);
            if (edge) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int tok = tok0 + h * kKv8Unit + g + 8 * (e >> 1), lim = limit[nt][e & 1];
                            if (kscale[h] < 0.f || tok > lim || (p.window > 0 && tok <= lim - p.window)) s[h][nt][e] = -INFINITY;
                        }
            }
            bool rise = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) rise |= fmaxf(vscale[0], vscale[1]) * fmaxf(lift[nt][0], lift[nt][1]) > kWeightScale;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) rise |= fmaxf(fmaxf(s[0][nt][j], s[0][nt][2 + j]), fmaxf(s[1][nt][j], s[1][nt][2 + j])) > m[nt][j];
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (!(vscale[h] >= 1.17549435e-38f)) vscale[h] = isnan(vscale[h]) ? vscale[h] : 0.f;
            if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float corr[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float mx = fmaxf(m[nt][j], fmaxf(fmaxf(s[0][nt][j], s[0][nt][2 + j]), fmaxf(s[1][nt][j], s[1][nt][2 + j])));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        corr[j] = mx == -INFINITY ? 1.f : fast_exp2(m[nt][j] - mx);
                        m[nt][j] = mx;
                        l[nt][j] *= corr[j];
                        float top = 0.f;        // the largest value scale that the column sees: a block that it does not see may be of any size
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int from = tok0 + h * kKv8Unit, lim = limit[nt][j];
                            if (!edge || (from <= lim && !(p.window > 0 && from + kKv8Unit - 1 <= lim - p.window))) top = fmaxf(top, vscale[h]);
                        }
                        const float old = lift[nt][j];
                        lift[nt][j] = top * old > kWeightScale ? lift_below(top) : old;
                        corr[j] *= lift[nt][j] * inverse_lift(old);
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[nt][i][e] *= corr[e & 1];
                            if constexpr (kSplit) keep[i][e] *= corr[e & 1];
                        }
                    }
                }
            }
            uint32_t wh[2][NT][2], wl[2][kSplitW ? NT : 1][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float pr = fast_exp2(s[h][nt][e] - (m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1]));
                        l[nt][e & 1] += pr;
                        w[e] = pr * (vscale[h] * lift[nt][e & 1]);
                        if (edge && s[h][nt][e] == -INFINITY) w[e] = 0.f;      // a hidden row of a block with a NaN scale weighs nothing
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if constexpr (kSplitW) {
                            uint32_t hi, lo;
                            split_half2(w[2 * x], w[2 * x + 1], hi, lo);
                            wh[h][nt][x] = transpose8x8(hi);
                            wl[h][nt][x] = transpose8x8(lo);
                        } else if constexpr (Pairs) {
                            uint32_t hi, lo;
                            split_half2(w[2 * x], w[2 * x + 1], hi, lo);
                            wh[h][nt][x] = transpose8x8(t < 2 ? hi : lo);
                        } else {
                            wh[h][nt][x] = transpose8x8(half2_bits(w[2 * x], w[2 * x + 1]));
                        }
                    }
                }
            }
            // ---- outputs: D dims x 8 NT query rows, token pairs (2t, 2t + 1) and 8 further ----
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t v[4][kOwn / 4];
#pragma unroll
                for (int rr = 0; rr < 4; ++rr) {
                    // D = 64: two rows share 128 bytes, so every other lane takes its pair of rows the other way round
                    const int row = 2 * t + ((rr ^ odd) & 1) + 8 * (rr >> 1);
                    if constexpr (D == 128) {
                        const uint4 x = *reinterpret_cast<const uint4*>(vs + h * Stage<D>::kHalf + Stage<D>::at(row, g));
                        v[rr][0] = x.x; v[rr][1] = x.y; v[rr][2 % (kOwn / 4)] = x.z; v[rr][3 % (kOwn / 4)] = x.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2*>(vs + h * Stage<D>::kHalf + Stage<D>::at(row, g >> 1) + (g & 1) * 8);
                        v[rr][0] = x.x; v[rr][1] = x.y;
                    }
                }
                if (edge) {             // bytes that are nobody's row may be codes of NaN
#pragma unroll
                    for (int rr = 0; rr < 4; ++rr) {
                        const bool nobody = kscale[h] < 0.f || tok0 + h * kKv8Unit + 2 * t + ((rr ^ odd) & 1) + 8 * (rr >> 1) >= at.r.len;
#pragma unroll
                        for (int i = 0; i < kOwn / 4; ++i) v[rr][i] = nobody ? 0u : v[rr][i];
                    }
                }
#pragma unroll
                for (int i = 0; i < kOwn / 4; ++i) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {      // dims 4 i + 2 x, 4 i + 2 x + 1 of the lane's own
                        uint32_t a0, a1, a2, a3;
                        decode4<E4M3>(__byte_perm(v[0][i], v[1][i], x ? pairs_hi : pairs_lo), a0, a1);
                        decode4<E4M3>(__byte_perm(v[2][i], v[3][i], x ? pairs_hi : pairs_lo), a2, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816(o[nt][2 * i + x], a0, a1, a2, a3, wh[h][nt][0], wh[h][nt][1]);
                            if constexpr (kSplitW) mma16816(o[nt][2 * i + x], a0, a1, a2, a3, wl[h][nt][0], wl[h][nt][1]);
                        }
                    }
                }
            }
            if constexpr (kSplit) {
                if (++since == 8) {
                    since = 0;
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) { keep[i][e] += o[0][i][e]; o[0][i][e] = 0.f; }
                    }
                }
            }
            if constexpr (Long) {
                if (++since == kSumUnits) {
                    since = 0;
                    if (begun) add_sums();
                    begun = true;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            __stcg(sums + (nt * (MT + 1) + i) * 32, make_float4(o[nt][i][0], o[nt][i][1], o[nt][i][2], o[nt][i][3]));
                            o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
                        }
                        __stcg(sums + (nt * (MT + 1) + MT) * 32, make_float4(m[nt][0], m[nt][1], lift[nt][0], lift[nt][1]));
                    }
                }
            }
            cstage = cstage + 1 == kStages ? 0 : cstage + 1;
            cphase ^= cstage == 0 ? 1 : 0;
        }

        if (Long && begun) add_sums();
        const Place done = at;
        left -= seg;
        if (left > 0) {
            at.next_item(p);
            load_queries();
        }
        // ---- join the warps of the CTA ----
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float back[2] = {inverse_lift(lift[nt][0]), inverse_lift(lift[nt][1])};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
                l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
                l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (kSplit) o[nt][i][e] += keep[i][e];
                    o[nt][i][e] *= back[e & 1];
                }
            }
        }
        auto leave = [&](int slot) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int col = nt * 8 + 2 * t + j;
                    if (g == 0) *reinterpret_cast<float2*>(join_ml + (slot * kRows + col) * 2) = make_float2(m[nt][j], l[nt][j]);
                    float* row = join + (slot * kRows + col) * kJoinRow + 2 * g;   // dim kOwn g + 2 i + e at 16 i + 2 g + e
#pragma unroll
                    for (int i = 0; i < MT; ++i) *reinterpret_cast<float2*>(row + 16 * i) = make_float2(o[nt][i][j], o[nt][i][2 + j]);
                }
            }
        };
        if (warp >= kJoin) leave(warp - kJoin);
        __syncthreads();
        if (warp < kJoin) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int col = nt * 8 + 2 * t + j;
                    const float2 ml = *reinterpret_cast<const float2*>(join_ml + (warp * kRows + col) * 2);
                    const float M = fmaxf(m[nt][j], ml.x), M0 = M == -INFINITY ? 0.f : M;
                    const float mine = fast_exp2(m[nt][j] - M0), other = fast_exp2(ml.x - M0);
                    m[nt][j] = M;
                    l[nt][j] = l[nt][j] * mine + ml.y * other;
                    const float* row = join + (warp * kRows + col) * kJoinRow + 2 * g;
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const float2 v = *reinterpret_cast<const float2*>(row + 16 * i);
                        o[nt][i][j] = o[nt][i][j] * mine + v.x * other;
                        o[nt][i][2 + j] = o[nt][i][2 + j] * mine + v.y * other;
                    }
                }
            }
            __syncwarp();            // the slot has been read before it is filled again
            leave(warp);
        }
        __syncthreads();
        const bool whole = done.unit == 0 && seg == done.r.units;
        const int cols = min(kRows, rows - rt * kRows);
        for (int e = threadIdx.x; e < cols * (D / 2); e += kThreads) {
            const int col = e / (D / 2), d = (e % (D / 2)) * 2;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kJoin; ++w) M = fmaxf(M, join_ml[(w * kRows + col) * 2]);
            const float M0 = M == -INFINITY ? 0.f : M;
            float L = 0.f, x = 0.f, y = 0.f;
            const int pos = 16 * ((d % kOwn) / 2) + 2 * (d / kOwn);
#pragma unroll
            for (int w = 0; w < kJoin; ++w) {
                const float f = fast_exp2(join_ml[(w * kRows + col) * 2] - M0);
                float2 v = *reinterpret_cast<const float2*>(join + (w * kRows + col) * kJoinRow + pos);
                if constexpr (Pairs) {
                    const float2 low = *reinterpret_cast<const float2*>(join + (w * kRows + col + 4) * kJoinRow + pos);
                    v = make_float2(v.x + low.x, v.y + low.y);
                }
                L = fmaf(f, join_ml[(w * kRows + col) * 2 + 1], L);
                x = fmaf(f, v.x, x);
                y = fmaf(f, v.y, y);
            }
            if (whole) {
                const int r = rt * kRows + col;
                const float inv = L == 0.f ? 0.f : 1.f / L;
                T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(done.r.begin + r / p.group) * p.out_token + (head * p.group + r % p.group) * p.out_head + d;
                store_pair(dst, x * inv, y * inv);
            } else {
                float* dst = p.partial + ((static_cast<int64_t>(cta) * 2 + (first_segment ? 0 : 1)) * kRows + col) * partial_stride<D>();
                if (d == 0) { dst[0] = M; dst[1] = L; }
                store_pair(dst + 4 + d, x, y);
            }
        }
        __syncthreads();
        first_segment = false;
    }
    cp_async_wait<0>();
    if (*abort_flag) {                  // a wait gave up: the copies that are still on their way write into this CTA's memory
        const uint64_t start = global_timer_ns();
        for (int k = max(0, produced - kStages); k < produced; ++k)
            while (!mbar_try_wait(my_bars + k % kStages, (k / kStages) & 1) && global_timer_ns() - start < 1000000000ull) {}
    }
}

// Joins the partials of the items that more than one CTA worked on.  At most one item begins in a CTA's range and goes on behind it: block
// (c, row) looks for that of CTA c and, if there is one, joins query row `row` of it: its warps take the parts in turn, a lane D / 32 dims.
constexpr int kJoinThreads = 256;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kJoinThreads) kv8_decode_join_kernel(const __grid_constant__ Kv8Decode p) {
    constexpr int kWarps = kJoinThreads / 32, kRows = decode_rows<NT>(), V = D / 32;
    __shared__ ListScratch scratch;
    __shared__ float ml[kWarps][2], rows[kWarps][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.y;
    // every block waits, also one with nothing to do: this grid must not end before the one whose partials it stands for
    auto wait = [] { asm volatile("griddepcontrol.wait;" ::: "memory"); };
    const int cta = blockIdx.x;
    const Found list = find_in_list(p, &scratch, [&](int64_t total) {
        const int n = used_ctas(total, gridDim.x);
        return cta < n - 1 ? cta_begin(total, n, cta + 1) - 1 : -1;
    });
    const int64_t total = list.total;
    const int n = used_ctas(total, gridDim.x);
    if (cta >= n - 1) { wait(); return; }
    const int64_t begin = cta_begin(total, n, cta), end = cta_begin(total, n, cta + 1);
    const Place last = list.place;
    const int64_t item_begin = end - 1 - last.unit, item_end = item_begin + last.r.units;
    const int head = last.item / last.r.row_tiles, r = (last.item % last.r.row_tiles) * kRows + row;
    const int last_cta = cta_of(total, n, item_end - 1);
    wait();
    if (item_end <= end || item_begin < begin || r >= last.r.n * p.group) return;
    float M = -INFINITY, L = 0.f, acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    for (int c = cta + warp; c <= last_cta; c += kWarps) {
        const int slot = c == cta && item_begin > begin ? 1 : 0;
        const float* src = p.partial + ((static_cast<int64_t>(c) * 2 + slot) * kRows + row) * partial_stride<D>();
        const float m = __ldcg(src), m_new = fmaxf(M, m), m0 = m_new == -INFINITY ? 0.f : m_new;
        const float f_old = fast_exp2(M - m0), f = fast_exp2(m - m0);
        L = L * f_old + __ldcg(src + 1) * f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = acc[i] * f_old + __ldcg(src + 4 + lane * V + i) * f;
        M = m_new;
    }
    if (lane == 0) { ml[warp][0] = M; ml[warp][1] = L; }
#pragma unroll
    for (int i = 0; i < V; ++i) rows[warp][lane * V + i] = acc[i];
    __syncthreads();
    if (threadIdx.x < D / 2) {
        const int d = threadIdx.x * 2;
        float A = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) A = fmaxf(A, ml[w][0]);
        const float A0 = A == -INFINITY ? 0.f : A;
        float S = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = fast_exp2(ml[w][0] - A0);
            S = fmaf(f, ml[w][1], S);
            x = fmaf(f, rows[w][d], x);
            y = fmaf(f, rows[w][d + 1], y);
        }
        const float inv = S == 0.f ? 0.f : 1.f / S;
        T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(last.r.begin + r / p.group) * p.out_token + (head * p.group + r % p.group) * p.out_head + d;
        store_pair(dst, x * inv, y * inv);
    }
}

}  // namespace
int kv8_sm_count() {
    int device = 0, sms = 0;
    if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) sms = 0;
    return sms;
}
namespace {
bool long_visits(const er_kv8_cache* c, const er_kv8_attention_params* u) {
    if (u->type == ER_TYPE_FLOAT32) return false;
    const uint64_t rows = kv8_table_rows(c);
    return (u->sliding_window > 0 ? std::min<uint64_t>(rows, static_cast<uint64_t>(u->sliding_window) + 64) : rows) > kPlainRows;
}
// Two columns of eight query rows where they are needed and fit: float32 rows take two operands each and stay at eight.
int tiles_of(uint32_t type, int rows) { return type != ER_TYPE_FLOAT32 && rows > 8 ? 2 : 1; }

// Codes as a 2-D tensor of bytes, swizzled as the kernel reads them: rows of 128 (64) bytes, 16-byte chunk c of row r at c ^ (r % 8) (c ^ (r / 2 % 4)).
bool encode_rows(CUtensorMap* map, const uint8_t* codes, const Kv8Cache& c, int head_dim) {
    const EncodeTiledFn fn = tensor_map_encode_entry();
    if (fn == nullptr) return false;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(c.num_pages) * c.num_kv_heads * c.page_size};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(head_dim)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(head_dim), kKv8Unit}, one[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, bool E4M3, int NT, bool Long, bool Pairs>
int32_t launch(Kv8Decode& p, int most_rows, int sms, cudaStream_t s) {
    constexpr int kSmem = decode_smem<T, D, NT>();
    static_assert(kSmem <= 232448, "decode kernel exceeds the shared memory of an sm_100 CTA");
    p.tile_rows = Pairs ? 4 : 8 * NT;
    static std::atomic<uint64_t> devices{0};
    cudaError_t e = kv8_allow_smem(kv8_decode_kernel<T, D, E4M3, NT, Long, Pairs>, kSmem, devices);
    if (e != cudaSuccess) return kv8_launched(e, "kv8_decode_kernel");
    kv8_decode_kernel<T, D, E4M3, NT, Long, Pairs><<<sms, decode_warps<T, NT>() * 32, kSmem, s>>>(p);
    const int32_t rc = kv8_launched(cudaGetLastError(), "kv8_decode_kernel");
    if (rc != ER_OK) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(sms, p.starts != nullptr ? 8 * NT : std::min(8 * NT, most_rows));
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kv8_decode_join_kernel<T, D, NT>, p);
    return kv8_launched(e, "kv8_decode_join_kernel");
}
template <typename T, int D, bool E4M3>
int32_t launch_rows(Kv8Decode& p, int most_rows, int sms, cudaStream_t s) {
    if constexpr (sizeof(T) == 2) {
        const bool two = tiles_of(ER_TYPE_FLOAT16, most_rows) == 2;
        if constexpr (std::is_same<T, __half>::value) {
            if (p.starts == nullptr && most_rows <= 4)
                return p.sums != nullptr ? launch<T, D, E4M3, 1, true, true>(p, most_rows, sms, s) : launch<T, D, E4M3, 1, false, true>(p, most_rows, sms, s);
        }
        if (p.sums != nullptr) return two ? launch<T, D, E4M3, 2, true, false>(p, most_rows, sms, s) : launch<T, D, E4M3, 1, true, false>(p, most_rows, sms, s);
        if (two) return launch<T, D, E4M3, 2, false, false>(p, most_rows, sms, s);
    }
    return launch<T, D, E4M3, 1, false, false>(p, most_rows, sms, s);
}
template <typename T>
int32_t launch_shape(Kv8Decode& p, int most_rows, int head_dim, bool e4m3, int sms, cudaStream_t s) {
    if (head_dim == 128) return e4m3 ? launch_rows<T, 128, true>(p, most_rows, sms, s) : launch_rows<T, 128, false>(p, most_rows, sms, s);
    return e4m3 ? launch_rows<T, 64, true>(p, most_rows, sms, s) : launch_rows<T, 64, false>(p, most_rows, sms, s);
}

}  // namespace

// Checks shared by the two attention operators.
int32_t kv8_check_attention(const er_kv8_cache* c, const er_kv8_attention_params* u) {
    if (!u->q || !u->out) return report_error(ER_ERR_INVALID_ARGUMENT, "null argument");
    if (u->type > ER_TYPE_BFLOAT16) return report_error(ER_ERR_INVALID_ARGUMENT, "type must be one of ER_TYPE_*");
    if (u->num_heads == 0 || u->num_heads % c->num_kv_heads != 0) return report_error(ER_ERR_SHAPE, "num_heads must be a multiple of num_kv_heads");
    if (u->num_heads > 65535u || static_cast<uint64_t>(u->num_tokens) * (u->num_heads / c->num_kv_heads) > (1u << 30))
        return report_error(ER_ERR_UNSUPPORTED, "num_heads beyond 65535, or more than 2^30 query rows of a kv head");
    if (!kv8_aligned(u->q) || !kv8_aligned(u->out)) return report_error(ER_ERR_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
    const int64_t vec = u->type == ER_TYPE_FLOAT32 ? 4 : 8;
    for (const int64_t st : {u->q_token_stride, u->q_head_stride, u->out_token_stride, u->out_head_stride})
        if (st < 0 || st % vec != 0) return report_error(ER_ERR_INVALID_ARGUMENT, "strides must be multiples of 16 bytes");
    if (!kv8_rows_apart(u->out_token_stride, u->out_head_stride, u->num_tokens, u->num_heads, c->head_dim)) return report_error(ER_ERR_SHAPE, "rows of out overlap");
    if (!(u->softmax_scale >= 0.f && std::isfinite(u->softmax_scale))) return report_error(ER_ERR_INVALID_ARGUMENT, "softmax_scale must be finite and not negative");
    if (u->num_tokens > 0x7FFFFF00u || u->sliding_window > 0x7FFFFFFFu) return report_error(ER_ERR_UNSUPPORTED, "num_tokens or sliding_window beyond 2^31");
    if (u->sliding_window > 0 && u->sliding_window < kv8_table_rows(c) && kv8_table_rows(c) + u->num_tokens > 0x7FFFFFFFull)
        return report_error(ER_ERR_UNSUPPORTED, "with a window, num_tokens and the rows that a block table addresses must stay below 2^31 together");
    return ER_OK;
}

// Rows of the longest sequence, as far as the host knows.
static int most_rows_of(const er_kv8_cache* c, const er_kv8_attention_params* u, bool ragged) {
    uint64_t n = u->query_len;
    if (ragged) n = u->max_query_len > 0 ? std::min(u->max_query_len, u->num_tokens) : u->num_tokens;
    return static_cast<int>(std::min<uint64_t>(n * (u->num_heads / c->num_kv_heads), 1u << 30));
}

// Bytes of the partial rows of a grid of `sms` CTAs, and behind them of the sums of long visits (12 warps at most).
static int64_t partial_bytes(const er_kv8_cache* c, const er_kv8_attention_params* u, int sms, int most_rows) {
    return static_cast<int64_t>(sms) * 2 * 8 * tiles_of(u->type, most_rows) * (c->head_dim + 4) * 4;
}
int64_t kv8_decode_workspace(const er_kv8_cache* c, const er_kv8_attention_params* u, bool ragged) {
    const int sms = kv8_sm_count(), most_rows = most_rows_of(c, u, ragged), tiles = tiles_of(u->type, most_rows);
    if (sms == 0) return report_error(ER_ERR_CUDA, "no CUDA device (no CPU fallback)");
    return partial_bytes(c, u, sms, most_rows) + (long_visits(c, u) ? static_cast<int64_t>(sms) * (tiles == 1 ? 12 : 8) * tiles * (c->head_dim / 16 + 1) * 32 * 16 : 0);
}

int32_t kv8_check_workspace(const er_kv8_attention_params* u, int64_t need) {
    if (need < 0) return static_cast<int32_t>(need);
    if (need > 0 && (!u->workspace || u->workspace_bytes < static_cast<uint64_t>(need)))
        return report_error(ER_ERR_INVALID_ARGUMENT, "workspace is smaller than er_kv8_*_workspace_bytes");
    if (!kv8_aligned(u->workspace)) return report_error(ER_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    return ER_OK;
}

// The kernel over a checked call.  ragged: queries by query_starts, of the sequences with up to `few_rows` query rows (0: all).
int32_t kv8_launch_decode(const Kv8Cache& cache, const er_kv8_cache* c, const er_kv8_attention_params* u, bool ragged, int few_rows, cudaStream_t s) {
    const int most_rows = few_rows > 0 ? std::min(few_rows, most_rows_of(c, u, ragged)) : most_rows_of(c, u, ragged);
    const bool e4m3 = c->format == ER_KV8_E4M3;
    Kv8Decode p{};
    p.cache = cache;
    p.q = u->q; p.out = u->out;
    p.q_token = u->q_token_stride; p.q_head = u->q_head_stride; p.out_token = u->out_token_stride; p.out_head = u->out_head_stride;
    p.partial = static_cast<float*>(u->workspace);
    p.starts = ragged ? u->query_starts : nullptr;
    p.num_tokens = static_cast<int>(u->num_tokens);
    p.few_rows = few_rows;
    p.group = static_cast<int>(u->num_heads) / cache.num_kv_heads;
    p.query_len = static_cast<int>(u->query_len); p.window = kv8_window(c, u);
    if (!encode_rows(&p.maps[0], cache.codes[0], cache, static_cast<int>(c->head_dim)) || !encode_rows(&p.maps[1], cache.codes[1], cache, static_cast<int>(c->head_dim)))
        return report_error(ER_ERR_CUDA, "cuTensorMapEncodeTiled refused the cache's shape");
    p.scale_log2 = kv8_scale_log2(u->softmax_scale, c->head_dim);
    const int sms = kv8_sm_count(), d = static_cast<int>(c->head_dim);
    if (long_visits(c, u)) p.sums = reinterpret_cast<float4*>(static_cast<uint8_t*>(u->workspace) + partial_bytes(c, u, sms, most_rows_of(c, u, ragged)));
    switch (u->type) {
        case ER_TYPE_FLOAT32: return launch_shape<float>(p, most_rows, d, e4m3, sms, s);
        case ER_TYPE_FLOAT16: return launch_shape<__half>(p, most_rows, d, e4m3, sms, s);
        default: return launch_shape<__nv_bfloat16>(p, most_rows, d, e4m3, sms, s);
    }
}

}  // namespace er

extern "C" int64_t er_kv8_decode_workspace_bytes(const er_kv8_cache* cache, const er_kv8_attention_params* u) {
    using namespace er;
    if (!cache || !u || cache->num_kv_heads == 0) return report_error(ER_ERR_INVALID_ARGUMENT, "null argument");
    return kv8_decode_workspace(cache, u, false);
}

extern "C" int32_t er_kv8_attention_decode(const er_kv8_cache* cache, const er_kv8_attention_params* u, void* stream) {
    using namespace er;
    if (!cache || !u) return report_error(ER_ERR_INVALID_ARGUMENT, "null argument");
    Kv8Cache c{};
    int32_t rc = kv8_check(cache, &c);
    if (rc == ER_OK) rc = kv8_check_attention(cache, u);
    if (rc != ER_OK) return rc;
    if (u->query_len == 0 || u->query_len > 16) return report_error(ER_ERR_UNSUPPORTED, "query_len must be between 1 and 16 (longer runs: er_kv8_attention_prefill)");
    if (u->num_tokens != static_cast<uint64_t>(cache->num_seqs) * u->query_len) return report_error(ER_ERR_SHAPE, "num_tokens must be num_seqs * query_len");
    rc = kv8_check_device(cache->keys);
    if (rc == ER_OK) rc = kv8_check_workspace(u, kv8_decode_workspace(cache, u, false));
    if (rc != ER_OK || cache->num_seqs == 0) return rc;
    return kv8_launch_decode(c, cache, u, false, 0, static_cast<cudaStream_t>(stream));
}
