// Decode attention over a cache held in 4 bits (format: q4.cuh): one new token per request.
//
//   o_h = sum_t p_t v_t   p = softmax over the keys in sight of scale * q_h . k_t (a sink, a distance bias: as in attention.cu)
//
// with k_t and v_t read straight from their codes.  A row is mid + scale (code - 7.5) = z + scale (code - 7), z = mid - scale / 2, and codes less 7 are
// small whole numbers that float16 holds exactly, so
//
//   q . k_t = scale_t (q . (code_t - 7)) + z_t sum(q)                      the product on the tensor cores, the rest per score in float32
//   o       = sum_t (p_t scale_t) (code_t - 7) + sum_t p_t z_t             the same for the values
//
// The tensor cores' operands are float16:
//   * codes less 7: a nibble n under the exponent of 1024 is 1024 + n, in the next four bits 1024 + 16 n, and one addition or multiply-add (two
//     codes an instruction) leaves n - 7.  (A nibble alone is the subnormal number n 2^-24 and would need neither, but the tensor cores align what
//     they add by the operands' exponent fields: sums of such products were off by 1e-4.  The 7 is taken off the codes rather than out of the
//     sums, where it would grow over the keys and lose what cancels.)
//   * q times a power of two per head that brings its largest element to 2^14 .. 2^15 (taken out of the scores again): a bfloat16 element loses
//     bits only if it is 2^-29 of the largest, and then at most 2^-40 of that; a float32 q goes in as two parts, 22 bits and more.  (Codes of K as
//     unsigned bytes against q as whole numbers in two bytes take three instructions a word instead of nine, 64 requests of up to 8,192 keys 47.3 us
//     where this took 51.1, but the keys' weights were then off by 4e-6 instead of 2e-7; with three bytes it was 51.5.)
//   * the weights p_t scale_t in float16, formed relative to the running maximum M of score_t + e_t, e_t the exponent of the key's own scale (of its mid
//     less 20 where that is more), so that they stay below 2^16, whatever the scales are, and are rounded once (2^-11 of a weight, or 2^-35 of the
//     largest where that is more; two parts for a float32 model).  The unrounded p_t enter the sum of the middles.  The denominator is a sum of its own,
//     of 2^(score - largest score): a weight may vanish beside those of larger values, its probability must not.  (Formed of the weights, the
//     exponents put back: 2 to 4 % less time, and wrong from rows 2^73 times the others' size on.)
// For a float32 model the products of each chunk of 16 keys are added to the running sums in float32 registers: in the tensor cores' own accumulation
// over thousands of keys every step's cut-off adds up (measured behind 8,000 keys: 3.9e-6 of the output's norm against 0.5e-6).
//
// A warp takes a range of keys of one (request, key/value head) for up to 16 query heads that share it, in the transposed form (16 keys in the M
// dimension of mma.sync m16n8k16, eight heads in N):
//   S^T [16 keys x 8 heads] = (C_k - 7) [16 x hd] . Q^T     a lane's words of a key row hold eight codes each, two neighbouring dimensions in a
//                             register's halves as the A fragment wants them;
//   O^T [hd x 8 heads] += (C_v - 7)^T [hd x 16 keys] . P^T  the A fragment wants one dimension of two keys in a register: a byte permute joins
//                             the same byte of two keys' words, and its two nibbles are two dimensions (two row tiles' halves).
// A group of more heads is served by several warps (that each read its rows, from the L2 after the first).
// M is raised only when a score exceeds it by more than 2^4: until then the weights are formed relative to the old one, which saves the exchange
// between lanes and the correction of the sums in nearly every chunk.
//
// The cut: every (request, key/value head) is cut into ranges of one length, a warp each (plan_ranges).  The warps of a block that have ranges of
// one (request, head) join them in shared memory; what covers it whole is the output, else the block leaves one partial result, and the block that
// is the last to do so joins those, in ascending order; in both joins the heads go round the block's warps.  (With one partial result per warp, joined
// by the last warp, a request of 131,000 tokens took 270 us, most of it in that.)
//
// Memory: a warp's ring in shared memory is filled by bulk copies, up to 64 keys at a time: codes and factors of K, then of V.  (A whole page of
// 64 tokens is one run of bytes per plane; of other pages a lane each asks for the codes and the factors.)  Every wait is bounded: when the limit
// runs out the warp records it in the module's error word, waits for its other copies with the same limit and goes on to the end without a further copy.
// What a key's four factors come to is worked out by one lane and left in the place of its chunks' codes of K, which are in registers by then: all
// four lanes of a row of fragments need it (64 requests of up to 8,192 keys: 52.6 -> 51.1 us).
// Dead keys of an edge chunk (before a window, behind the range's end) have their factors replaced, as unwritten factors may be any bits; codes of
// any bits are numbers.
//
// What bounds it (16 + 16 heads of 128, bfloat16; 12 warps of 163 registers, 104 KB of copies on their way per SM): the instructions that take codes
// apart and the latencies between them, at three warps a scheduler.  A copy of the kernel without the arithmetic (descriptors, cut, copies and joins as
// they are) takes 37.5 of the 52.1 us of 64 requests of 777 to 8,192 keys (28 heads on 4; 171 MB, 3.3 TB/s): the last keys are there at 31 us instead of
// 47, of 8 requests of 4,096 keys (71 MB, which the L2 holds from call to call) 11.9 of 25.5.  For few keys it is latency:
// descriptors and cut 3 to 4 us, first page ids and rows 2 to 2.7, joins 1 to 6.  Sixteen warps of 128 registers, eight of 255, one or four chunks at a
// time, smaller stages: slower by 3 to 18 % (for 8 requests of 4,096 keys).
//
// With weights: the scores are written out as they are formed, and a second kernel (q4_weigh_kernel) adds every key's p_t, summed over the heads
// of its group, to a number per (slot, key/value head).  The softmax's denominator is known only behind the last range.
#include <cuda_fp16.h>

#include "distance.cuh"
#include "mask.cuh"
#include "q4.cuh"
#include "sink.cuh"

struct Q4Args {
    const void* q;            // [T, nh * hd]
    const uint8_t* pool;      // this layer's pages
    void* out;                // [T, nh * hd]
    const int* seg_q0;
    const int* seg_ctx;
    const int* block_table;
    int table_stride;
    const int* items;         // [n_items] segments with one new token
    int nh, nkv, page_tokens, window, chunk;  // (mask.cuh)
    const float* sink_val;
    int keep_first, sink;
    const float* slopes;
    float scale;
    float* part_o;            // [ranges * nh][hd]
    float* part_ml;           // [ranges * nh][2]
    int* counters;            // [n_items * nh], zero between launches
    float* scores;            // with weights: [n_items][nkv][table_stride * P][heads of a group], in base 2
    float* lse;               // with weights: [n_items * nh][2], what a head's weights are relative to, and 1 / denominator
    uint32_t k1024;           // 0x64006400, 1024 twice in float16: as an argument it stays in a register (codes_low)
};

#define Q4_WAIT_LIMIT 2000000000LL   // cycles a warp waits for a copy before it gives up (about a second)

__device__ int g_q4_error = 0;
extern "C" int locus_attn_q4_error() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_q4_error, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_q4_error, &zero, sizeof(int));
    }
    return v;
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (clock64() - t0 > Q4_WAIT_LIMIT) {
            atomicCAS(&g_q4_error, 0, 1);
            return false;
        }
    }
    return true;
}
// `bytes` (a multiple of 16) from global to shared memory, both 16-byte aligned; completion on the mbarrier
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// this thread's accesses to shared memory so far come before copies into it that are issued behind the next barrier
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// N (1, 2, 4 or 8) words of shared memory
template <int N>
__device__ __forceinline__ void lds_words(uint32_t* v, const unsigned char* p) {
    if constexpr (N == 1) {
        v[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        v[0] = x.x; v[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(p + 4 * i);
            v[i] = x.x; v[i + 1] = x.y; v[i + 2] = x.z; v[i + 3] = x.w;
        }
    }
}

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of 16-bit elements held as mma fragments (two elements of a row per lane)
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 halves(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
// the codes in bits 0 .. 3 of a register's halves, less 7: 0x6400 | n is 1024 + n.  (Mask and exponent in one LOP3 need one of the two constants in
// a register; from two immediates the compiler makes two instructions.)
__device__ __forceinline__ uint32_t codes_low(uint32_t x, uint32_t k1024) {
    return bits(__hsub2(halves((x & 0x000f000fu) | k1024), halves(0x64076407u)));
}
// the codes in bits 4 .. 7: (1024 + 16 n) / 16 - 71
__device__ __forceinline__ uint32_t codes_high(uint32_t x, uint32_t k1024) {
    return bits(__hfma2(halves((x & 0x00f000f0u) | k1024), halves(0x2c002c00u), halves(0xd470d470u)));
}
// a pair of values as PARTS pairs of float16: one, rounded, or two
template <int PARTS>
__device__ __forceinline__ void split2(float a, float b, uint32_t* out) {
    const __half2 h = __floats2half2_rn(a, b);
    out[0] = bits(h);
    if constexpr (PARTS == 2) {
        const float2 f = __half22float2(h);
        out[1] = bits(__floats2half2_rn(a - f.x, b - f.y));
    }
}
// x 2^k in two factors: 2^k alone falls below float32's range where x 2^k does not
__device__ __forceinline__ float scale2(float x, float k) {
    const float a = fmaxf(k, -100.f);
    return x * exp2f(a) * exp2f(k - a);
}
__device__ __forceinline__ float pow2i(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }   // -126 .. 127

template <bool B>
struct Bool {
    static constexpr bool value = B;
};

// ---------------------------------------------------------------------------
// The cut of a step's keys into ranges.
#define Q4_MAX_ITEMS 1024
#define Q4_CAND 64        // candidate range lengths looked at
#define Q4_ODD 16         // what ranges that do not end where stages of 64 keys do cost more, in keys: a further stage, asked for in pieces

// What a warp of a block does in a round.
struct Q4Unit {
    int active;
    int item, vh, range, n_ranges;   // range of the item's n_ranges
    int wa, wb;                       // the warps of the block that have ranges of the same (item, head)
    int parts;                        // blocks that have some
    int lead;                         // packed: ranges of this (item, head) that its first block has
};
struct Q4Plan {
    int pos[Q4_MAX_ITEMS];       // position of item i's query
    int seg[Q4_MAX_ITEMS];
    int row[Q4_MAX_ITEMS];       // row of q / out
    int pref[Q4_MAX_ITEMS + 1];  // ranges of the items before i
    int block_pref[Q4_MAX_ITEMS + 1];   // not packed: block-loads of the items before i
    int ranges[Q4_CAND], blocks[Q4_CAND];
    int longest[32], total[32], blocks_of[32];
    Q4Unit units[16];            // this round's, by warp
    int len, packed, n_blocks;
};

// position of a segment's query, held to what its row of the table describes (and to -1, no key: no page is read then)
__device__ __forceinline__ int q4_position(const Q4Args& a, int seg) { return max(-1, min(a.seg_ctx[seg], a.table_stride * a.page_tokens - 1)); }
// first key that a query at position p sees (besides kept first tokens), rounded down to 16
__device__ __forceinline__ int q4_first(const Q4Args& a, int p) { return first_key(a.window, a.chunk, p) & ~15; }
// kept first tokens of an item that lie in front of its window's first chunk: a range of their own, the item's first
__device__ __forceinline__ int q4_kept(const Q4Args& a, int first) { return a.window > 0 ? min(a.keep_first, first) : 0; }
// Ranges of `n` keys at a length of about len (inv its reciprocal).  By a product, which may be one more than need be; the same everywhere.
__device__ __forceinline__ int q4_ranges(int n, int len, float inv) { return max(1, static_cast<int>(static_cast<float>(n + len - 1) * inv)); }
// The length of an item's ranges: all alike, whole pieces of 16, 32 or 64 keys (long ranges begin where pages do).
__device__ __forceinline__ int q4_length(int n, int ranges) {
    const int even = (n + ranges - 1) / ranges;
    const int step = even >= 512 ? 64 : even >= 128 ? 32 : 16;
    return (even + step - 1) / step * step;
}
// Blocks of W warps that an item of `ranges` ranges takes when no block holds parts of a (request, head) that another one holds parts of, unless
// it has more ranges than a block warps.  table[r], r 1 .. W: for r ranges.
template <int W>
__device__ __forceinline__ int q4_blocks(const int* table, int ranges, int n_vh) {
    return ranges > W ? n_vh * ((ranges + W - 1) / W) : table[ranges];
}

// Fills the plan (all threads of the block; ends with a barrier) and returns the length, 0 when not even one range per item fits max_ranges.
// Two ways to deal the units to blocks, for each of Q4_CAND lengths: `packed`, unit after unit, W to a block, and by whole blocks (q4_blocks), where
// some warps may have nothing to do but fewer (request, head)s are joined across blocks.  The cost of a cut, in keys: rounds over the grid x
// (length + cost_range, and Q4_ODD), and cost_join once where blocks join, and cost_merge per partial result of the longest item.  Lengths
// from what fills every warp once, 2 % apart, some shorter and longer ones, and the longest item's.
// (8 requests of 4,096 keys on 16 heads: unit after unit 3 % more than by whole blocks; 64 requests of 777 to 8,192 keys on 4: by whole blocks 19 % more than unit after
// unit.  One request of 4,096 keys on 16: ranges of 48 keys 14.5 us, of 64 13.2.)
template <int W>
__device__ __forceinline__ int plan_ranges(Q4Plan& pl, const Q4Args& a, int n_items, int n_vh, long long max_ranges, int cost_range, int cost_join,
                                           int cost_merge) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int longest = 1, total = 0;
    for (int i = tid; i < n_items; i += 32 * W) {
        const int seg = a.items[i], p = q4_position(a, seg), row = a.seg_q0[seg];
        const int first = q4_first(a, p);
        pl.row[i] = row;
        pl.pos[i] = p;
        pl.seg[i] = seg;
        longest = max(longest, p + 1 - first);
        total += p + 1 - first;
    }
    if (tid >= 1 && tid <= W) {
        const int heads = W / tid;   // (request, head)s of tid ranges that a block holds
        pl.blocks_of[tid] = (n_vh + heads - 1) / heads;
    }
    if (tid < Q4_CAND) pl.ranges[tid] = pl.blocks[tid] = 0;
    longest = __reduce_max_sync(0xffffffffu, longest);
    total = __reduce_add_sync(0xffffffffu, total);
    if (lane == 0) {
        pl.longest[warp] = longest;
        pl.total[warp] = total;
    }
    __syncthreads();
    longest = __reduce_max_sync(0xffffffffu, lane < W ? pl.longest[lane] : 1);
    total = __reduce_add_sync(0xffffffffu, lane < W ? pl.total[lane] : 0);
    const float fill = static_cast<float>(total) * static_cast<float>(n_vh) / static_cast<float>(gridDim.x * W);
    auto length = [&](int c) {
        if (c == Q4_CAND - 1) return (longest + 15) & ~15;
        const float x = static_cast<float>(c);
        const float times = c < 56 ? 1.f + 0.03f * x : c < 60 ? 0.2f * (x - 55.f) : 3.f + (x - 60.f) * (x - 60.f);
        return 16 * max(1, static_cast<int>(fminf(fill * times, 1e8f) * (1.f / 16.f) + 0.5f));
    };
    const bool kept_ranges = a.window > 0 && a.keep_first > 0;
    auto ranges_of = [&](int i, int len, float inv) {
        const int p = pl.pos[i], first = q4_first(a, p);
        return q4_ranges(p + 1 - first, len, inv) + (kept_ranges && q4_kept(a, first) > 0);
    };
    // every warp sums up some of the items, a lane two of the lengths
    const int my_len[2] = {length(lane), length(lane + 32)};
    const float my_inv[2] = {1.f / static_cast<float>(my_len[0]), 1.f / static_cast<float>(my_len[1])};
    if (warp < n_items) {
        int ranges[2] = {0, 0}, blocks[2] = {0, 0};
        for (int i = warp; i < n_items; i += W)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int r = ranges_of(i, my_len[k], my_inv[k]);
                ranges[k] += r;
                blocks[k] += q4_blocks<W>(pl.blocks_of, r, n_vh);
            }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            atomicAdd(&pl.ranges[lane + 32 * k], ranges[k]);
            atomicAdd(&pl.blocks[lane + 32 * k], blocks[k]);
        }
    }
    __syncthreads();
    if (warp == 0) {
        const float grid_inv = 1.f / static_cast<float>(gridDim.x);
        unsigned best = 0xffffffffu;   // cost << 7 | 2 candidate | packed: ties go to the shorter range
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int c = lane + 32 * k, ranges = pl.ranges[c];
            const int most = min(my_len[k], longest) + (my_len[k] & 63 ? Q4_ODD : 0) + cost_range, merge = cost_merge * (static_cast<int>(static_cast<float>(longest) * my_inv[k]) / W);
            auto consider = [&](int loads, bool joins, int packed) {
                const float rounds = floorf((static_cast<float>(loads) + static_cast<float>(gridDim.x - 1)) * grid_inv);
                const float cost = fminf(rounds * static_cast<float>(most) + static_cast<float>(merge + (joins ? cost_join : 0)), 16777215.f);
                best = min(best, static_cast<unsigned>(cost) << 7 | static_cast<unsigned>(2 * c + packed));
            };
            if (ranges <= max_ranges) {   // (the scratch holds that many partial results)
                consider(pl.blocks[c], longest > my_len[k] * W, 0);
                consider((ranges * n_vh + W - 1) / W, ranges > n_items, 1);
            }
        }
        best = __reduce_min_sync(0xffffffffu, best);
        const int packed = best & 1, len = best == 0xffffffffu ? 0 : length(static_cast<int>(best & 127u) >> 1);
        const float inv = len ? 1.f / static_cast<float>(len) : 0.f;
        int acc = 0, acc_blocks = 0;
        for (int i0 = 0; i0 < n_items; i0 += 32) {
            const int i = i0 + lane;
            int mine = 0, mine_blocks = 0;
            if (i < n_items && len) {
                mine = ranges_of(i, len, inv);
                if (!packed) mine_blocks = q4_blocks<W>(pl.blocks_of, mine, n_vh);
            }
            int run = mine, run_blocks = mine_blocks;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, run, o), w = __shfl_up_sync(0xffffffffu, run_blocks, o);
                if (lane >= o) {
                    run += v;
                    run_blocks += w;
                }
            }
            if (i < n_items) {
                pl.pref[i] = acc + run - mine;
                pl.block_pref[i] = acc_blocks + run_blocks - mine_blocks;
            }
            acc += __shfl_sync(0xffffffffu, run, 31);
            acc_blocks += __shfl_sync(0xffffffffu, run_blocks, 31);
        }
        if (lane == 0) {
            pl.pref[n_items] = acc;
            pl.block_pref[n_items] = acc_blocks;
            pl.len = len;
            pl.packed = packed;
            pl.n_blocks = packed ? (acc * n_vh + W - 1) / W : acc_blocks;
        }
    }
    __syncthreads();
    return pl.len;
}

// a / b for small whole numbers (a below 2^20 by a product)
__device__ __forceinline__ int q4_div(int a, int b) {
    return a < 1 << 20 ? static_cast<int>(__fdividef(static_cast<float>(a) + 0.5f, static_cast<float>(b))) : a / b;
}
// What warp `warp` of block-load `load` (of plan.n_blocks) does.
template <int W>
__device__ __forceinline__ Q4Unit q4_unit(const Q4Plan& pl, int load, int warp, int n_items, int n_vh) {
    Q4Unit u;
    const int at = pl.packed ? load * W + warp : load;
    auto begin = [&](int i) { return pl.packed ? pl.pref[i] * n_vh : pl.block_pref[i]; };
    int item = 0, hi = n_items;   // the last item that begins at or in front of `at`
    while (hi - item > 1) {
        const int mid = (item + hi) >> 1;
        if (begin(mid) <= at) item = mid;
        else hi = mid;
    }
    u.item = item;
    u.n_ranges = pl.pref[item + 1] - pl.pref[item];
    const int k = at - begin(item), nr = u.n_ranges;
    if (pl.packed) {
        const int left = pl.pref[n_items] * n_vh - load * W;   // units from this block's first on
        u.active = warp < left;
        u.vh = q4_div(k, nr);
        u.range = k - u.vh * nr;
        const int u0 = at - u.range;                            // the (item, head)'s first unit
        u.wa = max(0, warp - u.range);
        u.wb = min(min(W, left), warp - u.range + nr);
        u.parts = (u0 + nr - 1) / W - u0 / W + 1;
        u.lead = W - u0 % W;
    } else if (nr > W) {
        const int loads = (nr + W - 1) / W;
        u.vh = q4_div(k, loads);
        u.range = (k - u.vh * loads) * W + warp;
        u.active = u.range < nr;
        u.wa = 0;
        u.wb = min(W, nr - (u.range - warp));
        u.parts = loads;
        u.lead = W;
    } else {
        const int heads = q4_div(W, nr), h = q4_div(warp, nr);
        u.vh = k * heads + h;
        u.range = warp - h * nr;
        u.active = h < heads && u.vh < n_vh;
        u.wa = h * nr;
        u.wb = u.wa + nr;
        u.parts = 1;
        u.lead = W;
    }
    return u;
}

// T: the model's type.  HD: head size.  HT: tiles of eight heads per warp.  N: chunks of 16 keys at a time.  W warps of a block, S stages of SK keys in flight per warp.
template <typename T, int HD, int HT, int N, int W, int S, int SK, bool WEIGH>
__global__ void __launch_bounds__(32 * W, 1) attn_decode_q4_kernel(Q4Args a, int n_items, long long max_units, int cost_range, int cost_join, int cost_merge) {
    pdl_trigger();  // every block of this grid is resident from the start
    constexpr int PARTS = sizeof(T) == 4 ? 2 : 1;
    constexpr int KW = HD / 32;      // words of a lane per key row (keys): HD / 4 dimensions
    constexpr int VW = HD / 64;      // words of a lane per value row: HD / 8 dimensions
    constexpr int MT = HD / 16;      // row tiles of O^T
    constexpr int DL = HD / 32;      // dimensions of a lane where a warp has a head's row
    constexpr int RB = HD / 2;       // bytes of a row's codes
    constexpr uint32_t PLANE = SK * (RB + Q4_FACTOR_BYTES);   // K (or V) of a stage
    constexpr uint32_t STAGE = 2 * PLANE;
    constexpr float RAISE = 4.f, TOP = 10.f;   // weights are 2^TOP at M, at most 2^(TOP + RAISE + 1/2), times scale / 2^exponent < 2: below 65,504
    constexpr int LEAST = -64;                 // smallest exponent that is taken out (smaller scales leave smaller weights)
    // Denominators are kept apart from the weights that enter the sums: a row of zeros beside rows of 2^100 has a weight that adds nothing to
    // these (relative to their size it is below 2^-126) and a probability like theirs.  A warp's is relative to the largest score at the last
    // raise (relative to `from`, terms of large rows would be rounded beside exponents of 100, denominators 1e-6 off); a key that raises nothing
    // scores at most NEAR - LEAST above that, so its term stays in range.  (Values of more than 2^(NEAR - RAISE) raise at every key near M.)  A part's
    // is relative to its sums' `from` less LIFT, where the largest key's term lies between 2^(TOP - 126 + LIFT) and 2^(TOP - LEAST + RAISE + LIFT).
    constexpr float NEAR = 40.f, LIFT = 20.f;
    constexpr int MID = 20;                    // a mid's exponent counts less this: products with z / 2^exponent < 2^(MID + 2) stay in range
    extern __shared__ __align__(16) unsigned char q4_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gq = lane >> 2, t4 = lane & 3;   // row of the fragments, and the lane's place in its row
    // the key of a chunk's eight that row r of the fragments stands for, r with its low bit turned round in every other pair: rows of even
    // and of odd keys alternate both among the rows 2 t4 (values) and among neighbouring rows (keys), half the banks each
    const int kr0 = gq ^ ((gq >> 1) & 1);
    const int va_row = (2 * t4) ^ (t4 & 1), vb_row = (2 * t4 + 1) ^ (t4 & 1);
    const uint32_t k1024 = a.k1024;
    const int P = a.page_tokens, G = a.nh / a.nkv;
    const int n_sub = (G + 8 * HT - 1) / (8 * HT), n_vh = a.nkv * n_sub;   // warps that serve a group, heads of a range

    __shared__ Q4Plan pl;
    __shared__ __align__(8) unsigned long long q4_bars[W * S];
    __shared__ int is_last[W];
    const uint32_t bars = smem_u32(q4_bars) + warp * (S * 8);  // this warp's barriers, one per stage
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < S; ++i) mbar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    uint32_t parity = 0;  // bit i: the phase of stage i's barrier that the next wait on it looks for
    bool ok = true;
    const int len = plan_ranges<W>(pl, a, n_items, n_vh, max_units / a.nh, cost_range, cost_join, cost_merge);
    // (the cut read only the step's descriptors; q and the newest rows come from the kernel in front)
    pdl_entry();
    if (len == 0) return;
    const float qscale = a.scale * 1.4426950408889634f;  // scores in base 2
    const size_t plane_step = static_cast<size_t>(a.nkv) * P * (RB + Q4_FACTOR_BYTES);
    const uint32_t ring = smem_u32(q4_smem) + warp * (S * STAGE);
    // a warp's result, in its ring's place once the ring is empty: [heads][HD] sums, then [heads] pairs (maximum, denominator)
    constexpr int RES = 8 * HT * (HD + 2);
    static_assert(RES * 4 <= S * static_cast<int>(STAGE), "a warp's result fits its ring");
    float* const res0 = reinterpret_cast<float*>(q4_smem);
    constexpr int RES_STEP = S * STAGE / 4;   // floats from a warp's result to the next one's

    for (int load = blockIdx.x; load < pl.n_blocks; load += gridDim.x) {
        const Q4Unit un = q4_unit<W>(pl, load, warp, n_items, n_vh);
        if (lane == 0) pl.units[warp] = un;   // (for the joins)
        const bool active = un.active;
        const int item = un.item, vh = un.vh, range = un.range, n_ranges = un.n_ranges, wa = un.wa;
        const int kvh = n_sub == 1 ? vh : vh / n_sub, g0 = (vh - kvh * n_sub) * 8 * HT;
        const int nG = min(G - g0, 8 * HT), h0 = kvh * G + g0;   // this warp's heads: h0 .. h0 + nG - 1
        const int seg = pl.seg[item], p = pl.pos[item], first = q4_first(a, p);
        const int row = pl.row[item];
        const bool whole = un.parts == 1;

        if (active) {
            const int keep = a.keep_first, kept = q4_kept(a, first);
            const bool kept_range = kept > 0 && range == 0;
            const int t_lo = kept_range ? 0 : first_key(a.window, a.chunk, p);
            const int n_even = n_ranges - (kept > 0);
            const int length = q4_length(p + 1 - first, n_even);
            const int k_begin = kept_range ? 0 : min(p + 1, first + (range - (kept > 0)) * length);   // a multiple of 16, or no key
            const int k_end = kept_range ? kept : min(p + 1, k_begin + length);                         // exclusive
            const int* table = a.block_table + static_cast<size_t>(seg) * a.table_stride;

            // A stage of the ring: the keys of one run of SK, counted from position 0, that lie in the range.  (Every chunk holds a live key, so
            // its page is the request's: the first of a window's ranges begins with the chunk of the window's first key, and kept tokens in front
            // of that are a range of their own.)
            const int k_stop = k_begin < k_end ? (k_end + 15) & ~15 : k_begin;
            const uint8_t* const pool_head = a.pool + q4_place(0, 0, kvh, a.nkv, P, HD);
            int k0 = k_begin, k_next = k_begin;                          // first key that is not read yet; that is not asked for yet
            int page_at = k_begin / P, end_next = (page_at + 1) * P;     // page of k_next, and where it ends
            // the ids of 32 pages from page_from on, one a lane (looked up one by one, each lookup would stand in front of its copy)
            const int last_page = k_begin < k_stop ? (k_stop - 1) / P : 0;
            int page_from = page_at, page_ids = table[min(page_from + lane, last_page)];
            auto stage_end = [&](int k) { return min((k / SK + 1) * SK, k_stop); };
            auto issue = [&](int st) {
                constexpr int MOST = SK / 16;   // pages of a stage
                const int end = stage_end(k_next), n = end - k_next;
                if (page_at - page_from > 32 - MOST) {
                    page_from = page_at;
                    page_ids = table[min(page_from + lane, last_page)];
                }
                const int page = __shfl_sync(0xffffffffu, page_ids, (page_at - page_from + lane) & 31);
                const uint32_t dst = ring + st * STAGE, bar = bars + 8 * st;
                if (lane == 0) {
                    mbar_expect_tx(bar, 2 * n * (RB + Q4_FACTOR_BYTES));
                    if (n == SK && P == SK) {
                        const uint8_t* src = pool_head + page * (2 * plane_step);
                        bulk_copy(dst, src, PLANE, bar);
                        bulk_copy(dst + PLANE, src + plane_step, PLANE, bar);
                    }
                }
                if (n != SK || P != SK) {
                    __syncwarp();
                    // a page a lane
                    const int lo = lane == 0 ? k_next : end_next + (lane - 1) * P, hi = min(end, end_next + lane * P);
                    if (lane < MOST && lo < hi) {
                        const int off = lane == 0 ? k_next - (end_next - P) : 0, m = hi - lo, at = lo - k_next;
                        const uint8_t* src = pool_head + page * (2 * plane_step);
                        const uint8_t* codes = src + static_cast<size_t>(off) * RB;
                        const uint8_t* factors = src + static_cast<size_t>(P) * RB + static_cast<size_t>(off) * Q4_FACTOR_BYTES;
                        bulk_copy(dst + at * RB, codes, m * RB, bar);
                        bulk_copy(dst + SK * RB + at * Q4_FACTOR_BYTES, factors, m * Q4_FACTOR_BYTES, bar);
                        bulk_copy(dst + PLANE + at * RB, codes + plane_step, m * RB, bar);
                        bulk_copy(dst + PLANE + SK * RB + at * Q4_FACTOR_BYTES, factors + plane_step, m * Q4_FACTOR_BYTES, bar);
                    }
                }
                k_next = end;
                while (end_next <= end) {
                    ++page_at;
                    end_next += P;
                }
            };
            // q is asked for in front of the copies, whose page ids are on their way
            float x[HT][8 * KW];
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) {
                const int g = gq + 8 * ht;
                const T* q0 = static_cast<const T*>(a.q) + (static_cast<size_t>(row) * a.nh + h0 + (g < nG ? g : 0)) * HD + t4 * (HD / 4);
#pragma unroll
                for (int w = 0; w < KW; ++w) load8(q0 + 8 * w, x[ht] + 8 * w);
            }
            int st = 0;
            if (ok) {
#pragma unroll
                for (int c = 0; c < S - 1; ++c)
                    if (k_next < k_stop) issue(c);
            }

            // Q as B fragments: head gq (and gq + 8 of the second tile), dimensions t4 HD / 4 + 8 w + 4 x + {0, 1} and + {2, 3}: words w, x = 0, 1
            uint32_t qb[HT][2 * KW][2][PARTS];
            float hq[HT][2], sq[HT][2];   // of this lane's two heads per tile: the scores' factor, and times sum(q)
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) {
                const int g = gq + 8 * ht;
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 8 * KW; ++i) {
                    if (g >= nG) x[ht][i] = 0.f;
                    top = fmaxf(top, fabsf(x[ht][i]));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int k = min(14 - (static_cast<int>(__float_as_uint(top) >> 23) - 127), 126);   // (-114 for infinities)
                const float up = pow2i(k);
                float sum = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * KW; ++i) {
                    split2<PARTS>(x[ht][4 * i] * up, x[ht][4 * i + 1] * up, qb[ht][i][0]);
                    split2<PARTS>(x[ht][4 * i + 2] * up, x[ht][4 * i + 3] * up, qb[ht][i][1]);
                    sum += (x[ht][4 * i] + x[ht][4 * i + 1]) + (x[ht][4 * i + 2] + x[ht][4 * i + 3]);
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                const float down = qscale * pow2i(-k);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    hq[ht][c] = __shfl_sync(0xffffffffu, down, 4 * (2 * t4 + c));
                    sq[ht][c] = __shfl_sync(0xffffffffu, sum, 4 * (2 * t4 + c)) * qscale;
                }
            }
            // O^T: byte b of word w of a lane's value row is row tile 4 w + b: its low nibble's dimension in row gq, its high nibble's in row
            // gq + 8; columns are heads 2 t4 + {0, 1}.  l, z: this lane's share of the keys.
            float o[HT][MT][4], l[HT][2], z[HT][2], slope[HT][2];
            // A weight times 2^exponent is formed relative to `from`, up to `limit`: M - TOP and M + RAISE; no live key yet: limit -infinity.
            // l is relative to `s_from`.
            float limit[HT][2], from[HT][2], s_from[HT][2];
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
                for (int j = 0; j < MT; ++j) o[ht][j][0] = o[ht][j][1] = o[ht][j][2] = o[ht][j][3] = 0.f;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int g = 8 * ht + 2 * t4 + c;
                    limit[ht][c] = -INFINITY;
                    l[ht][c] = z[ht][c] = from[ht][c] = s_from[ht][c] = 0.f;
                    slope[ht][c] = a.slopes && g < nG ? slope_log2(a.slopes, h0 + g) : 0.f;
                }
            }

            float* const scores = WEIGH ? a.scores + (static_cast<size_t>(item) * a.nkv + kvh) * a.table_stride * P * G + g0 + 2 * t4 : nullptr;
            // N chunks of sixteen keys, from c0 (those from `stop` on are dead), whose rows lie at `at` (K; V's are PLANE further on) and factors at `fac`
            // (SPECIAL: dead keys among them, or a distance bias; a copy of its own, for the plain steps' sake)
            const bool biased_call = a.slopes != nullptr;
            auto step = [&](auto special, int c0, int stop, unsigned char* at, const unsigned char* fac) {
                constexpr bool SPECIAL = decltype(special)::value;
                const bool edge = SPECIAL && (c0 < t_lo || c0 + 16 * N > stop), biased = SPECIAL && biased_call;
                // chunk n: keys c0 + 16 n + kr0 and + 8 + kr0
                float s[N][HT][4];
                uint32_t k_lo[N][KW], k_hi[N][KW];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    lds_words<KW>(k_lo[n], at + (16 * n + kr0) * RB + t4 * (RB / 4));
                    lds_words<KW>(k_hi[n], at + (16 * n + kr0 + 8) * RB + t4 * (RB / 4));
                }
                // a key's factors, a lane each: (scales of K and, times 2^-exponent, of V | z of K | z of V times 2^-exponent | exponent)
                auto dead = [&](int key) { return edge && !((key >= t_lo || key < keep) && key < stop); };
                {
                    const int at_key = lane & (16 * N - 1);
                    uint32_t kf, vf;
                    lds_words<1>(&kf, fac + 4 * at_key);
                    lds_words<1>(&vf, fac + PLANE + 4 * at_key);
                    if (dead(c0 + at_key)) kf = vf = 0u;
                    const float kz = fmaf(-0.5f, q4_scale(kf), q4_mid(kf));
                    const int of_scale = static_cast<int>(vf << 16 & 0x7f800000u), of_mid = static_cast<int>(vf & 0x7f800000u);
                    const int top = min(__vimax3_s32(of_scale, of_mid - (MID << 23), (LEAST + 127) << 23), 253 << 23);   // (NaN: any)
                    const float ve = __int_as_float(0x4b000000 | top >> 23) - 8388735.f;   // (2^23 + 127)
                    const float down = __int_as_float((254 << 23) - top), vs = q4_scale(vf) * down, vz = fmaf(-0.5f, vs, q4_mid(vf) * down);
                    __syncwarp();
                    *reinterpret_cast<uint4*>(at + 16 * at_key) = make_uint4((__float_as_uint(vs) & 0xffff0000u) | (kf & 0xffffu), __float_as_uint(kz), __float_as_uint(vz), __float_as_uint(ve));
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
#pragma unroll
                    for (int ht = 0; ht < HT; ++ht) s[n][ht][0] = s[n][ht][1] = s[n][ht][2] = s[n][ht][3] = 0.f;
#pragma unroll
                    for (int w = 0; w < KW; ++w)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t a0 = k_lo[n][w] >> (8 * x), a1 = k_hi[n][w] >> (8 * x);
                            const uint32_t af[4] = {codes_low(a0, k1024), codes_low(a1, k1024), codes_high(a0, k1024), codes_high(a1, k1024)};
#pragma unroll
                            for (int ht = 0; ht < HT; ++ht)
#pragma unroll
                                for (int y = PARTS - 1; y >= 0; --y) mma_f16(s[n][ht], af, qb[ht][2 * w + x][0][y], qb[ht][2 * w + x][1][y]);
                        }
                }
                // scores; of the two keys of a chunk V's exponent, and scale and z of V times 2^-exponent
                float sc[N][HT][4], ve[N][2], vs[N][2], vz[N][2];
                bool raise = false;
                __syncwarp();
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int key[2] = {c0 + 16 * n + kr0, c0 + 16 * n + 8 + kr0};
                    float ks[2], kz[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint4 f = *reinterpret_cast<const uint4*>(at + 16 * (16 * n + kr0 + 8 * i));
                        ks[i] = q4_scale(f.x);
                        vs[n][i] = q4_mid(f.x);
                        kz[i] = __uint_as_float(f.y);
                        vz[n][i] = __uint_as_float(f.z);
                        ve[n][i] = __uint_as_float(f.w);
                    }
#pragma unroll
                    for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int c = i & 1, y = i >> 1;
                            float w = fmaf(s[n][ht][i], ks[y] * hq[ht][c], kz[y] * sq[ht][c]);
                            if (biased) w = fmaf(slope[ht][c], static_cast<float>(key[y] - p), w);
                            if (WEIGH) {
                                const int g = 8 * ht + 2 * t4 + c;
                                if (g < nG && !dead(key[y])) scores[static_cast<size_t>(key[y]) * G + 8 * ht + c] = w;
                            }
                            if (dead(key[y])) w = -INFINITY;
                            sc[n][ht][i] = w;
                            raise |= w + ve[n][y] > limit[ht][c];
                        }
                    }
                }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int ht = 0; ht < HT; ++ht)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float top = fmaxf(sc[0][ht][c] + ve[0][0], sc[0][ht][2 + c] + ve[0][1]), top_s = fmaxf(sc[0][ht][c], sc[0][ht][2 + c]);
#pragma unroll
                            for (int n = 1; n < N; ++n) {
                                top = fmaxf(top, fmaxf(sc[n][ht][c] + ve[n][0], sc[n][ht][2 + c] + ve[n][1]));
                                top_s = fmaxf(top_s, fmaxf(sc[n][ht][c], sc[n][ht][2 + c]));
                            }
#pragma unroll
                            for (int x = 4; x < 32; x <<= 1) {
                                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                                top_s = fmaxf(top_s, __shfl_xor_sync(0xffffffffu, top_s, x));
                            }
                            const bool none = limit[ht][c] == -INFINITY;   // (no live key so far)
                            const float now = none ? rintf(top) - TOP : fmaxf(from[ht][c], rintf(top) - TOP);
                            const float s_now = none ? rintf(top_s) : fmaxf(s_from[ht][c], rintf(top_s));
                            const float corr = none ? 0.f : ex2(from[ht][c] - now);
                            l[ht][c] = none ? 0.f : l[ht][c] * ex2(s_from[ht][c] - s_now);
                            s_from[ht][c] = s_now == -INFINITY ? 0.f : s_now;
                            limit[ht][c] = fminf(now + (TOP + RAISE), s_now + NEAR);
                            from[ht][c] = now == -INFINITY ? 0.f : now;
                            z[ht][c] *= corr;
#pragma unroll
                            for (int j = 0; j < MT; ++j) {
                                o[ht][j][c] *= corr;
                                o[ht][j][2 + c] *= corr;
                            }
                        }
                }
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    uint32_t pb[HT][2][PARTS];
#pragma unroll
                    for (int ht = 0; ht < HT; ++ht) {
                        float e[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) e[i] = ex2(sc[n][ht][i] + ve[n][i >> 1] - from[ht][i & 1]);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            l[ht][c] += ex2(sc[n][ht][c] - s_from[ht][c]) + ex2(sc[n][ht][2 + c] - s_from[ht][c]);
                            z[ht][c] = fmaf(e[c], vz[n][0], fmaf(e[2 + c], vz[n][1], z[ht][c]));
                        }
                        // P^T as the B fragment: the transpose of the accumulator layout, 8 keys at a time
                        split2<PARTS>(e[0] * vs[n][0], e[1] * vs[n][0], pb[ht][0]);
                        split2<PARTS>(e[2] * vs[n][1], e[3] * vs[n][1], pb[ht][1]);
#pragma unroll
                        for (int y = 0; y < PARTS; ++y) {
                            pb[ht][0][y] = movmatrix_trans(pb[ht][0][y]);
                            pb[ht][1][y] = movmatrix_trans(pb[ht][1][y]);
                        }
                    }
                    uint32_t v_a[2][VW], v_b[2][VW];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        lds_words<VW>(v_a[i], at + PLANE + (16 * n + 8 * i + va_row) * RB + gq * (RB / 8));
                        lds_words<VW>(v_b[i], at + PLANE + (16 * n + 8 * i + vb_row) * RB + gq * (RB / 8));
                    }
#pragma unroll
                    for (int w = 0; w < VW; ++w)
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            const uint32_t sel = b | ((4 + b) << 8);   // byte b of one key and of the other; the bytes between do not count
                            const uint32_t x0 = __byte_perm(v_a[0][w], v_b[0][w], sel), x1 = __byte_perm(v_a[1][w], v_b[1][w], sel);
                            const uint32_t af[4] = {codes_low(x0, k1024), codes_high(x0, k1024), codes_low(x1, k1024), codes_high(x1, k1024)};
#pragma unroll
                            for (int ht = 0; ht < HT; ++ht) {
                                float* t = o[ht][4 * w + b];
                                if constexpr (PARTS == 1) {
                                    mma_f16(t, af, pb[ht][0][0], pb[ht][1][0]);
                                } else {
                                    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                    for (int y = PARTS - 1; y >= 0; --y) mma_f16(d, af, pb[ht][0][y], pb[ht][1][y]);
#pragma unroll
                                    for (int i = 0; i < 4; ++i) t[i] += d[i];
                                }
                            }
                        }
                }
            };

            while (ok && k0 < k_stop) {
                fence_async();
                __syncwarp();  // every lane is done with the stage before this one, its writes there ordered in front of the copy that overwrites them
                if (k_next < k_stop) issue(st + S - 1 < S ? st + S - 1 : st - 1);
                const int end = stage_end(k0);
                ok = mbar_wait(bars + 8 * st, (parity >> st) & 1u);
                if (!ok) break;
                parity ^= 1u << st;
                unsigned char* src = q4_smem + warp * (S * STAGE) + st * STAGE;
                if (++st == S) st = 0;
                const int n = end - k0;
                // (a second chunk behind the stage's last key reads what an earlier stage left, as dead keys)
                const int stop = min(end, k_end);
#pragma unroll 1
                for (int c = 0; c < n; c += 16 * N) {
                    const int c0 = k0 + c;
                    if (biased_call || c0 < t_lo || c0 + 16 * N > stop) step(Bool<true>(), c0, stop, src + c * RB, src + SK * RB + c * Q4_FACTOR_BYTES);
                    else step(Bool<false>(), c0, stop, src + c * RB, src + SK * RB + c * Q4_FACTOR_BYTES);
                }
                k0 = end;
            }
            if (!ok) {
                // a copy never came: the error word is set.  Those behind it are waited for, with the same limit
                while (k0 < k_next) {
                    const int end = stage_end(k0);
                    if (++st == S) st = 0;
                    if (end < k_next) mbar_wait(bars + 8 * st, (parity >> st) & 1u);
                    k0 = end;
                }
            }
            __syncwarp();
            // this warp's result, into its ring.  A head's denominator lives in the eight lanes of its column.
            float* res = res0 + warp * RES_STEP;
#pragma unroll
            for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float lc = l[ht][c], zc = z[ht][c];
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) {
                        lc += __shfl_xor_sync(0xffffffffu, lc, x);
                        zc += __shfl_xor_sync(0xffffffffu, zc, x);
                    }
                    const int g = 8 * ht + 2 * t4 + c;
                    if (g < nG) {
                        float* po = res + g * HD + gq * (HD / 8);
                        auto low = [&](const float* t) { return t[c] + zc; };        // the low nibbles' dimensions, the high ones'
                        auto high = [&](const float* t) { return t[2 + c] + zc; };
#pragma unroll
                        for (int w = 0; w < VW; ++w) {
                            const float (*t)[4] = &o[ht][4 * w];
                            *reinterpret_cast<float4*>(po + 8 * w) = make_float4(low(t[0]), low(t[2]), high(t[0]), high(t[2]));
                            *reinterpret_cast<float4*>(po + 8 * w + 4) = make_float4(low(t[1]), low(t[3]), high(t[1]), high(t[3]));
                        }
                        if (gq == 0)
                            *reinterpret_cast<float2*>(res + 8 * HT * HD + 2 * g) =
                                limit[ht][c] == -INFINITY ? make_float2(-INFINITY, lc) : make_float2(from[ht][c], scale2(lc, s_from[ht][c] - from[ht][c] + LIFT));
                    }
                }
            }
        }
        __syncthreads();
        // joins: the weight of a part whose sums are relative to ml.x, relative to M (a part without a live key: 0; NaN stays)
        auto part_weight = [](float2 ml, float M) { return ml.x == -INFINITY && ml.y == 0.f ? 0.f : exp2f(ml.x - M); };
        auto part_sum = [](float2 ml, float M) { return ml.x == -INFINITY && ml.y == 0.f ? 0.f : scale2(ml.y, ml.x - M); };
        auto finish = [&](int g, const float* acc, float L, float M, int h_first, int at_row, int at_item) {
            const int h = h_first + g;
            // (the sink: one more term, of score 0 or its own; scores are in base 2.  One far above all scores: everything less 2^60)
            float ref = M - LIFT, full = L, lift = exp2f(LIFT);
            if (a.sink) {
                const float high = sink_term2(a.sink_val, h, ref + 60.f);
                if (high > 1.f) {
                    ref += 60.f;
                    lift *= 0x1p-60f;
                    full = fmaf(L, 0x1p-60f, high);
                } else {
                    full += sink_term2(a.sink_val, h, ref);
                }
            }
            const float inv = lift / full;
            T* dst = static_cast<T*>(a.out) + (static_cast<size_t>(at_row) * a.nh + h) * HD + lane * DL;
#pragma unroll
            for (int d = 0; d < DL; d += 2) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(dst + d) = make_float2(acc[d] * inv, acc[d + 1] * inv);
                else *reinterpret_cast<__nv_bfloat162*>(dst + d) = __floats2bfloat162_rn(acc[d] * inv, acc[d + 1] * inv);
            }
            if (WEIGH && lane == 0) {
                // (the denominator's own exponent goes to what scores are relative to, so that no weight above 2^-126 is flushed)
                const int k = min(max(static_cast<int>(__float_as_uint(full) >> 23 & 255u) - 127, -126), 126);
                *reinterpret_cast<float2*>(a.lse + 2 * (static_cast<size_t>(at_item) * a.nh + h)) =
                    make_float2(ref + static_cast<float>(k), 1.f / (full * pow2i(-k)));
            }
        };
        // what a (request, head) that a warp leads is, and the first of its heads that this warp takes: the block's heads go round the warps
        struct Led {
            int item, range, n, h0, n_heads, parts, lead;
        };
        auto led = [&](int at) {
            const Q4Unit& u = pl.units[at];
            const int lkv = n_sub == 1 ? u.vh : u.vh / n_sub, g = (u.vh - lkv * n_sub) * 8 * HT;
            return Led{u.item, u.range, u.wb - u.wa, lkv * G + g, min(G - g, 8 * HT), u.parts, u.lead};
        };
        int turn = warp;   // heads until this warp's next one
        for (unsigned leads = __ballot_sync(0xffffffffu, lane < W && pl.units[lane].active && pl.units[lane].wa == lane); leads; leads &= leads - 1) {
            const int at = __ffs(leads) - 1;
            const Led r = led(at);
            int g = turn;
            for (; g < r.n_heads; g += W) {
                const float* ml = res0 + 8 * HT * HD + 2 * g;
                const float2 mine = lane < r.n ? *reinterpret_cast<const float2*>(ml + (at + lane) * RES_STEP) : make_float2(-INFINITY, 0.f);
                const float M = warp_max(mine.x);
                const float w = part_weight(mine, M);
                const float L = warp_sum(part_sum(mine, M));
                float acc[DL];
#pragma unroll
                for (int d = 0; d < DL; ++d) acc[d] = 0.f;
#pragma unroll 4
                for (int j = 0; j < r.n; ++j) {
                    const float wj = __shfl_sync(0xffffffffu, w, j);
                    const float* src = res0 + (at + j) * RES_STEP + g * HD + lane * DL;
#pragma unroll
                    for (int d = 0; d < DL; d += 2) {
                        const float2 x = *reinterpret_cast<const float2*>(src + d);
                        acc[d] = fmaf(x.x, wj, acc[d]);
                        acc[d + 1] = fmaf(x.y, wj, acc[d + 1]);
                    }
                }
                if (r.parts == 1) {
                    finish(g, acc, L, M, r.h0, pl.row[r.item], r.item);
                } else {
                    const size_t place = static_cast<size_t>(pl.pref[r.item] + r.range) * a.nh + r.h0 + g;   // of the run's first range
                    float* dst = a.part_o + place * HD + lane * DL;
#pragma unroll
                    for (int d = 0; d < DL; d += 2) *reinterpret_cast<float2*>(dst + d) = make_float2(acc[d], acc[d + 1]);
                    if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * place) = make_float2(M, L);
                }
            }
            turn = g - r.n_heads;
        }
        fence_async();
        if (!__syncthreads_or(active && !whole)) continue;   // (the rings are free again behind this)
        // (request, head)s that several blocks have ranges of: the last block to bring its partial result joins them all
        if (lane == 0) {
            int last = 0;
            if (active && warp == wa && !whole) {
                __threadfence();   // (with the barrier in front: the whole block's results are out before the count is)
                int* counter = a.counters + static_cast<size_t>(item) * a.nh + vh;
                last = atomicAdd(counter, 1) == un.parts - 1;
                if (last) *counter = 0;
                __threadfence();
            }
            is_last[warp] = last;
        }
        __syncthreads();
        turn = warp;   // (all warps of the block take part)
        for (unsigned leads = __ballot_sync(0xffffffffu, lane < W && is_last[lane]); leads; leads &= leads - 1) {
            const Led r = led(__ffs(leads) - 1);
            const int parts = r.parts;
            // a part begins with the first range that its block has
            auto place = [&](int k, int g) {
                const int first_range = k == 0 ? 0 : r.lead + (k - 1) * W;
                return static_cast<size_t>(pl.pref[r.item] + first_range) * a.nh + r.h0 + g;
            };
            int g = turn;
            for (; g < r.n_heads; g += W) {
                constexpr int ROWS = 16;   // rows on their way together, with the first of the factors
                float M = -INFINITY, L = 0.f, acc[DL];
#pragma unroll
                for (int d = 0; d < DL; ++d) acc[d] = 0.f;
                for (int k0 = 0; k0 < parts; k0 += ROWS) {
                    const int n = min(ROWS, parts - k0);
                    float2 mine = make_float2(-INFINITY, 0.f);
                    if (lane < n) mine = __ldcg(reinterpret_cast<const float2*>(a.part_ml + 2 * place(k0 + lane, g)));
                    float2 x[ROWS][DL / 2];
#pragma unroll
                    for (int y = 0; y < ROWS; ++y)
#pragma unroll
                        for (int d = 0; d < DL; d += 2)
                            x[y][d / 2] = y < n ? __ldcg(reinterpret_cast<const float2*>(a.part_o + place(k0 + y, g) * HD + lane * DL + d))
                                                : make_float2(0.f, 0.f);
                    const float top = fmaxf(M, warp_max(mine.x)), corr = M == -INFINITY ? 0.f : exp2f(M - top);
                    const float w = part_weight(mine, top);
                    L = part_sum(make_float2(M, L), top) + warp_sum(part_sum(mine, top));
#pragma unroll
                    for (int d = 0; d < DL; ++d) acc[d] = k0 == 0 ? 0.f : acc[d] * corr;
                    M = top;
#pragma unroll
                    for (int y = 0; y < ROWS; ++y) {
                        if (y >= n) break;
                        const float wj = __shfl_sync(0xffffffffu, w, y);
#pragma unroll
                        for (int d = 0; d < DL; d += 2) {
                            acc[d] = fmaf(x[y][d / 2].x, wj, acc[d]);
                            acc[d + 1] = fmaf(x[y][d / 2].y, wj, acc[d + 1]);
                        }
                    }
                }
                finish(g, acc, L, M, r.h0, pl.row[r.item], r.item);
            }
            turn = g - r.n_heads;
        }
        __syncthreads();   // (is_last is written again in the next round)
    }
}

// weights[page][kvh][offset] += sum over the heads of the group of 2^(score - M) / denominator, for every key of the listed requests: scores,
// maxima and denominators as the kernel above left them.  WG_KEYS keys per thread, whose pages are looked up in front of the wait for that kernel and
// whose scores are on their way together (bound by such latencies: with one key per thread a call for 8 requests of 4,096 keys on 16 heads took 3 %
// more, with eight 2 %).
// A slot is added to once per request that lists it, so the sum does not depend on the order (an atomic: a request may be listed twice).
#define WG_THREADS 256
#define WG_KEYS 4
// Groups of one head: four keys in a row, whose scores are one load and whose weights one atomic of 16 bytes.  (8 requests of 4,096 keys
// 29.1 us, 64 162, of which 151 without weights; by the other kernel 1 and 8 more.  In groups of several heads four keys' scores are 4 G floats in a row, too wide a stride between a warp's lanes.)
__global__ void __launch_bounds__(WG_THREADS) q4_weigh_one_kernel(Q4Args a, float* __restrict__ weights) {
    const int item = blockIdx.z, h = blockIdx.y, P = a.page_tokens;
    const int seg = a.items[item];
    const int n = q4_position(a, seg) + 1;
    const int t = 4 * (blockIdx.x * WG_THREADS + threadIdx.x), i = t / P;
    float* at = t < n ? weights + (static_cast<size_t>(a.block_table[static_cast<size_t>(seg) * a.table_stride + i]) * a.nkv + h) * P + (t - i * P) : nullptr;
    pdl_entry();
    pdl_trigger();
    if (t >= n) return;
    const float4 s = *reinterpret_cast<const float4*>(a.scores + (static_cast<size_t>(item) * a.nkv + h) * a.table_stride * P + t);
    const float2 ml = reinterpret_cast<const float2*>(a.lse)[static_cast<size_t>(item) * a.nh + h];
    const float w[4] = {ex2(s.x - ml.x) * ml.y, ex2(s.y - ml.x) * ml.y, ex2(s.z - ml.x) * ml.y, ex2(s.w - ml.x) * ml.y};
    if (t + 4 <= n) {
        asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(w[0]), "f"(w[1]), "f"(w[2]), "f"(w[3]) : "memory");
    } else {
#pragma unroll
        for (int u = 0; u < 3; ++u)
            if (t + u < n) atomicAdd(at + u, w[u]);
    }
}
__global__ void __launch_bounds__(WG_THREADS) q4_weigh_kernel(Q4Args a, float* __restrict__ weights) {
    const int item = blockIdx.z, kvh = blockIdx.y, G = a.nh / a.nkv, P = a.page_tokens;
    const int seg = a.items[item];
    const int n = q4_position(a, seg) + 1;
    const int t0 = blockIdx.x * (WG_THREADS * WG_KEYS) + threadIdx.x;
    const int* table = a.block_table + static_cast<size_t>(seg) * a.table_stride;
    float* at[WG_KEYS];
#pragma unroll
    for (int u = 0; u < WG_KEYS; ++u) {
        const int t = t0 + u * WG_THREADS, i = t / P;
        at[u] = t < n ? weights + (static_cast<size_t>(table[i]) * a.nkv + kvh) * P + (t - i * P) : nullptr;
    }
    pdl_entry();
    pdl_trigger();
    if (t0 >= n) return;
    const float* score = a.scores + ((static_cast<size_t>(item) * a.nkv + kvh) * a.table_stride * P + t0) * G;
    const float2* ml = reinterpret_cast<const float2*>(a.lse) + static_cast<size_t>(item) * a.nh + static_cast<size_t>(kvh) * G;
    float sum[WG_KEYS];
#pragma unroll
    for (int u = 0; u < WG_KEYS; ++u) sum[u] = 0.f;
    for (int g = 0; g < G; ++g) {
        const float2 v = ml[g];
#pragma unroll
        for (int u = 0; u < WG_KEYS; ++u)
            if (at[u]) sum[u] = fmaf(ex2(score[static_cast<size_t>(u) * WG_THREADS * G + g] - v.x), v.y, sum[u]);
    }
#pragma unroll
    for (int u = 0; u < WG_KEYS; ++u)
        if (at[u]) atomicAdd(at[u], sum[u]);
}

template <typename T, int HD, int HT, int N, int W, int S, int SK, bool WEIGH>
static int q4_decode_launch(const Q4Args& a, int n_items, long long max_units, int cost_range, int cost_join, int cost_merge, int n_sm, int dev, cudaStream_t stream) {
    constexpr size_t smem = static_cast<size_t>(W) * S * 2 * SK * (HD / 2 + Q4_FACTOR_BYTES);
    static unsigned long long asked = 0;   // devices that know of the kernel's shared memory (asked again at worst)
    if (dev >= 64 || !(asked >> dev & 1)) {
        if (cudaFuncSetAttribute(attn_decode_q4_kernel<T, HD, HT, N, W, S, SK, WEIGH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(smem)) != cudaSuccess)
            return static_cast<int>(cudaGetLastError());
        if (dev < 64) asked |= 1ull << dev;
    }
    locus_launch(attn_decode_q4_kernel<T, HD, HT, N, W, S, SK, WEIGH>, n_sm, 32 * W, smem, stream, a, n_items, max_units, cost_range, cost_join, cost_merge);
    return locus_launch_status();
}

// What a call brings.  (One pointer to all of it: a foreign-function call pays for each of its arguments, a tenth of a microsecond from Python.)
// part_o holds max_units partial results of hd floats (at least n_items * nh; twice that with kept first tokens), part_ml two floats each, counters
// n_items * nh ints that are zero before and after the call.  weights (or null) [n_pages][nkv][P] float32, with scores of n_items * nh *
// table_stride * P floats and lse of 2 n_items * nh; then neither a window nor chunks.
struct Q4DecodeCall {
    const void *q, *pool;
    void* out;
    const int *seg_q0, *seg_ctx, *block_table, *items;
    float *part_o, *part_ml;
    int* counters;
    const float *sink_val, *slopes;
    float *weights, *scores, *lse;
    long long dt, table_stride, n_items, nh, nkv, hd, page_tokens, window, chunk, max_units, cost_range, cost_join, cost_merge, keep_first, sink;
    double scale;
};

extern "C" int locus_attn_decode_q4(const Q4DecodeCall* call, cudaStream_t stream) {
    const Q4DecodeCall& v = *call;
    if (v.n_items <= 0) return 0;
    if ((v.dt != LOCUS_DT_F32 && v.dt != LOCUS_DT_BF16) || v.nkv <= 0 || v.nh <= 0 || v.nh % v.nkv != 0 || !q4_head_ok(static_cast<int>(v.hd)) ||
        v.page_tokens <= 0 || v.page_tokens % 16 != 0 || v.n_items > Q4_MAX_ITEMS || v.table_stride <= 0 || v.table_stride > 0x7fffffff / v.page_tokens || v.nkv > 65535 || v.counters == nullptr ||
        !mask_ok(static_cast<int>(v.window), static_cast<int>(v.chunk), static_cast<int>(v.keep_first)) ||
        ((reinterpret_cast<uintptr_t>(v.q) | reinterpret_cast<uintptr_t>(v.pool) | reinterpret_cast<uintptr_t>(v.part_o)) & 15) != 0 ||
        (reinterpret_cast<uintptr_t>(v.part_ml) & 7) != 0 ||
        (reinterpret_cast<uintptr_t>(v.out) & (v.dt == LOCUS_DT_F32 ? 7 : 3)) != 0)   // (two elements a store)
        return LOCUS_ERR_UNSUPPORTED;
    const int keep_first = v.window == 0 ? 0 : static_cast<int>(v.keep_first);
    if (v.max_units < v.n_items * v.nh * (keep_first > 0 ? 2 : 1)) return LOCUS_ERR_UNSUPPORTED;
    if (v.weights && (((reinterpret_cast<uintptr_t>(v.weights) | reinterpret_cast<uintptr_t>(v.scores)) & 15) != 0 || v.scores == nullptr || v.lse == nullptr ||
                      (reinterpret_cast<uintptr_t>(v.lse) & 7) != 0 || v.window > 0 || v.chunk > 0))
        return LOCUS_ERR_UNSUPPORTED;
    int dev = 0, n_sm = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n_sm <= 0)
        return static_cast<int>(cudaGetLastError());
    Q4Args a;
    a.q = v.q; a.pool = static_cast<const uint8_t*>(v.pool); a.out = v.out;
    a.seg_q0 = v.seg_q0; a.seg_ctx = v.seg_ctx; a.block_table = v.block_table; a.table_stride = static_cast<int>(v.table_stride); a.items = v.items;
    a.nh = static_cast<int>(v.nh); a.nkv = static_cast<int>(v.nkv); a.page_tokens = static_cast<int>(v.page_tokens);
    a.window = static_cast<int>(v.window); a.chunk = static_cast<int>(v.chunk); a.scale = static_cast<float>(v.scale);
    a.keep_first = keep_first; a.sink = static_cast<int>(v.sink); a.sink_val = v.sink ? v.sink_val : nullptr; a.slopes = v.slopes;
    a.part_o = v.part_o; a.part_ml = v.part_ml; a.counters = v.counters; a.scores = v.scores; a.lse = v.lse; a.k1024 = 0x64006400u;
    const int n = static_cast<int>(v.n_items), cr = static_cast<int>(v.cost_range), cj = static_cast<int>(v.cost_join), cm = static_cast<int>(v.cost_merge);
    const bool wide = a.nh / a.nkv > 8;
#define Q4_GO(T_, HD_, HT_, N_, W_, S_, SK_)                                                                            \
    (v.weights ? q4_decode_launch<T_, HD_, HT_, N_, W_, S_, SK_, true>(a, n, v.max_units, cr, cj, cm, n_sm, dev, stream)      \
               : q4_decode_launch<T_, HD_, HT_, N_, W_, S_, SK_, false>(a, n, v.max_units, cr, cj, cm, n_sm, dev, stream))
    int code;
    if (v.dt == LOCUS_DT_F32) {
        code = v.hd == 64 ? Q4_GO(float, 64, 1, 1, 8, 3, 64) : v.hd == 128 ? Q4_GO(float, 128, 1, 1, 8, 2, 64) : Q4_GO(float, 256, 1, 1, 8, 2, 32);
    } else if (v.hd == 64) {
        code = wide ? Q4_GO(bf16, 64, 2, 1, 12, 3, 64) : Q4_GO(bf16, 64, 1, 2, 12, 3, 64);
    } else if (v.hd == 128) {
        code = wide ? Q4_GO(bf16, 128, 2, 1, 8, 2, 64) : Q4_GO(bf16, 128, 1, 2, 12, 2, 64);
    } else {
        code = Q4_GO(bf16, 256, 1, 1, 8, 2, 32);
    }
#undef Q4_GO
    if (code || !v.weights) return code;
    const dim3 grid(ceil_div(a.table_stride * a.page_tokens, WG_THREADS * WG_KEYS), a.nkv, n);
    if (a.nh == a.nkv) locus_launch(q4_weigh_one_kernel, grid, WG_THREADS, 0, stream, a, v.weights);
    else locus_launch(q4_weigh_kernel, grid, WG_THREADS, 0, stream, a, v.weights);
    return locus_launch_status();
}
