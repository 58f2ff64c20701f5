// Decode attention over a cache held in 4 bits (format: q4.cuh): one new token per request.
//
//   o_h = sum_t p_t v_t   p = softmax over the keys in sight of scale * q_h . k_t (a sink, a distance bias: as in attention.cu)
//
// with k_t and v_t read straight from their codes.  A key's row is mid + scale (code - 7.5) = z + scale (code - 7), z = mid - scale / 2, and codes
// less 7 are small whole numbers that bfloat16 holds exactly, so
//
//   q . k_t = scale_t (q . (code_t - 7)) + z_t sum(q)                      the product on the tensor cores, the rest per score in float32
//   o       = sum_t (p_t scale_t) (code_t - 7) + sum_t p_t z_t             the same for the values
//
// and nothing is rounded but the weights p_t scale_t, to bfloat16 (an operand of the tensor cores; the unrounded p_t enter the denominator
// and z's sum).  The 7 is taken off the codes rather than out of the sums: sums of codes of one sign would lose what cancels in them.
// A float32 model's q and weights go through the tensor cores as three bfloat16 parts each (bf16_parts.cuh), so nothing is rounded there.
//
// The work is cut as in attention_gqa.cu: a warp takes a range of keys of one (request, key/value head) for up to 16 query heads that share
// it, in the transposed form (16 keys in the M dimension of mma.sync m16n8k16, eight heads in N):
//   S^T [16 keys x 8 heads] = (C_k - 7) [16 x hd] . Q^T     a lane's words of a key row hold eight codes each: one shift, one mask-and-or and
//                             one subtraction give two neighbouring dimensions as bfloat16, as the A fragment wants them;
//   O^T [hd x 8 heads] += (C_v - 7)^T [hd x 16 keys] . P^T  the A fragment wants one dimension of two keys in a register: a byte permute joins
//                             the same byte of two keys' words, and its two nibbles are two dimensions (two row tiles' halves).
// A group of more heads is served by several warps (that each read its rows, from the L2 after the first).
// The running maximum of a head is raised only when a score exceeds it by more than 2^8: until then the weights are formed relative to the
// old one (at most 2^8, well inside float32), which saves the exchange between lanes and the correction of the sums in nearly every chunk.
//
// Memory: a warp's ring in shared memory is filled by bulk copies of up to 64 keys of one page: codes and factors of K, then of V.  (A whole
// page of 64 tokens is one run of bytes per plane.)  Every wait is bounded: when the limit runs out the warp records it in the module's error
// word, waits for its other copies with the same limit and leaves.
// Dead keys of an edge chunk (before a window, behind the range's end) have their factors replaced, as unwritten factors may be any bits; codes of
// any bits are numbers.
//
// With weights: the scores are written out as they are formed, and a second kernel (q4_weigh_kernel) adds every key's p_t, summed over the heads
// of its group, to a number per (slot, key/value head).  The softmax's denominator is known only behind the last range.
#include "attn_ranges.cuh"
#include "bf16_parts.cuh"
#include "distance.cuh"
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
    float* lse;               // with weights: [n_items * nh][2], a head's maximum and denominator
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
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t lds4(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
// N (1, 2, 4 or 8) words from shared memory
template <int N>
__device__ __forceinline__ void lds_words(uint32_t* v, uint32_t addr) {
    if constexpr (N == 1) v[0] = lds4(addr);
    else if constexpr (N == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr) : "memory");
    else {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
                         : "r"(addr + 4 * i)
                         : "memory");
    }
}

__device__ __forceinline__ void mma_bf16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of 16-bit elements held as mma fragments (two elements of a row per lane)
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// the low nibbles of a register's halves, less 7, as two bfloat16: 0x4300 | n is 128 + n, and 135 comes off exactly
__device__ __forceinline__ uint32_t codes2(uint32_t x) {
    const uint32_t y = (x & 0x000f000fu) | 0x43004300u;
    const uint32_t k = 0x43074307u;
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&y), *reinterpret_cast<const __nv_bfloat162*>(&k));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// a pair of values as PARTS pairs of bfloat16: one, rounded, or three that sum to them
template <int PARTS>
__device__ __forceinline__ void split2(float a, float b, uint32_t* out) {
    if constexpr (PARTS == 3) bf16_parts(a, b, out[0], out[1], out[2]);
    else out[0] = pack2(a, b);
}
__device__ __forceinline__ void load_pair(const bf16* p, uint32_t* out) { out[0] = *reinterpret_cast<const uint32_t*>(p); }
__device__ __forceinline__ void load_pair(const float* p, uint32_t* out) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    split2<3>(v.x, v.y, out);
}

// T: the model's type.  HD: head size.  HT: tiles of eight heads per warp.  W warps of a block, S stages of SK keys in flight per warp.
template <typename T, int HD, int HT, int W, int S, int SK, bool WEIGH>
__global__ void __launch_bounds__(32 * W, 1) attn_decode_q4_kernel(Q4Args a, int n_items, long long max_units, int cost_range, int cost_merge) {
    pdl_trigger();  // every block of this grid is resident from the start
    constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;
    constexpr int KW = HD / 32;      // words of a lane per key row (keys): HD / 4 dimensions
    constexpr int VW = HD / 64;      // words of a lane per value row: HD / 8 dimensions
    constexpr int MT = HD / 16;      // row tiles of O^T
    constexpr int RB = HD / 2;       // bytes of a row's codes
    constexpr uint32_t PLANE = SK * (RB + Q4_FACTOR_BYTES);   // K (or V) of a stage
    constexpr uint32_t STAGE = 2 * PLANE;
    extern __shared__ __align__(16) unsigned char q4_smem[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int gq = lane >> 2, t4 = lane & 3;   // row of the fragments, and the lane's place in its row
    // the key of a chunk's eight that row r of the fragments stands for, r with its low bit turned round in every other pair: rows of even
    // and of odd keys alternate both among the rows 2 t4 (values) and among neighbouring rows (keys), half the banks each
    const int kr0 = gq ^ ((gq >> 1) & 1);
    const int va_row = (2 * t4) ^ (t4 & 1), vb_row = (2 * t4 + 1) ^ (t4 & 1);
    const int P = a.page_tokens, G = a.nh / a.nkv;
    const int n_sub = (G + 8 * HT - 1) / (8 * HT), n_vh = a.nkv * n_sub;   // warps that serve a group, heads of a range

    __shared__ KeyRanges kr;
    __shared__ __align__(8) unsigned long long q4_bars[W * S];
    const uint32_t bars = smem_u32(q4_bars) + warp * (S * 8);  // this warp's barriers, one per stage
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < S; ++i) mbar_init(bars + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncwarp();
    uint32_t parity = 0;  // bit i: the phase of stage i's barrier that the next wait on it looks for
    const int n_warps = gridDim.x * W;
    const int len = plan_key_ranges(kr, a.items, a.seg_ctx, a.seg_q0, a.window, a.chunk, n_items, n_vh, max_units / a.nh * n_vh, n_warps,
                                    cost_range, cost_merge, a.keep_first);
    // (the cut read only the step's descriptors; q and the newest rows come from the kernel in front)
    pdl_entry();
    if (len == 0) return;
    const long long n_units = static_cast<long long>(kr.pref[n_items]) * n_vh;
    const float qscale = a.scale * 1.4426950408889634f;  // scores in base 2
    const size_t plane_step = static_cast<size_t>(a.nkv) * P * (RB + Q4_FACTOR_BYTES);
    const uint32_t ring = smem_u32(q4_smem) + warp * (S * STAGE);

    for (long long u = static_cast<long long>(blockIdx.x) * W + warp; u < n_units; u += n_warps) {
        const int vh = static_cast<int>(u % n_vh);
        const int kvh = vh / n_sub, g0 = (vh % n_sub) * 8 * HT;
        const int nG = min(G - g0, 8 * HT), h0 = kvh * G + g0;   // this warp's heads: h0 .. h0 + nG - 1
        const int r = static_cast<int>(u / n_vh);
        int item = 0;
        while (kr.pref[item + 1] <= r) ++item;
        const int seg = kr.seg[item], p = kr.pos[item], row = kr.row[item];
        // an item's first range may be its kept first tokens (see attention_gqa.cu)
        const int kept = kr.kept[item], keep = a.keep_first;
        const bool kept_range = kept > 0 && r == kr.pref[item];
        const int split = r - kr.pref[item] - (kept > 0);
        const int t_lo = kept_range ? 0 : first_key(a.window, a.chunk, p);
        const int k_begin = kept_range ? 0 : kr.first[item] + split * len;   // a multiple of 32
        const int k_end = kept_range ? kept : min(p + 1, k_begin + len);      // exclusive
        const int* table = a.block_table + static_cast<size_t>(seg) * a.table_stride;

        // Q as B fragments: head gq (and gq + 8 of the second tile), dimensions t4 HD / 4 + 8 w + 4 s + {0, 1} and + {2, 3}: words w, s = 0, 1
        uint32_t qb[HT][2 * KW][2][PARTS];
        float sq[HT][2];   // sum(q) of this lane's two heads per tile, times the scores' factor
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
            const int g = gq + 8 * ht;
            const T* q0 = static_cast<const T*>(a.q) + (static_cast<size_t>(row) * a.nh + h0 + (g < nG ? g : 0)) * HD + t4 * (HD / 4);
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            const uint32_t ones[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
#pragma unroll
            for (int i = 0; i < 2 * KW; ++i) {
                load_pair(q0 + 4 * i, qb[ht][i][0]);
                load_pair(q0 + 4 * i + 2, qb[ht][i][1]);
#pragma unroll
                for (int x = PARTS - 1; x >= 0; --x) {
                    if (g >= nG) qb[ht][i][0][x] = qb[ht][i][1][x] = 0u;
                    mma_bf16(sum, ones, qb[ht][i][0][x], qb[ht][i][1][x]);
                }
            }
            sq[ht][0] = sum[0] * qscale;
            sq[ht][1] = sum[1] * qscale;
        }
        // O^T: byte b of word w of a lane's value row is row tile 4 w + b: its low nibble's dimension in row gq, its high nibble's in row
        // gq + 8; columns are heads 2 t4 + {0, 1}.  l, z: this lane's share of the keys.
        float o[HT][MT][4], m[HT][2], l[HT][2], z[HT][2], slope[HT][2];
#pragma unroll
        for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
            for (int j = 0; j < MT; ++j) o[ht][j][0] = o[ht][j][1] = o[ht][j][2] = o[ht][j][3] = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int g = 8 * ht + 2 * t4 + c;
                m[ht][c] = -INFINITY;
                l[ht][c] = z[ht][c] = 0.f;
                slope[ht][c] = a.slopes && g < nG ? slope_log2(a.slopes, h0 + g) : 0.f;
            }
        }

        // keys k0 .. end - 1 of one page into a stage of the ring
        const int k_stop = (k_end + 15) & ~15;
        auto stage_end = [&](int k0) { return min(min((k0 / P + 1) * P, k0 + SK), k_stop); };
        auto issue = [&](int k0, int end, int st) {
            if (lane == 0) {
                const int n = end - k0, off = k0 % P;
                const uint8_t* src = a.pool + q4_place(table[k0 / P], 0, kvh, a.nkv, P, HD);
                const uint32_t dst = ring + st * STAGE, bar = bars + 8 * st;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // behind this warp's reads of the stage
                mbar_expect_tx(bar, 2 * n * (RB + Q4_FACTOR_BYTES));
                if (n == SK && P == SK) {
                    bulk_copy(dst, src, PLANE, bar);
                    bulk_copy(dst + PLANE, src + plane_step, PLANE, bar);
                } else {
                    const uint8_t* codes = src + static_cast<size_t>(off) * RB;
                    const uint8_t* factors = src + static_cast<size_t>(P) * RB + static_cast<size_t>(off) * Q4_FACTOR_BYTES;
                    bulk_copy(dst, codes, n * RB, bar);
                    bulk_copy(dst + SK * RB, factors, n * Q4_FACTOR_BYTES, bar);
                    bulk_copy(dst + PLANE, codes + plane_step, n * RB, bar);
                    bulk_copy(dst + PLANE + SK * RB, factors + plane_step, n * Q4_FACTOR_BYTES, bar);
                }
            }
        };
        // the first chunk that holds a live key (see attention_gqa.cu: every chunk from there on holds one, so its page is the request's)
        int k0 = keep > k_begin ? k_begin : max(k_begin, t_lo & ~15);
        int k_next = k0;   // first key that is not asked for yet
        bool ok = true;
#pragma unroll
        for (int c = 0; c < S - 1; ++c)
            if (k_next < k_stop) {
                const int e = stage_end(k_next);
                issue(k_next, e, c);
                k_next = e;
            }
        int st = 0;
        while (k0 < k_stop) {
            __syncwarp();  // every lane has read the stage before this one: its place may be overwritten
            if (k_next < k_stop) {
                int st_new = st + S - 1;
                if (st_new >= S) st_new -= S;
                const int e = stage_end(k_next);
                issue(k_next, e, st_new);
                k_next = e;
            }
            const int end = stage_end(k0);
            if (!mbar_wait(bars + 8 * st, (parity >> st) & 1u)) {
                ok = false;
                break;
            }
            parity ^= 1u << st;
            const uint32_t src = ring + st * STAGE;
            if (++st == S) st = 0;
            for (int c0 = k0; c0 < end; c0 += 16) {
                const uint32_t kbase = src + (c0 - k0) * RB, kfac = src + SK * RB + (c0 - k0) * Q4_FACTOR_BYTES;
                // keys c0 + kr0 and c0 + 8 + kr0: words, factors of the key's and of the value's row
                uint32_t k_lo[KW], k_hi[KW];
                lds_words<KW>(k_lo, kbase + kr0 * RB + t4 * (RB / 4));
                lds_words<KW>(k_hi, kbase + (kr0 + 8) * RB + t4 * (RB / 4));
                uint32_t kf[2], vf[2];
                kf[0] = lds4(kfac + 4 * kr0);
                kf[1] = lds4(kfac + 4 * (kr0 + 8));
                vf[0] = lds4(kfac + PLANE + 4 * kr0);
                vf[1] = lds4(kfac + PLANE + 4 * (kr0 + 8));
                uint32_t v_a[2][VW], v_b[2][VW];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    lds_words<VW>(v_a[x], kbase + PLANE + (8 * x + va_row) * RB + gq * (RB / 8));
                    lds_words<VW>(v_b[x], kbase + PLANE + (8 * x + vb_row) * RB + gq * (RB / 8));
                }
                float s[HT][2][4];
#pragma unroll
                for (int ht = 0; ht < HT; ++ht)
#pragma unroll
                    for (int x = 0; x < 2; ++x) s[ht][x][0] = s[ht][x][1] = s[ht][x][2] = s[ht][x][3] = 0.f;
#pragma unroll
                for (int w = 0; w < KW; ++w)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t af[4] = {codes2(k_lo[w] >> (8 * x)), codes2(k_hi[w] >> (8 * x)), codes2(k_lo[w] >> (8 * x + 4)),
                                                codes2(k_hi[w] >> (8 * x + 4))};
#pragma unroll
                        for (int ht = 0; ht < HT; ++ht)
#pragma unroll
                            for (int y = PARTS - 1; y >= 0; --y) mma_bf16(s[ht][x], af, qb[ht][2 * w + x][0][y], qb[ht][2 * w + x][1][y]);
                    }
                const int key0 = c0 + kr0, key1 = c0 + 8 + kr0;
                const bool edge = c0 < t_lo || c0 + 16 > k_end;
                bool live0 = true, live1 = true;
                if (edge) {
                    live0 = (key0 >= t_lo || key0 < keep) && key0 < k_end;
                    live1 = (key1 >= t_lo || key1 < keep) && key1 < k_end;
                    if (!live0) kf[0] = vf[0] = 0u;
                    if (!live1) kf[1] = vf[1] = 0u;
                }
                const float ks0 = q4_scale(kf[0]), ks1 = q4_scale(kf[1]), vs0 = q4_scale(vf[0]), vs1 = q4_scale(vf[1]);
                const float kz0 = fmaf(-0.5f, ks0, q4_mid(kf[0])), kz1 = fmaf(-0.5f, ks1, q4_mid(kf[1]));
                const float vz0 = fmaf(-0.5f, vs0, q4_mid(vf[0])), vz1 = fmaf(-0.5f, vs1, q4_mid(vf[1]));
                float sc[HT][4];
                bool raise = false;
#pragma unroll
                for (int ht = 0; ht < HT; ++ht) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c = i & 1;
                        float v = fmaf(s[ht][0][i] + s[ht][1][i], (i < 2 ? ks0 : ks1) * qscale, (i < 2 ? kz0 : kz1) * sq[ht][c]);
                        if (a.slopes) v = fmaf(slope[ht][c], static_cast<float>((i < 2 ? key0 : key1) - p), v);
                        if (edge && !(i < 2 ? live0 : live1)) v = -INFINITY;
                        sc[ht][i] = v;
                        raise |= v > m[ht][c] + 8.f;
                    }
                    if (WEIGH) {
                        float* at = a.scores + (static_cast<size_t>(item) * a.nkv + kvh) * a.table_stride * P * G + g0 + 8 * ht + 2 * t4;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (8 * ht + 2 * t4 + (i & 1) < nG && (i < 2 ? live0 : live1))
                                at[static_cast<size_t>(i < 2 ? key0 : key1) * G + (i & 1)] = sc[ht][i];
                    }
                }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int ht = 0; ht < HT; ++ht)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float n = fmaxf(sc[ht][c], sc[ht][2 + c]);
                            n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 4));
                            n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 8));
                            n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, 16));
                            n = fmaxf(n, m[ht][c]);
                            const float corr = m[ht][c] == -INFINITY ? 0.f : ex2(m[ht][c] - n);
                            m[ht][c] = n;
                            l[ht][c] *= corr;
                            z[ht][c] *= corr;
#pragma unroll
                            for (int j = 0; j < MT; ++j) {
                                o[ht][j][c] *= corr;
                                o[ht][j][2 + c] *= corr;
                            }
                        }
                }
                uint32_t pb[HT][2][PARTS];
#pragma unroll
                for (int ht = 0; ht < HT; ++ht) {
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float mu = m[ht][i & 1];
                        e[i] = ex2(sc[ht][i] - (mu == -INFINITY ? 0.f : mu));   // (no live key yet: all weights 0)
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        l[ht][c] += e[c] + e[2 + c];
                        z[ht][c] = fmaf(e[c], vz0, fmaf(e[2 + c], vz1, z[ht][c]));
                    }
                    // P^T as the B fragment: the transpose of the accumulator layout, 8 keys at a time
                    split2<PARTS>(e[0] * vs0, e[1] * vs0, pb[ht][0]);
                    split2<PARTS>(e[2] * vs1, e[3] * vs1, pb[ht][1]);
#pragma unroll
                    for (int y = 0; y < PARTS; ++y) {
                        pb[ht][0][y] = movmatrix_trans(pb[ht][0][y]);
                        pb[ht][1][y] = movmatrix_trans(pb[ht][1][y]);
                    }
                }
#pragma unroll
                for (int w = 0; w < VW; ++w)
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const uint32_t sel = b | ((4 + b) << 8);   // byte b of one key and of the other; the bytes between do not count
                        const uint32_t x0 = __byte_perm(v_a[0][w], v_b[0][w], sel), x1 = __byte_perm(v_a[1][w], v_b[1][w], sel);
                        const uint32_t af[4] = {codes2(x0), codes2(x0 >> 4), codes2(x1), codes2(x1 >> 4)};
#pragma unroll
                        for (int ht = 0; ht < HT; ++ht)
#pragma unroll
                            for (int y = PARTS - 1; y >= 0; --y) mma_bf16(o[ht][4 * w + b], af, pb[ht][0][y], pb[ht][1][y]);
                    }
            }
            k0 = end;
        }
        if (!ok) {
            // a copy never came: the error word is set.  Those still in flight are waited for, with the same limit, and the warp leaves
            while (k0 < k_next) {
                const int end = stage_end(k0);
                if (++st == S) st = 0;
                if (end < k_next) mbar_wait(bars + 8 * st, (parity >> st) & 1u);
                k0 = end;
            }
            return;
        }
        // partial results: head h of range r is place r * nh + h.  A head's denominator lives in the eight lanes of its column.
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
                    const size_t place = static_cast<size_t>(r) * a.nh + h0 + g;
                    float* po = a.part_o + place * HD + gq * (HD / 8);
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        const float (*t)[4] = &o[ht][4 * w];
                        *reinterpret_cast<float4*>(po + 8 * w) = make_float4(t[0][c] + zc, t[2][c] + zc, t[0][2 + c] + zc, t[2][2 + c] + zc);
                        *reinterpret_cast<float4*>(po + 8 * w + 4) = make_float4(t[1][c] + zc, t[3][c] + zc, t[1][2 + c] + zc, t[3][2 + c] + zc);
                    }
                    if (gq == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * place) = make_float2(m[ht][c], lc);
                }
            }
        }
        // the warp that finishes the last range of these heads merges their ranges, in ascending order
        __syncwarp();
        int last = 0;
        const int n_splits = kr.pref[item + 1] - kr.pref[item];
        if (lane == 0) {
            __threadfence();
            int* counter = a.counters + static_cast<size_t>(item) * a.nh + vh;
            last = atomicAdd(counter, 1) == n_splits - 1;
            if (last) *counter = 0;
        }
        last = __shfl_sync(0xffffffffu, last, 0);
        if (!last) continue;
        __threadfence();
        constexpr int GM = 4;          // heads at a time: a lane forms the weights of one range for all of them
        constexpr int DL = HD / 32;    // dimensions of a lane
        for (int g1 = 0; g1 < nG; g1 += GM) {
            const int n_g = min(GM, nG - g1);
            const size_t u0 = static_cast<size_t>(kr.pref[item]) * a.nh + h0 + g1;   // range s of head g1 + g: u0 + g + s nh
            float M[GM], L[GM], acc[GM][DL];
#pragma unroll
            for (int g = 0; g < GM; ++g) {
                M[g] = -INFINITY;
                L[g] = 0.f;
#pragma unroll
                for (int d = 0; d < DL; ++d) acc[g][d] = 0.f;
            }
            for (int x = lane; x < n_splits; x += 32)
#pragma unroll
                for (int g = 0; g < GM; ++g)
                    if (g < n_g) M[g] = fmaxf(M[g], __ldcg(a.part_ml + 2 * (u0 + g + static_cast<size_t>(x) * a.nh)));
#pragma unroll
            for (int g = 0; g < GM; ++g) M[g] = warp_max(M[g]);
            for (int s0 = 0; s0 < n_splits; s0 += 32) {
                float w[GM], lw[GM];   // of range s0 + lane
#pragma unroll
                for (int g = 0; g < GM; ++g) {
                    w[g] = lw[g] = 0.f;
                    if (g < n_g && s0 + lane < n_splits) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2*>(a.part_ml + 2 * (u0 + g + static_cast<size_t>(s0 + lane) * a.nh)));
                        w[g] = ml.x == -INFINITY && !(ml.y != ml.y) ? 0.f : exp2f(ml.x - M[g]);
                        lw[g] = ml.y;
                    }
                }
                const int n = min(32, n_splits - s0);
                const float* po = a.part_o + (u0 + static_cast<size_t>(s0) * a.nh) * HD + lane * DL;
                for (int j = 0; j < n; ++j) {
#pragma unroll
                    for (int g = 0; g < GM; ++g) {
                        if (g >= n_g) break;
                        const float wj = __shfl_sync(0xffffffffu, w[g], j);
                        L[g] = fmaf(__shfl_sync(0xffffffffu, lw[g], j), wj, L[g]);
                        const float* src = po + (static_cast<size_t>(j) * a.nh + g) * HD;
#pragma unroll
                        for (int d = 0; d < DL; d += 2) {
                            const float2 v = __ldcg(reinterpret_cast<const float2*>(src + d));
                            acc[g][d] = fmaf(v.x, wj, acc[g][d]);
                            acc[g][d + 1] = fmaf(v.y, wj, acc[g][d + 1]);
                        }
                    }
                }
            }
#pragma unroll
            for (int g = 0; g < GM; ++g) {
                if (g >= n_g) break;
                // (the sink: one more term of score 0; scores are in base 2 here)
                const int h = h0 + g1 + g;
                const float full = a.sink ? L[g] + sink_term2(a.sink_val, h, M[g]) : L[g];
                const float inv = 1.0f / full;
                T* dst = static_cast<T*>(a.out) + (static_cast<size_t>(row) * a.nh + h) * HD + lane * DL;
#pragma unroll
                for (int d = 0; d < DL; ++d) dst[d] = from_f<T>(acc[g][d] * inv);
                if (WEIGH && lane == 0)
                    *reinterpret_cast<float2*>(a.lse + 2 * (static_cast<size_t>(item) * a.nh + h)) = make_float2(M[g], inv);
            }
        }
    }
}

// weights[page][kvh][offset] += sum over the heads of the group of 2^(score - M) / denominator, for every key of the listed requests: scores,
// maxima and denominators as the kernel above left them.  One thread per key; a slot is added to once per request that lists it, so the sum
// does not depend on the order (an atomic: a request may be listed twice).
#define WG_THREADS 256
__global__ void __launch_bounds__(WG_THREADS) q4_weigh_kernel(Q4Args a, float* __restrict__ weights) {
    pdl_entry();
    pdl_trigger();
    const int item = blockIdx.z, kvh = blockIdx.y, G = a.nh / a.nkv, P = a.page_tokens;
    const int seg = a.items[item];
    const int n = min(a.seg_ctx[seg] + 1, a.table_stride * P);
    const int t = blockIdx.x * WG_THREADS + threadIdx.x;
    if (t >= n) return;
    const float* at = a.scores + ((static_cast<size_t>(item) * a.nkv + kvh) * a.table_stride * P + t) * G;
    const float2* ml = reinterpret_cast<const float2*>(a.lse) + static_cast<size_t>(item) * a.nh + static_cast<size_t>(kvh) * G;
    float sum = 0.f;
    for (int g = 0; g < G; ++g) {
        const float2 v = __ldg(ml + g);
        sum = fmaf(ex2(at[g] - v.x), v.y, sum);
    }
    const int page = a.block_table[static_cast<size_t>(seg) * a.table_stride + t / P];
    atomicAdd(weights + (static_cast<size_t>(page) * a.nkv + kvh) * P + t % P, sum);
}

template <typename T, int HD, int HT, int W, int S, int SK, bool WEIGH>
static int q4_decode_launch(const Q4Args& a, int n_items, long long max_units, int cost_range, int cost_merge, int n_sm, cudaStream_t stream) {
    constexpr size_t smem = static_cast<size_t>(W) * S * 2 * SK * (HD / 2 + Q4_FACTOR_BYTES);
    if (cudaFuncSetAttribute(attn_decode_q4_kernel<T, HD, HT, W, S, SK, WEIGH>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(smem)) != cudaSuccess)
        return static_cast<int>(cudaGetLastError());
    locus_launch(attn_decode_q4_kernel<T, HD, HT, W, S, SK, WEIGH>, n_sm, 32 * W, smem, stream, a, n_items, max_units, cost_range, cost_merge);
    return locus_launch_status();
}

// part_o holds max_units partial results of hd floats (at least n_items * nh; twice that with kept first tokens), part_ml two floats each, counters
// n_items * nh ints that are zero before and after the call.  weights (or null) [n_pages][nkv][P] float32, with scores of n_items * nh *
// table_stride * P floats and lse of 2 n_items * nh; then neither a window nor chunks.
extern "C" int locus_attn_decode_q4(const void* q, int dt, const void* pool, void* out, const int* seg_q0, const int* seg_ctx,
                                    const int* block_table, int table_stride, const int* items, int n_items, int nh, int nkv, int hd,
                                    int page_tokens, int window, int chunk, float scale, float* part_o, float* part_ml, int* counters,
                                    long long max_units, int cost_range, int cost_merge, int keep_first, int sink,
                                    const float* sink_val, const float* slopes, float* weights, float* scores, float* lse,
                                    cudaStream_t stream) {
    if (n_items <= 0) return 0;
    if ((dt != LOCUS_DT_F32 && dt != LOCUS_DT_BF16) || nkv <= 0 || nh <= 0 || nh % nkv != 0 || !q4_head_ok(hd) || page_tokens <= 0 ||
        page_tokens % 16 != 0 || n_items > DS_MAX_ITEMS || !mask_ok(window, chunk, keep_first) || counters == nullptr || table_stride <= 0 ||
        nkv > 65535 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(part_o)) & 15) != 0)
        return LOCUS_ERR_UNSUPPORTED;
    if (window == 0) keep_first = 0;
    if (max_units < static_cast<long long>(n_items) * nh * (keep_first > 0 ? 2 : 1)) return LOCUS_ERR_UNSUPPORTED;
    if (weights && (scores == nullptr || lse == nullptr || window > 0 || chunk > 0)) return LOCUS_ERR_UNSUPPORTED;
    int dev = 0, n_sm = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n_sm, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n_sm <= 0)
        return static_cast<int>(cudaGetLastError());
    Q4Args a;
    a.q = q; a.pool = static_cast<const uint8_t*>(pool); a.out = out;
    a.seg_q0 = seg_q0; a.seg_ctx = seg_ctx; a.block_table = block_table; a.table_stride = table_stride; a.items = items;
    a.nh = nh; a.nkv = nkv; a.page_tokens = page_tokens; a.window = window; a.chunk = chunk; a.scale = scale;
    a.keep_first = keep_first; a.sink = sink; a.sink_val = sink ? sink_val : nullptr; a.slopes = slopes;
    a.part_o = part_o; a.part_ml = part_ml; a.counters = counters; a.scores = scores; a.lse = lse;
    const bool wide = nh / nkv > 8;
#define Q4_GO(T_, HD_, HT_, W_, S_, SK_)                                                                                        \
    (weights ? q4_decode_launch<T_, HD_, HT_, W_, S_, SK_, true>(a, n_items, max_units, cost_range, cost_merge, n_sm, stream)   \
             : q4_decode_launch<T_, HD_, HT_, W_, S_, SK_, false>(a, n_items, max_units, cost_range, cost_merge, n_sm, stream))
    int code;
    if (dt == LOCUS_DT_F32) {
        code = hd == 64 ? Q4_GO(float, 64, 1, 8, 3, 64) : hd == 128 ? Q4_GO(float, 128, 1, 8, 2, 64) : Q4_GO(float, 256, 1, 8, 2, 32);
    } else if (hd == 64) {
        code = wide ? Q4_GO(bf16, 64, 2, 12, 3, 64) : Q4_GO(bf16, 64, 1, 12, 3, 64);
    } else if (hd == 128) {
        code = wide ? Q4_GO(bf16, 128, 2, 11, 2, 64) : Q4_GO(bf16, 128, 1, 11, 2, 64);
    } else {
        code = Q4_GO(bf16, 256, 1, 8, 2, 32);
    }
#undef Q4_GO
    if (code || !weights) return code;
    const dim3 grid(ceil_div(table_stride * page_tokens, WG_THREADS), nkv, n_items);
    locus_launch(q4_weigh_kernel, grid, WG_THREADS, 0, stream, a, weights);
    return locus_launch_status();
}
