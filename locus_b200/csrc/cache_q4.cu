// The cache held in 4 bits (format: q4.cuh), apart from the attention over single tokens (attention_q4.cu):
//
//   write    rotates q and k of a step's new tokens and writes q in the model's type, k and v as rows of 4 bits;
//   expand   lays the rows of some requests out in ordinary pages of the model's type, which the kernels of prompt portions read;
//   evict    chooses, per layer, request and key/value head, the keys that stay, and moves their rows.
//
// All three are bound by memory; what each reads and writes is at its kernel.
#include "q4.cuh"

__device__ __forceinline__ void load8(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const bf16* p, float* v) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store8(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16* p, const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// ---------------------------------------------------------------------------
// write: out of qkv [T, (nh + 2 nkv) hd] q rotated [T, nh, hd], and the rows of k (rotated) and v in the pages of slots[t].
// Rotated by pairs (i, i + rot / 2), or (2 i, 2 i + 1) (pairing 1), by the angle position * inv_freq[i], of which product and reduction
// to one turn are 64 bits (in 32 a position of 30,000 is off by up to 1/1000 of a radian, a hundredth of a cell, and codes near a border change).
// k and v are not rounded to the model's type on the way.
//
// A block takes one token: its angles' sines and cosines, once, then its heads by groups of hd / 8 lanes, eight values (one word of codes) a
// lane.  The pair's other half comes by a shuffle where halves lie a multiple of eight values apart, else through shared memory.
#define W_THREADS 256
template <typename T, int HD>
__global__ void __launch_bounds__(W_THREADS) q4_write_kernel(const T* __restrict__ qkv, const int* __restrict__ positions,
                                                            const float* __restrict__ inv_freq, T* __restrict__ q_out,
                                                            uint8_t* __restrict__ pool, const int* __restrict__ slots,
                                                            float* __restrict__ weights, int nh, int nkv, int rot, int pairing, int P,
                                                            int write_kv) {
    constexpr int GL = HD / 8;            // lanes of a row
    constexpr int ROWS = W_THREADS / GL;  // rows of the block at a time
    __shared__ float cs[HD / 2], sn[HD / 2];
    __shared__ __align__(16) float stage[W_THREADS * 8];
    const int t = blockIdx.x, tid = threadIdx.x;
    const int half = rot / 2;
    const double pos = positions[t];
    const int slot = slots ? slots[t] : 0;
    for (int i = tid; i < half; i += W_THREADS) {
        const double turns = pos * static_cast<double>(inv_freq[i]) * 0.15915494309189533577;
        sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &sn[i], &cs[i]);
    }
    __syncthreads();
    pdl_entry();
    pdl_trigger();
    const T* src = qkv + static_cast<size_t>(t) * (nh + 2 * nkv) * HD;
    const int page = slot / P, off = slot % P;
    const int n_rows = nh + (write_kv ? 2 * nkv : 0);
    const int g = tid / GL, l = tid % GL, d0 = 8 * l;
    const bool aligned = half % 8 == 0;
    const bool staged = pairing == 0 && !aligned && rot > 0;
    for (int r0 = 0; r0 < n_rows; r0 += ROWS) {
        const int r = r0 + g;
        const bool live = r < n_rows;
        float x[8];
        if (live) load8(src + static_cast<size_t>(r) * HD + d0, x);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.f;
        if (rot > 0) {   // (q and k; the rows of v take the shuffles with the others and keep their values)
            const bool turn = r < nh + nkv;
            if (pairing == 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int p = d0 / 2 + i;
                    if (turn && p < half) {
                        const float c = cs[p], s = sn[p], a = x[2 * i], b = x[2 * i + 1];
                        x[2 * i] = a * c - b * s;
                        x[2 * i + 1] = a * s + b * c;
                    }
                }
            } else if (!staged) {
                const bool low = d0 < half;
                const int lane = tid & 31, other = (lane - l) + (low ? l + half / 8 : l - half / 8);
                const bool in = turn && d0 < rot;
                const int p = low ? d0 : d0 - half;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = __shfl_sync(0xffffffffu, x[i], d0 < rot ? other : lane);
                    if (in) x[i] = low ? x[i] * cs[p + i] - y * sn[p + i] : y * sn[p + i] + x[i] * cs[p + i];
                }
            } else {
                float* mine = stage + static_cast<size_t>(g) * HD;
#pragma unroll
                for (int i = 0; i < 8; ++i) mine[d0 + i] = x[i];
                __syncwarp();
                if (turn)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int d = d0 + i;
                        if (d < half) x[i] = x[i] * cs[d] - mine[d + half] * sn[d];
                        else if (d < rot) x[i] = mine[d - half] * sn[d - half] + x[i] * cs[d - half];
                    }
                __syncwarp();
            }
        }
        // (all lanes of a warp take part: rows of q leave theirs unused)
        float lo = x[0], hi = x[0];
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo = fminf(lo, x[i]);
            hi = fmaxf(hi, x[i]);
            bad = bad || !(fabsf(x[i]) <= 3.402823466e38f);
        }
        if (bad) hi = INFINITY;
#pragma unroll
        for (int m = 1; m < GL; m <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, m));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, m));
        }
        if (!live) continue;
        if (r < nh) {
            store8(q_out + (static_cast<size_t>(t) * nh + r) * HD + d0, x);
            continue;
        }
        const int plane = (r - nh) / nkv, h = (r - nh) % nkv;
        const float scale = to_f(from_f<bf16>((0.5f * hi - 0.5f * lo) / 7.5f)), mid = to_f(from_f<bf16>(0.5f * lo + 0.5f * hi));
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = scale == 0.f ? 8.f : floorf((x[i] - mid) / scale) + 8.f;
            word |= static_cast<uint32_t>(fminf(fmaxf(c, 0.f), 15.f)) << q4_shift(i);
        }
        uint8_t* at = pool + q4_place(page, plane, h, nkv, P, HD);
        reinterpret_cast<uint32_t*>(at + static_cast<size_t>(off) * (HD / 2))[l] = word;
        if (l == 0) {
            reinterpret_cast<uint32_t*>(at + static_cast<size_t>(P) * (HD / 2))[off] =
                hi == INFINITY ? 0x7fff7fffu : q4_factors(scale, mid);
            if (weights && plane == 0) weights[(static_cast<size_t>(page) * nkv + h) * P + off] = 0.f;
        }
    }
}

template <typename T>
static int write_launch(const void* qkv, const int* positions, const float* inv_freq, void* q_out, uint8_t* pool, const int* slots,
                        float* weights, int n, int nh, int nkv, int hd, int rot, int pairing, int P, int write_kv, cudaStream_t stream) {
#define Q4_WRITE(HD_)                                                                                                               \
    locus_launch(q4_write_kernel<T, HD_>, n, W_THREADS, 0, stream, static_cast<const T*>(qkv), positions, inv_freq,                \
                 static_cast<T*>(q_out), pool, slots, weights, nh, nkv, rot, pairing, P, write_kv)
    if (hd == 64) Q4_WRITE(64);
    else if (hd == 128) Q4_WRITE(128);
    else Q4_WRITE(256);
#undef Q4_WRITE
    return locus_launch_status();
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// What a call brings, behind one pointer (see attention_q4.cu).  inv_freq null: no rotation (rot is then taken as 0).  weights (or null)
// [n_pages][nkv][P] float32: 0 for the slots that are written.
struct Q4WriteCall {
    const void* qkv;
    const int* positions;
    const float* inv_freq;
    void *q_out, *pool;
    const int* slots;
    float* weights;
    long long dt, T, nh, nkv, hd, rot, pairing, P, write_kv;
};
extern "C" int locus_rope_kv_write_q4(const Q4WriteCall* call, cudaStream_t stream) {
    const Q4WriteCall& v = *call;
    if (v.T <= 0) return 0;
    const int hd = static_cast<int>(v.hd), rot = v.inv_freq == nullptr ? 0 : static_cast<int>(v.rot), P = static_cast<int>(v.P);
    if (!q4_head_ok(hd) || v.nh <= 0 || v.nkv <= 0 || P <= 0 || P % 16 != 0 || rot < 0 || rot > hd || (rot & 1) || (v.pairing != 0 && v.pairing != 1) ||
        !aligned16(v.qkv) || !aligned16(v.q_out) || !aligned16(v.pool) || (v.write_kv && v.slots == nullptr))
        return LOCUS_ERR_UNSUPPORTED;
    auto go = [&](auto launch) {
        return launch(v.qkv, v.positions, v.inv_freq, v.q_out, static_cast<uint8_t*>(v.pool), v.slots, v.weights, static_cast<int>(v.T),
                      static_cast<int>(v.nh), static_cast<int>(v.nkv), hd, rot, static_cast<int>(v.pairing), P, static_cast<int>(v.write_kv), stream);
    };
    if (v.dt == LOCUS_DT_F32) return go(write_launch<float>);
    if (v.dt == LOCUS_DT_BF16) return go(write_launch<bf16>);
    return LOCUS_ERR_UNSUPPORTED;
}

// ---------------------------------------------------------------------------
// expand: the rows of positions 0 .. seg_ctx + seg_qn - 1 of the listed segments into ordinary pages [n_pages][2][nkv][P][hd] of the same
// page ids, in the model's type (float32: as they are; bfloat16: one rounding, the tensor cores' operand).  Rows behind a request's last
// token and pages that went back (-1) stay as they were.
// One block per (page of the request, plane, head): P rows, a lane takes words of eight values.
#define E_THREADS 256
template <typename T, int HD>
__global__ void __launch_bounds__(E_THREADS) q4_expand_kernel(const uint8_t* __restrict__ pool, T* __restrict__ out,
                                                              const int* __restrict__ segs, const int* __restrict__ seg_ctx,
                                                              const int* __restrict__ seg_qn, const int* __restrict__ block_table,
                                                              int table_stride, int nkv, int P) {
    constexpr int WR = HD / 8;   // words of a row
    pdl_entry();
    pdl_trigger();
    const int seg = segs[blockIdx.z];
    const int n = seg_ctx[seg] + seg_qn[seg];
    const int first = blockIdx.y * P;
    if (first >= n) return;
    const int page = block_table[static_cast<size_t>(seg) * table_stride + blockIdx.y];
    if (page < 0) return;
    const int plane = blockIdx.x / nkv, h = blockIdx.x % nkv;
    const uint8_t* src = pool + q4_place(page, plane, h, nkv, P, HD);
    T* dst = out + ((static_cast<size_t>(page) * 2 + plane) * nkv + h) * static_cast<size_t>(P) * HD;
    const int words = min(P, n - first) * WR;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(src);
    const uint32_t* factors = reinterpret_cast<const uint32_t*>(src + static_cast<size_t>(P) * (HD / 2));
#pragma unroll 4
    for (int i = threadIdx.x; i < words; i += E_THREADS) {
        const uint32_t w = codes[i], f = factors[i / WR];
        const float scale = q4_scale(f), mid = q4_mid(f);
        float v[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) v[d] = fmaf(scale, static_cast<float>((w >> q4_shift(d)) & 15u) - 7.5f, mid);
        store8(dst + static_cast<size_t>(i) * 8, v);
    }
}

// max_keys: at least the tokens of the longest of these segments.
struct Q4ExpandCall {
    const void* pool;
    void* out;
    const int *segs, *seg_ctx, *seg_qn, *block_table;
    long long dt, n_segs, table_stride, nkv, hd, P, max_keys;
};
extern "C" int locus_expand_q4(const Q4ExpandCall* call, cudaStream_t stream) {
    const Q4ExpandCall& v = *call;
    if (v.n_segs <= 0 || v.max_keys <= 0) return 0;
    const int hd = static_cast<int>(v.hd), P = static_cast<int>(v.P), nkv = static_cast<int>(v.nkv), table_stride = static_cast<int>(v.table_stride);
    const long long pages = min(v.table_stride, (v.max_keys + max(P, 1) - 1) / max(P, 1));
    if (!q4_head_ok(hd) || nkv <= 0 || P <= 0 || P % 16 != 0 || !aligned16(v.pool) || !aligned16(v.out) || pages > 65535 || v.n_segs > 65535)
        return LOCUS_ERR_UNSUPPORTED;
    if (pages <= 0) return 0;
    const dim3 grid(2 * nkv, static_cast<unsigned>(pages), static_cast<unsigned>(v.n_segs));
    const uint8_t* p8 = static_cast<const uint8_t*>(v.pool);
#define Q4_EXPAND(T_, HD_)                                                                                                          \
    locus_launch(q4_expand_kernel<T_, HD_>, grid, E_THREADS, 0, stream, p8, static_cast<T_*>(v.out), v.segs, v.seg_ctx, v.seg_qn,   \
                 v.block_table, table_stride, nkv, P)
#define Q4_EXPAND_T(T_)                                                                                                             \
    do {                                                                                                                            \
        if (hd == 64) Q4_EXPAND(T_, 64);                                                                                            \
        else if (hd == 128) Q4_EXPAND(T_, 128);                                                                                     \
        else Q4_EXPAND(T_, 256);                                                                                                    \
    } while (0)
    if (v.dt == LOCUS_DT_F32) Q4_EXPAND_T(float);
    else if (v.dt == LOCUS_DT_BF16) Q4_EXPAND_T(bf16);
    else return LOCUS_ERR_UNSUPPORTED;
#undef Q4_EXPAND_T
#undef Q4_EXPAND
    return locus_launch_status();
}

// ---------------------------------------------------------------------------
// evict, first half: which keys stay.  Of a request's n tokens its first `first`, its last `recent` and, of those between, the heaviest,
// `keep` in all; of equal weights the earlier key counts as the heavier one, and a weight that is not a number as lighter than all others.
// kept [layers][n_items][nkv][keep]: their indices, ascending; -1 behind a request of fewer than `keep` tokens, all of which stay.
//
// One block per (layer, request, head) finds the weight of the last key that stays digit by digit: the weights as unsigned numbers of the same
// order, three digits of 11, 11 and 10 bits, a histogram in shared memory of those that agree in the digits before.  Then every warp takes
// a run of keys, counts those that stay, and behind a sum over the warps writes their indices in order.  The keys are read once into shared
// memory where they fit (SK_MAX), else from memory (the L2) in every pass.
#define S_THREADS 1024
#define S_WARPS (S_THREADS / 32)
#define SK_MAX 49152      // weights in shared memory (192 KB)
#define S_BINS 2048

// an unsigned number of the weight's order
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);   // (-0 and 0 are one weight)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(S_THREADS) q4_select_kernel(const float* __restrict__ weights, const int* __restrict__ block_table,
                                                              int table_stride, const int* __restrict__ n_tokens, int n_items, int nkv,
                                                              int P, size_t layer_slots, int keep, int first, int recent,
                                                              int room, int* __restrict__ kept) {
    extern __shared__ uint32_t s_keys[];
    __shared__ int hist[S_BINS];
    __shared__ int warp_sum_[S_WARPS], warp_tie[S_WARPS];
    __shared__ int chosen_bin, above_bin;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_entry();
    pdl_trigger();
    const int h = blockIdx.x, item = blockIdx.y, layer = blockIdx.z;
    const int n = min(n_tokens[item], table_stride * P);
    int* dst = kept + ((static_cast<size_t>(layer) * n_items + item) * nkv + h) * keep;
    if (n <= keep) {
        for (int j = tid; j < keep; j += S_THREADS) dst[j] = j < n ? j : -1;
        return;
    }
    const float* w = weights + static_cast<size_t>(layer) * layer_slots;
    const int* table = block_table + static_cast<size_t>(item) * table_stride;
    const int lo = first, hi = n - recent;       // the keys between, of which `want` stay
    const int want = keep - first - recent;
    auto read = [&](int t) {
        const int page = table[t / P];
        return page < 0 ? 0u : ordered(w[(static_cast<size_t>(page) * nkv + h) * P + t % P]);
    };
    const bool in_smem = hi - lo <= room;
    if (in_smem && want > 0) {
        for (int t = lo + tid; t < hi; t += S_THREADS) s_keys[t - lo] = read(t);
    }
    auto key = [&](int t) { return in_smem ? s_keys[t - lo] : read(t); };
    uint32_t prefix = 0;   // the digits found so far, in place
    int left = want;       // keys of those digits that still stay
    if (want > 0) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
            for (int i = tid; i < S_BINS; i += S_THREADS) hist[i] = 0;
            __syncthreads();
            for (int t = lo + tid; t < hi; t += S_THREADS) {
                const uint32_t u = key(t);
                if (pass == 0 || (u >> (shift + bits)) == (prefix >> (shift + bits))) atomicAdd(&hist[(u >> shift) & ((1u << bits) - 1)], 1);
            }
            __syncthreads();
            // keys in higher bins, from the top: thread i has bins 2047 - 2 i and 2046 - 2 i
            const int b0 = hist[S_BINS - 1 - 2 * tid], b1 = hist[S_BINS - 2 - 2 * tid];
            int run = b0 + b1;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, run, m);
                if (lane >= m) run += v;
            }
            if (lane == 31) warp_sum_[warp] = run;
            __syncthreads();
            if (warp == 0) {
                int v = warp_sum_[lane];
#pragma unroll
                for (int m = 1; m < 32; m <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, v, m);
                    if (lane >= m) v += o;
                }
                warp_sum_[lane] = v;
            }
            __syncthreads();
            const int before = (warp ? warp_sum_[warp - 1] : 0) + run - b0 - b1;   // keys above this thread's bins
            if (before < left && before + b0 >= left) {
                chosen_bin = S_BINS - 1 - 2 * tid;
                above_bin = before;
            } else if (before + b0 < left && before + b0 + b1 >= left) {
                chosen_bin = S_BINS - 2 - 2 * tid;
                above_bin = before + b0;
            }
            __syncthreads();
            prefix |= static_cast<uint32_t>(chosen_bin) << shift;
            left -= above_bin;
            __syncthreads();
        }
    }
    // keys above `prefix` stay, and the first `left` of those equal to it
    const int per = ((n + S_WARPS - 1) / S_WARPS + 31) & ~31;
    const int a = min(n, warp * per), b = min(n, a + per);
    auto look = [&](int t, bool& stays, bool& tie) {
        stays = t < b && (t < lo || t >= hi);
        tie = false;
        if (t < b && !stays && want > 0) {
            const uint32_t u = key(t);
            stays = u > prefix;
            tie = u == prefix;
        }
    };
    int n_stay = 0, n_tie = 0;
    for (int t0 = a; t0 < b; t0 += 32) {
        bool s, e;
        look(t0 + lane, s, e);
        n_stay += __popc(__ballot_sync(0xffffffffu, s));
        n_tie += __popc(__ballot_sync(0xffffffffu, e));
    }
    if (lane == 0) {
        warp_sum_[warp] = n_stay;
        warp_tie[warp] = n_tie;
    }
    __syncthreads();
    // ties taken and keys written by the warps in front
    int ties = 0, at = 0;
    for (int v = 0; v < warp; ++v) {
        at += warp_sum_[v] + max(0, min(warp_tie[v], left - ties));
        ties += warp_tie[v];
    }
    const uint32_t below = (1u << lane) - 1;
    for (int t0 = a; t0 < b; t0 += 32) {
        bool s, e;
        look(t0 + lane, s, e);
        const uint32_t tie_mask = __ballot_sync(0xffffffffu, e);
        const bool in = s || (e && ties + __popc(tie_mask & below) < left);
        const uint32_t in_mask = __ballot_sync(0xffffffffu, in);
        if (in) dst[at + __popc(in_mask & below)] = t0 + lane;
        at += __popc(in_mask);
        ties += __popc(tie_mask);
    }
}

// evict, second half: key kept[j] of a request's pages becomes key j of the pages of dst_table, rows, factors and weight.
// In place (dst_table the request's own table) a row's old place may be another row's new one, but never that of a row in front of it
// (kept[j] >= j): a block takes (layer, request, head, plane) and walks its rows from the front, a tile at a time, and reads a tile before it
// writes it.  Into other pages the order is free, and several blocks share the rows.
#define M_THREADS 256
#define M_UNROLL 4       // 16-byte pieces of a thread in flight per tile, two tiles

template <int HD>
__global__ void __launch_bounds__(M_THREADS) q4_move_kernel(uint8_t* pool, float* weights, const int* __restrict__ block_table,
                                                            int table_stride, const int* __restrict__ dst_table, int dst_stride,
                                                            const int* __restrict__ n_tokens, int n_items, int nkv, int P,
                                                            size_t layer_bytes, size_t layer_slots, int keep, int n_parts,
                                                            const int* __restrict__ kept) {
    constexpr int PR = HD / 32;                           // pieces of a row
    constexpr int TILE = M_THREADS * M_UNROLL / PR;       // rows of a tile
    constexpr int FU = (TILE + M_THREADS - 1) / M_THREADS;
    pdl_entry();
    pdl_trigger();
    const int tid = threadIdx.x;
    const int part = blockIdx.x % n_parts, hp = blockIdx.x / n_parts;
    const int plane = hp & 1, h = hp >> 1, item = blockIdx.y, layer = blockIdx.z;
    const int n = min(min(keep, n_tokens[item]), min(table_stride, dst_stride) * P);
    const int* idx = kept + ((static_cast<size_t>(layer) * n_items + item) * nkv + h) * keep;
    const int* table = block_table + static_cast<size_t>(item) * table_stride;
    const int* to = dst_table + static_cast<size_t>(item) * dst_stride;
    uint8_t* base = pool + static_cast<size_t>(layer) * layer_bytes;
    float* w = weights + static_cast<size_t>(layer) * layer_slots;
    auto place = [&](int page) { return base + q4_place(page, plane, h, nkv, P, HD); };

    uint4 piece[M_UNROLL];
    uint32_t fac[FU];
    float wt[FU];
    bool has[M_UNROLL], fhas[FU];
    for (int j0 = part * TILE; j0 < n; j0 += n_parts * TILE) {
#pragma unroll
        for (int u = 0; u < M_UNROLL; ++u) {
            const int e = u * M_THREADS + tid, j = j0 + e / PR;
            has[u] = false;
            if (j < n) {
                const int t = idx[j], page = table[t / P];
                has[u] = page >= 0;
                if (has[u]) piece[u] = *reinterpret_cast<const uint4*>(place(page) + static_cast<size_t>(t % P) * (HD / 2) + (e % PR) * 16);
            }
        }
#pragma unroll
        for (int u = 0; u < FU; ++u) {
            const int e = u * M_THREADS + tid, j = j0 + e;
            fhas[u] = false;
            if (e < TILE && j < n) {
                const int t = idx[j], page = table[t / P];
                fhas[u] = page >= 0;
                if (fhas[u]) {
                    fac[u] = reinterpret_cast<const uint32_t*>(place(page) + static_cast<size_t>(P) * (HD / 2))[t % P];
                    if (plane == 0) wt[u] = w[(static_cast<size_t>(page) * nkv + h) * P + t % P];
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < M_UNROLL; ++u) {
            const int e = u * M_THREADS + tid, j = j0 + e / PR;
            if (has[u]) {
                const int page = to[j / P];
                if (page >= 0) *reinterpret_cast<uint4*>(place(page) + static_cast<size_t>(j % P) * (HD / 2) + (e % PR) * 16) = piece[u];
            }
        }
#pragma unroll
        for (int u = 0; u < FU; ++u) {
            const int j = j0 + u * M_THREADS + tid;
            if (fhas[u]) {
                const int page = to[j / P];
                if (page >= 0) {
                    reinterpret_cast<uint32_t*>(place(page) + static_cast<size_t>(P) * (HD / 2))[j % P] = fac[u];
                    if (plane == 0) w[(static_cast<size_t>(page) * nkv + h) * P + j % P] = wt[u];
                }
            }
        }
    }
}

// max_tokens: at least the tokens of the longest request (its weights' place in shared memory is sized by it).
struct Q4EvictCall {
    void* pool;
    float* weights;
    const int *block_table, *dst_table, *n_tokens;
    int* kept;
    long long table_stride, dst_stride, n_items, n_layers, layer_pages, nkv, hd, P, keep, first, recent, max_tokens;
};
extern "C" int locus_evict_q4(const Q4EvictCall* call, cudaStream_t stream) {
    const Q4EvictCall& v = *call;
    if (v.n_items <= 0 || v.n_layers <= 0) return 0;
    const int hd = static_cast<int>(v.hd), P = static_cast<int>(v.P), nkv = static_cast<int>(v.nkv), keep = static_cast<int>(v.keep);
    const int first = static_cast<int>(v.first), recent = static_cast<int>(v.recent), max_tokens = static_cast<int>(v.max_tokens);
    const int n_items = static_cast<int>(v.n_items), table_stride = static_cast<int>(v.table_stride), dst_stride = static_cast<int>(v.dst_stride);
    if (!q4_head_ok(hd) || nkv <= 0 || P <= 0 || P % 16 != 0 || keep <= 0 || first < 0 || recent < 0 || first > keep - recent ||
        n_items > 65535 || v.n_layers > 65535 || !aligned16(v.pool) || max_tokens <= 0)
        return LOCUS_ERR_UNSUPPORTED;
    const size_t slots = static_cast<size_t>(v.layer_pages) * nkv * P, bytes = slots * 2 * q4_row_bytes(hd);
    const int between = max(0, max_tokens - first - recent);
    const dim3 grid(nkv, n_items, static_cast<unsigned>(v.n_layers));
    const int room = between <= SK_MAX ? between : 0;   // (longer ones are read from memory in every pass)
    static unsigned long long asked = 0;   // devices that know of the kernel's shared memory (asked again at worst)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return static_cast<int>(cudaGetLastError());
    if (dev >= 64 || !(asked >> dev & 1)) {
        if (cudaFuncSetAttribute(q4_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SK_MAX * 4) != cudaSuccess)
            return static_cast<int>(cudaGetLastError());
        if (dev < 64) asked |= 1ull << dev;
    }
    locus_launch(q4_select_kernel, grid, S_THREADS, static_cast<size_t>(room) * 4, stream, v.weights, v.block_table, table_stride, v.n_tokens, n_items,
                 nkv, P, slots, keep, first, recent, room, v.kept);
    const int code = locus_launch_status();
    if (code) return code;
    const int tile = M_THREADS * M_UNROLL / (hd / 32);
    const int n_parts = v.dst_table == v.block_table ? 1 : max(1, min(ceil_div(min(keep, max_tokens), tile), 16));
    const dim3 mgrid(2 * nkv * n_parts, n_items, static_cast<unsigned>(v.n_layers));
#define Q4_MOVE(HD_)                                                                                                                        \
    locus_launch(q4_move_kernel<HD_>, mgrid, M_THREADS, 0, stream, static_cast<uint8_t*>(v.pool), v.weights, v.block_table, table_stride,   \
                 v.dst_table, dst_stride, v.n_tokens, n_items, nkv, P, bytes, slots, keep, n_parts, v.kept)
    if (hd == 64) Q4_MOVE(64);
    else if (hd == 128) Q4_MOVE(128);
    else Q4_MOVE(256);
#undef Q4_MOVE
    return locus_launch_status();
}
