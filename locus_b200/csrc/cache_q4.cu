// The cache held in 4 bits (format: q4.cuh), apart from the attention over single tokens (attention_q4.cu):
//
//   write    rotates q and k of a step's new tokens and writes q in the model's type, k and v as rows of 4 bits;
//   expand   lays the rows of some requests out in ordinary pages of the model's type, which the kernels of prompt portions read;
//   evict    chooses, per layer, request and key/value head, the keys that stay, and moves their rows.
//
// All three are bound by memory; what each reads and writes is at its kernel.
#include "q4.cuh"

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
// A block takes one token: its angles' sines and cosines, once, then its heads by groups of hd / 16 lanes, sixteen values (two words of codes) a
// lane: eight of either half of the head where the whole head is rotated by halves (SPLIT: a pair's two values lie in one lane), else sixteen in a row
// (a pair's other half comes by a shuffle where halves lie a multiple of sixteen values apart, else through shared memory).  The rows of the first
// W_AHEAD rounds are asked for in front of the angles.
// Bound by instructions (8,192 tokens of 16 + 16 heads of 128, of which the bytes alone take 26 us: 93 us with divisions and all rows through the
// quantising, 64 with a product and a remainder in their place, 54 with eight values a lane and a row's factors formed by twice as many, now 37.)
#define W_THREADS 128
#define W_AHEAD 1
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
    float d;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// a row's factors, of the sixteen values of each of its GL lanes (NaN or an infinity among them: `bad`)
template <int GL>
__device__ __forceinline__ void q4_row_factors(const float* x, float& scale, float& mid, bool& bad) {
    float lo = min_nan(x[0], x[1]), hi = max_nan(x[0], x[1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) {
        lo = min3_nan(lo, x[i], x[i + 1]);
        hi = max3_nan(hi, x[i], x[i + 1]);
    }
#pragma unroll
    for (int m = 1; m < GL; m <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
    bad = !(hi <= 3.402823466e38f && lo >= -3.402823466e38f);
    scale = to_f(from_f<bf16>((0.5f * hi - 0.5f * lo) / 7.5f));
    mid = to_f(from_f<bf16>(0.5f * lo + 0.5f * hi));
}
// The word of eight values.  floor((x - mid) / scale): the quotient by the reciprocal, raised by 2^-22 of itself, which is more than its rounding took
// off (so that a whole quotient counts as one; two bfloat16 and their difference never give a quotient that close below a whole number), plus
// 3 2^22, rounded down; a sum with a bound and one at zero clamps it.
__device__ __forceinline__ uint32_t q4_word(const float* x, float scale, float mid, float inv) {
    uint32_t word = 0;
    if (scale >= 1e-30f) {
        const float more = inv * 2.384185791e-07f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = x[i] - mid;
            const int cell = __float_as_int(__fadd_rd(fmaf(fabsf(d), more, d * inv), 12582912.f));
            word += static_cast<uint32_t>(__viaddmin_s32_relu(cell, 8 - 0x4b400000, 15)) << q4_shift(i);
        }
    } else {   // (no reciprocal to rely on; a row of equal values; not a number)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float c = scale > 0.f ? floorf((x[i] - mid) / scale) : 0.f;
            word += static_cast<uint32_t>(fminf(fmaxf(c, -8.f), 7.f) + 8.f) << q4_shift(i);
        }
    }
    return word;
}

template <typename T, int HD, bool SPLIT>
__global__ void __launch_bounds__(W_THREADS, 8) q4_write_kernel(const T* __restrict__ qkv, const int* __restrict__ positions,
                                                            const float* __restrict__ inv_freq, T* __restrict__ q_out,
                                                            uint8_t* __restrict__ pool, const int* __restrict__ slots,
                                                            float* __restrict__ weights, int nh, int nkv, int rot, int pairing, int P,
                                                            int write_kv) {
    constexpr int GL = HD / 16;           // lanes of a row
    constexpr int ROWS = W_THREADS / GL;  // rows of the block at a time
    constexpr int NEXT = SPLIT ? HD / 2 : 8;   // from a lane's first eight values to its other eight
    __shared__ __align__(16) float cs[HD / 2], sn[2][HD / 2];   // sines, negative and as they are
    extern __shared__ __align__(16) float stage[];   // W_THREADS * 16 floats where halves lie apart by other than a multiple of sixteen
    const int t = blockIdx.x, tid = threadIdx.x;
    const int half = SPLIT ? HD / 2 : rot / 2;
    const int n_rows = nh + (write_kv ? 2 * nkv : 0);
    const int g = tid / GL, l = tid % GL, d0 = SPLIT ? 8 * l : 16 * l;
    const T* src = qkv + static_cast<size_t>(t) * (nh + 2 * nkv) * HD + d0;
    const bool staged = !SPLIT && pairing == 0 && half % 16 != 0;
    // (positions, slots and frequencies were there before the kernel in front)
    pdl_entry();
    pdl_trigger();
    float x[W_AHEAD][16];
    auto load = [&](int r, float* v) {
        if (r < n_rows) {
            load8(src + static_cast<size_t>(r) * HD, v);
            load8(src + static_cast<size_t>(r) * HD + NEXT, v + 8);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = 0.f;
        }
    };
#pragma unroll
    for (int u = 0; u < W_AHEAD; ++u) load(u * ROWS + g, x[u]);
    if (tid < half) {
        const double turns = static_cast<double>(positions[t]) * static_cast<double>(inv_freq[tid]) * 0.15915494309189533577;
        float s;
        sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &cs[tid]);
        sn[0][tid] = -s;
        sn[1][tid] = s;
    }
    const int slot = slots ? slots[t] : 0;
    const int page = slot / P, off = slot - page * P;
    T* const q_row = q_out + static_cast<size_t>(t) * nh * HD + d0;
    uint8_t* const page_bytes = pool + q4_place(page, 0, 0, nkv, P, HD);
    const unsigned head_bytes = static_cast<unsigned>(P) * (HD / 2 + Q4_FACTOR_BYTES);
    __syncthreads();
    auto row = [&](int r, float* x) {
        const bool turn = r < nh + nkv;   // (q and k)
        if constexpr (SPLIT) {
            if (turn) {
                float c[8], s[8];
                load8(cs + d0, c);
                load8(sn[1] + d0, s);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a = x[i], b = x[8 + i];
                    x[i] = a * c[i] - b * s[i];
                    x[8 + i] = a * s[i] + b * c[i];
                }
            }
        } else if (half > 0 && __any_sync(0xffffffffu, turn)) {   // (rows of v beside rows of k take the shuffles with them and keep their values)
            if (pairing == 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int p = d0 / 2 + i;
                    if (turn && p < half) {
                        const float c = cs[p], s = sn[1][p], a = x[2 * i], b = x[2 * i + 1];
                        x[2 * i] = a * c - b * s;
                        x[2 * i + 1] = a * s + b * c;
                    }
                }
            } else if (!staged) {
                const bool low = d0 < half;
                const int lane = tid & 31, other = d0 < rot ? (lane - l) + (low ? l + half / 16 : l - half / 16) : lane;
                const bool in = turn && d0 < rot;
                const int p = low ? d0 : d0 - half;
                const float* sines = sn[low ? 0 : 1];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float y = __shfl_sync(0xffffffffu, x[i], other);
                    if (in) x[i] = fmaf(x[i], cs[p + i], y * sines[p + i]);
                }
            } else {
                float* mine = stage + static_cast<size_t>(g) * HD;
#pragma unroll
                for (int i = 0; i < 16; ++i) mine[d0 + i] = x[i];
                __syncwarp();
                if (turn)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int d = d0 + i;
                        if (d < half) x[i] = x[i] * cs[d] - mine[d + half] * sn[1][d];
                        else if (d < rot) x[i] = mine[d - half] * sn[1][d - half] + x[i] * cs[d - half];
                    }
                __syncwarp();
            }
        }
        if (r < nh) {
            store8(q_row + static_cast<size_t>(r) * HD, x);
            store8(q_row + static_cast<size_t>(r) * HD + NEXT, x + 8);
        }
        if (!__any_sync(0xffffffffu, r >= nh && r < n_rows)) return;   // (a warp of q's rows alone)
        float scale, mid;
        bool bad;
        q4_row_factors<GL>(x, scale, mid, bad);
        if (r < nh || r >= n_rows) return;
        const float inv = 1.f / scale;
        uint8_t* at = page_bytes + static_cast<unsigned>(r - nh) * head_bytes;   // (planes and heads lie as the rows of k and v do)
        uint32_t* words = reinterpret_cast<uint32_t*>(at + off * (HD / 2));
        const uint32_t w0 = q4_word(x, scale, mid, inv), w1 = q4_word(x + 8, scale, mid, inv);
        if (SPLIT) {
            words[l] = w0;
            words[l + GL] = w1;
        } else {
            reinterpret_cast<uint2*>(words)[l] = make_uint2(w0, w1);
        }
        if (l == 0) {
            reinterpret_cast<uint32_t*>(at + P * (HD / 2))[off] = bad ? 0x7fff7fffu : q4_factors(scale, mid);
            if (weights && turn) weights[(static_cast<size_t>(page) * nkv + (r - nh)) * P + off] = 0.f;
        }
    };
    for (int r0 = 0; r0 < n_rows; r0 += W_AHEAD * ROWS) {
        if (r0 > 0) {
#pragma unroll
            for (int u = 0; u < W_AHEAD; ++u) load(r0 + u * ROWS + g, x[u]);
        }
#pragma unroll
        for (int u = 0; u < W_AHEAD; ++u)
            if (r0 + u * ROWS < n_rows) row(r0 + u * ROWS + g, x[u]);
    }
}

template <typename T>
static int write_launch(const void* qkv, const int* positions, const float* inv_freq, void* q_out, uint8_t* pool, const int* slots,
                        float* weights, int n, int nh, int nkv, int hd, int rot, int pairing, int P, int write_kv, cudaStream_t stream) {
    const bool staged = pairing == 0 && (rot / 2) % 16 != 0, split = pairing == 0 && rot == hd;
#define Q4_WRITE_S(HD_, SPLIT_)                                                                                                         \
    locus_launch(q4_write_kernel<T, HD_, SPLIT_>, n, W_THREADS, staged ? W_THREADS * 16 * sizeof(float) : 0, stream,                    \
                 static_cast<const T*>(qkv), positions, inv_freq, static_cast<T*>(q_out), pool, slots, weights, nh, nkv, rot, pairing, \
                 P, write_kv)
#define Q4_WRITE(HD_)                     \
    do {                                  \
        if (split) Q4_WRITE_S(HD_, true); \
        else Q4_WRITE_S(HD_, false);      \
    } while (0)
    if (hd == 64) Q4_WRITE(64);
    else if (hd == 128) Q4_WRITE(128);
    else Q4_WRITE(256);
#undef Q4_WRITE
#undef Q4_WRITE_S
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
    if (!q4_head_ok(hd) || v.nh < 0 || v.nkv <= 0 || P <= 0 || P % 16 != 0 || rot < 0 || rot > hd || (rot & 1) || (v.pairing != 0 && v.pairing != 1) ||
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
// expand: the rows of positions 0 .. seg_ctx + seg_qn - 1 of the listed segments (null: the first ones) that have at least min_new new tokens
// into ordinary pages [n_pages][2][nkv][P][hd] of the same page ids, in the model's type (float32: as they are; bfloat16: one rounding, the tensor cores' operand).  Rows behind a request's last
// token and pages that went back (-1) stay as they were.
// One block per (page of the request, plane, head): P rows, a lane takes words of eight values, E_AHEAD at a time.  Bound by memory: 8,192 tokens of
// 16 heads of 128 in 13 us, 6.5 TB/s.
// bfloat16 without a detour: 16 + code is 0x4180 | code << 3, 23.5 off is exact, and one fused multiply-add rounds once.
#define E_THREADS 256
#define E_AHEAD 4
__device__ __forceinline__ void q4_eight(uint32_t w, uint32_t f, float* out) {
    float v[8];
    const float scale = q4_scale(f), mid = q4_mid(f);
#pragma unroll
    for (int d = 0; d < 8; ++d)   // (2^23 + code less 2^23 + 7.5, exactly)
        v[d] = fmaf(scale, (__uint_as_float(((w >> q4_shift(d)) & 15u) | 0x4b000000u) - 8388608.f) - 7.5f, mid);
    store8(out, v);
}
__device__ __forceinline__ void q4_eight(uint32_t w, uint32_t f, bf16* out) {
    const __nv_bfloat162 factors = *reinterpret_cast<const __nv_bfloat162*>(&f);
    const __nv_bfloat162 scale = __low2bfloat162(factors), mid = __high2bfloat162(factors);
    const uint32_t k = 0x41bc41bcu;   // 23.5 twice
    uint4 o;
    uint32_t* v = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t y = ((i == 0 ? w << 3 : w >> (4 * i - 3)) & 0x00780078u) | 0x41804180u;
        const __nv_bfloat162 c = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&y), *reinterpret_cast<const __nv_bfloat162*>(&k));
        const __nv_bfloat162 r = __hfma2(scale, c, mid);
        v[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
    *reinterpret_cast<uint4*>(out) = o;
}
template <typename T, int HD>
__global__ void __launch_bounds__(E_THREADS) q4_expand_kernel(const uint8_t* __restrict__ pool, T* __restrict__ out,
                                                              const int* __restrict__ segs, const int* __restrict__ seg_ctx,
                                                              const int* __restrict__ seg_qn, const int* __restrict__ block_table,
                                                              int table_stride, int nkv, int P, int min_new) {
    constexpr int WR = HD / 8;   // words of a row
    pdl_entry();
    pdl_trigger();
    const int seg = segs ? segs[blockIdx.z] : static_cast<int>(blockIdx.z);
    const int fresh = seg_qn[seg], n = seg_ctx[seg] + fresh;
    if (fresh < min_new) return;
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
    for (int i0 = threadIdx.x; i0 < words; i0 += E_AHEAD * E_THREADS) {
        uint32_t w[E_AHEAD], f[E_AHEAD];
#pragma unroll
        for (int u = 0; u < E_AHEAD; ++u) {
            const int i = i0 + u * E_THREADS;
            if (i < words) {
                w[u] = codes[i];
                f[u] = factors[i / WR];
            }
        }
#pragma unroll
        for (int u = 0; u < E_AHEAD; ++u) {
            const int i = i0 + u * E_THREADS;
            if (i < words) q4_eight(w[u], f[u], dst + static_cast<size_t>(i) * 8);
        }
    }
}

// max_keys: at least the tokens of the longest of these segments.
struct Q4ExpandCall {
    const void* pool;
    void* out;
    const int *segs, *seg_ctx, *seg_qn, *block_table;
    long long dt, n_segs, table_stride, nkv, hd, P, max_keys, min_new;
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
                 v.block_table, table_stride, nkv, P, static_cast<int>(v.min_new))
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
// One block per (layer, request, head).  The weights are read once, as unsigned numbers of the same order: into registers, a run of KPT x 32 keys a warp,
// where the block's threads hold them, else into shared memory (SK_MAX), else from memory (the L2) in every pass.  The weight of the last key that
// stays is found by histograms of S_BINS bins over the range of numbers that it must lie in, at first from the smallest to the largest, then one bin
// of the pass before: three passes at most, mostly two, and only keys of that range are counted, so that bins are hit evenly and seldom by a
// warp's lanes at once.  Then every warp counts the keys of its run that stay, and behind a sum over the warps writes their indices in order.
// (24 layers of 16 heads of one request of 4,096 tokens: a fixed cut of the 32 bits by 11, 11 and 10 and blocks of 1,024 threads 31 us, most of it
// atomics on the few bins that exponents hit; by ranges, blocks of 256 threads with the keys in shared memory 24, in registers 14.  28 layers of 4 heads
// of 8 requests of up to 8,192 tokens 38, in blocks of 512 threads of 16 keys; 256 of 32 and 1,024 of 8 are 5 to 10 us slower.)
#define SK_MAX 49152      // weights in shared memory (192 KB)
#define S_BINS 2048

// an unsigned number of the weight's order
__device__ __forceinline__ uint32_t ordered(float w) {
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);   // (-0 and 0 are one weight)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// t / P for t and 2^40 / P below 2^27 and 2^37: a multiplication by ceil(2^40 / P)
__device__ __forceinline__ int by_page(int t, unsigned long long page_inv) { return static_cast<int>((static_cast<unsigned long long>(t) * page_inv) >> 40); }

// KPT keys of a thread in registers (n_tokens at most THREADS * KPT); 0: keys in shared memory (up to `room`) or in memory.
template <int THREADS, int KPT>
__global__ void __launch_bounds__(THREADS) q4_select_kernel(const float* __restrict__ weights, const int* __restrict__ block_table, int table_stride,
                                                            const int* __restrict__ n_tokens, int n_items, int nkv, int P,
                                                            unsigned long long page_inv, size_t layer_slots, int keep, int first, int recent,
                                                            int room, int* __restrict__ kept) {
    constexpr int WARPS = THREADS / 32, BT = S_BINS / THREADS;   // bins of a thread
    constexpr uint32_t SURE = 0xffffffffu;                        // the first and the last keys (no weight maps to it), and keys behind the last
    extern __shared__ uint32_t s_keys[];
    __shared__ __align__(16) int hist[S_BINS];
    __shared__ int warp_a[WARPS], warp_b[WARPS];
    __shared__ uint32_t warp_lo[WARPS], warp_hi[WARPS];
    __shared__ int chosen_bin, above_bin;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_entry();
    pdl_trigger();
    const int h = blockIdx.x, item = blockIdx.y, layer = blockIdx.z;
    int n = min(n_tokens[item], table_stride * P);
    if (KPT > 0) n = min(n, THREADS * KPT);
    int* dst = kept + ((static_cast<size_t>(layer) * n_items + item) * nkv + h) * keep;
    if (n <= keep) {
        for (int j = tid; j < keep; j += THREADS) dst[j] = j < n ? j : -1;
        return;
    }
    const float* w = weights + static_cast<size_t>(layer) * layer_slots + static_cast<size_t>(h) * P;
    const int* table = block_table + static_cast<size_t>(item) * table_stride;
    const size_t page_step = static_cast<size_t>(nkv) * P;
    const int lo = first, hi = n - recent;       // the keys between, of which `left` stay
    int left = keep - first - recent;
    auto read = [&](int t) -> uint32_t {
        if (t < lo || t >= hi) return SURE;
        const int at = by_page(t, page_inv), page = table[at];
        return page < 0 ? 0u : ordered(w[page * page_step + (t - at * P)]);
    };
    const bool in_smem = KPT == 0 && n <= room;
    // a warp's run of keys: a .. b - 1, key i * 32 + lane of it in mine[i]
    const int per = KPT > 0 ? KPT * 32 : ((n + WARPS - 1) / WARPS + 31) & ~31;
    const int a = min(n, warp * per), b = min(n, a + per);
    uint32_t mine[KPT > 0 ? KPT : 1];
    auto each = [&](auto&& f) {   // f(key) for every key of the run: this lane's
        if constexpr (KPT > 0) {
#pragma unroll
            for (int i = 0; i < KPT; ++i) f(mine[i]);
        } else {
#pragma unroll 4
            for (int t = a + lane; t < b; t += 32) f(in_smem ? s_keys[t] : read(t));
        }
    };
    if constexpr (KPT > 0) {
        // pages first, then weights: eight of either on their way together
#pragma unroll
        for (int i0 = 0; i0 < KPT; i0 += 8) {
            int page[8];
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = a + (i0 + i) * 32 + lane;
                page[i] = t >= lo && t < hi ? table[by_page(t, page_inv)] : -2;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = a + (i0 + i) * 32 + lane;
                v[i] = page[i] >= 0 ? w[page[i] * page_step + (t - by_page(t, page_inv) * P)] : __int_as_float(0x7fffffff);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) mine[i0 + i] = page[i] == -2 ? SURE : ordered(v[i]);
        }
    } else if (in_smem) {
#pragma unroll 4
        for (int t = a + lane; t < b; t += 32) s_keys[t] = read(t);
    }
    uint32_t from = SURE - 1, to = 0;   // the numbers that the last key to stay lies between
    bool ties = false;                  // keys equal to `from`: the first `left` of them stay; else all from `from` on
    if (left > 0) {
        uint32_t least = SURE, most = 0u;
        each([&](uint32_t u) {
            least = min(least, u);
            if (u != SURE) most = max(most, u);
        });
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) {
            warp_lo[warp] = least;
            warp_hi[warp] = most;
        }
        for (int i = tid; i < S_BINS / 4; i += THREADS) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
        __syncthreads();
        from = __reduce_min_sync(0xffffffffu, lane < WARPS ? warp_lo[lane] : SURE);
        to = __reduce_max_sync(0xffffffffu, lane < WARPS ? warp_hi[lane] : 0u);
        while (true) {
            const uint32_t span = to - from;
            const int shift = span ? max(0, 32 - __clz(span) - 11) : 0;   // (span >> shift) < S_BINS
            each([&](uint32_t u) {
                u -= from;
                if (u <= span) atomicAdd(&hist[u >> shift], 1);
            });
            __syncthreads();
            // keys in higher bins, from the top: thread i has bins from S_BINS - 1 - BT i down
            int bins[BT], run = 0;
#pragma unroll
            for (int i = 0; i < BT; ++i) {
                bins[i] = hist[S_BINS - 1 - BT * tid - i];
                run += bins[i];
            }
            const int own_sum = run;
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, run, m);
                if (lane >= m) run += v;
            }
            if (lane == 31) warp_a[warp] = run;
            __syncthreads();
            int before = __reduce_add_sync(0xffffffffu, lane < warp ? warp_a[lane] : 0) + run - own_sum;   // keys above this thread's bins
#pragma unroll
            for (int i = 0; i < BT; ++i) {
                if (before < left && before + bins[i] >= left) {
                    chosen_bin = S_BINS - 1 - BT * tid - i;
                    above_bin = before;
                    warp_b[0] = bins[i];
                }
                before += bins[i];
                hist[S_BINS - 1 - BT * tid - i] = 0;   // (for the next pass)
            }
            __syncthreads();
            const int bin = chosen_bin, count = warp_b[0];
            left -= above_bin;
            from += static_cast<uint32_t>(bin) << shift;
            to = from + min(to - from, (1u << shift) - 1u);
            if (count == left) break;   // the whole bin stays
            if (shift == 0) {           // (equal weights)
                ties = true;
                break;
            }
        }
        __syncthreads();
    }
    // of the keys between those from `from` on stay, of those equal to it with `ties` only the first `left`
    int n_stay = 0, n_tie = 0;
    each([&](uint32_t u) {
        const bool tie = ties && u == from;
        n_stay += u >= from && !tie;
        n_tie += tie;
    });
    if constexpr (KPT > 0) {   // (less the places behind the last key)
        int dead = 0;
#pragma unroll
        for (int i = 0; i < KPT; ++i) dead += a + i * 32 + lane >= b;
        n_stay -= dead;
    }
    n_stay = __reduce_add_sync(0xffffffffu, n_stay);
    n_tie = __reduce_add_sync(0xffffffffu, n_tie);
    if (lane == 0) {
        warp_a[warp] = n_stay;
        warp_b[warp] = n_tie;
    }
    __syncthreads();
    // ties taken and keys written by the warps in front
    int taken = __reduce_add_sync(0xffffffffu, lane < warp ? warp_b[lane] : 0);
    int at = __reduce_add_sync(0xffffffffu, lane < warp ? warp_a[lane] : 0) + min(taken, max(left, 0));
    const uint32_t below = (1u << lane) - 1;
    int t = a + lane;
    auto put = [&](uint32_t u) {
        const bool tie = ties && u == from;
        bool in = t < b && u >= from && !tie;
        if (ties) {
            const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
            in = in || (tie && taken + __popc(tie_mask & below) < left);
            taken += __popc(tie_mask);
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, in);
        if (in) dst[at + __popc(mask & below)] = t;
        at += __popc(mask);
        t += 32;
    };
    if constexpr (KPT > 0) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) put(mine[i]);
    } else {
        for (int t0 = a; t0 < b; t0 += 32) put(t0 + lane >= b ? 0u : in_smem ? s_keys[t0 + lane] : read(t0 + lane));
    }
}

// evict, second half: key kept[j] of a request's pages becomes key j of the pages of dst_table, rows, factors and weight.
// In place (dst_table the request's own table) a row's old place may be another row's new one, but never that of a row in front of it
// (kept[j] >= j): a block takes (layer, request, head, plane) and walks its rows from the front, a tile at a time, and reads a tile before it
// writes it.  Into other pages the order is free, and several blocks share the rows.
// Bound by memory: 28 layers of 4 heads of 8 requests of 2,500 to 8,192 tokens, 4,000 of each staying, in 186 us, 970 MB read and written (5.2 TB/s), of
// which 100 MB are the rest of the 32-byte sectors that single factors and weights lie in.
#define M_THREADS 256
#define M_UNROLL 8       // 16-byte pieces of a thread in flight

// 16 bytes of a row; rows are read once, and rows that do not stay lie between them
__device__ __forceinline__ uint4 ld_row(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.L2::64B.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

template <int HD>
__global__ void __launch_bounds__(M_THREADS) q4_move_kernel(uint8_t* pool, float* weights, const int* __restrict__ block_table,
                                                            int table_stride, const int* __restrict__ dst_table, int dst_stride,
                                                            const int* __restrict__ n_tokens, int n_items, int nkv, int P,
                                                            unsigned long long page_inv, size_t layer_bytes, size_t layer_slots, int keep,
                                                            int n_parts, const int* __restrict__ kept) {
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

    // a row's old and new place in its layer, in pieces (of 16 bytes); rows without a page: none
    constexpr unsigned NONE = 0xffffffffu;
    __shared__ uint2 places[TILE];
    const unsigned page_pieces = 2u * nkv * P * (HD / 2 + Q4_FACTOR_BYTES) / 16;
    const unsigned head_pieces = (static_cast<unsigned>(plane) * nkv + h) * (P * (HD / 2 + Q4_FACTOR_BYTES) / 16);
    for (int j0 = part * TILE; j0 < n; j0 += n_parts * TILE) {
        uint32_t fac[FU];
        float wt[FU];
        int new_page[FU], new_off[FU];
#pragma unroll
        for (int u = 0; u < FU; ++u) {
            const int e = u * M_THREADS + tid, j = j0 + e;
            new_page[u] = -1;
            if (e < TILE) {
                uint2 at = make_uint2(NONE, NONE);
                if (j < n) {
                    const int s = idx[j], sp = by_page(max(s, 0), page_inv), so = s - sp * P, page = s < 0 ? -1 : table[sp];
                    const int dp = by_page(j, page_inv), dpage = to[dp];
                    if (page >= 0 && dpage >= 0) {
                        at = make_uint2(page * page_pieces + head_pieces + so * PR, dpage * page_pieces + head_pieces + (j - dp * P) * PR);
                        fac[u] = reinterpret_cast<const uint32_t*>(place(page) + P * (HD / 2))[so];
                        if (plane == 0) wt[u] = w[(static_cast<size_t>(page) * nkv + h) * P + so];
                        new_page[u] = dpage;
                        new_off[u] = j - dp * P;
                    }
                }
                places[e] = at;
            }
        }
        __syncthreads();
        uint4 piece[M_UNROLL];
        unsigned dst[M_UNROLL];
#pragma unroll
        for (int u = 0; u < M_UNROLL; ++u) {
            const uint2 at = places[(u * M_THREADS + tid) / PR];
            dst[u] = at.y;
            if (at.x != NONE) piece[u] = ld_row(base + (static_cast<size_t>(at.x) + tid % PR) * 16);
        }
        __syncthreads();   // (in place: every row of the tile is read before one is written; and `places` is free)
#pragma unroll
        for (int u = 0; u < M_UNROLL; ++u)
            if (dst[u] != NONE) *reinterpret_cast<uint4*>(base + (static_cast<size_t>(dst[u]) + tid % PR) * 16) = piece[u];
#pragma unroll
        for (int u = 0; u < FU; ++u)
            if (new_page[u] >= 0) {
                reinterpret_cast<uint32_t*>(place(new_page[u]) + P * (HD / 2))[new_off[u]] = fac[u];
                if (plane == 0) w[(static_cast<size_t>(new_page[u]) * nkv + h) * P + new_off[u]] = wt[u];
            }
    }
}

// max_tokens: at least the tokens of the longest request (a request's tokens behind that are not seen).  A layer of at most 64 GB.
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
        n_items > 65535 || v.n_layers > 65535 || !aligned16(v.pool) || max_tokens <= 0 || max_tokens >= 1 << 27 ||
        static_cast<unsigned long long>(v.layer_pages) * 2 * nkv * P * q4_row_bytes(hd) / 16 >= 0xffffffffull)
        return LOCUS_ERR_UNSUPPORTED;
    const size_t slots = static_cast<size_t>(v.layer_pages) * nkv * P, bytes = slots * 2 * q4_row_bytes(hd);
    const dim3 grid(nkv, n_items, static_cast<unsigned>(v.n_layers));
    static unsigned long long asked = 0;   // devices that know of the kernel's shared memory (asked again at worst)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return static_cast<int>(cudaGetLastError());
    if (dev >= 64 || !(asked >> dev & 1)) {
        if (cudaFuncSetAttribute(q4_select_kernel<1024, 0>, cudaFuncAttributeMaxDynamicSharedMemorySize, SK_MAX * 4) != cudaSuccess)
            return static_cast<int>(cudaGetLastError());
        if (dev < 64) asked |= 1ull << dev;
    }
    const unsigned long long page_inv = ((1ull << 40) + P - 1) / P;
#define Q4_SELECT(THREADS_, KPT_, ROOM_)                                                                                                    \
    locus_launch(q4_select_kernel<THREADS_, KPT_>, grid, THREADS_, static_cast<size_t>(ROOM_) * 4, stream, v.weights, v.block_table,        \
                 table_stride, v.n_tokens, n_items, nkv, P, page_inv, slots, keep, first, recent, ROOM_, v.kept)
    if (max_tokens <= 256 * 8) Q4_SELECT(256, 8, 0);
    else if (max_tokens <= 256 * 16) Q4_SELECT(256, 16, 0);
    else if (max_tokens <= 512 * 16) Q4_SELECT(512, 16, 0);
    else if (max_tokens <= 1024 * 16) Q4_SELECT(1024, 16, 0);
    else Q4_SELECT(1024, 0, (max_tokens <= SK_MAX ? max_tokens : 0));
#undef Q4_SELECT
    const int code = locus_launch_status();
    if (code) return code;
    const int tile = M_THREADS * M_UNROLL / (hd / 32);
    const int n_parts = v.dst_table == v.block_table ? 1 : max(1, min(ceil_div(min(keep, max_tokens), tile), 16));
    const dim3 mgrid(2 * nkv * n_parts, n_items, static_cast<unsigned>(v.n_layers));
#define Q4_MOVE(HD_)                                                                                                                        \
    locus_launch(q4_move_kernel<HD_>, mgrid, M_THREADS, 0, stream, static_cast<uint8_t*>(v.pool), v.weights, v.block_table, table_stride,   \
                 v.dst_table, dst_stride, v.n_tokens, n_items, nkv, P, page_inv, bytes, slots, keep, n_parts, v.kept)
    if (hd == 64) Q4_MOVE(64);
    else if (hd == 128) Q4_MOVE(128);
    else Q4_MOVE(256);
#undef Q4_MOVE
    return locus_launch_status();
}
