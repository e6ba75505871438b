// Tokens into and out of a paged cache, any number per sequence:
//   append  the fused q/k/v projection rows of every sequence's new tokens: q and k rotated, q written, k and v quantised
//           and stored at positions seq_lens[b], seq_lens[b] + 1, ... of sequence b (a prompt, a chunk of one, a step);
//   read    rows of tokens that the cache holds, as values (the prefix that a chunk of prompt attends to, a check of what
//           was stored, a move to another cache).
// No reference counterpart: the reference concatenates fp16 tensors (DynamicCache.update,
// benchmarks/llama_integration_benchmark.py:173).  skv_rope_quant_append stores one token per sequence.
//
// Caches: 4-bit page records (skv_kv4.cuh), 8-bit pools or fused page records (one fp32 scale a row), 8-bit keys with 4-bit
// values; all addressed through strides.
//
// Bound: HBM for prompts (D = 128, 16-bit activations: 256 bytes read per row, 256 written per query row, 72 per 4-bit
// row), latency for a step.  LPR = D/8 lanes hold one row, eight channels (16 bytes) a lane; a block keeps a few tokens and
// walks over heads, so sines and cosines are worked out once; U rows are worked on while the next U are on their way.  The group
// maxima are shuffles among the lanes that share a scale; a row's partner channels (half layout) come by shuffle too.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "skv_common.cuh"
#include "skv_kv4.cuh"

namespace skv {
namespace tok {

constexpr int THREADS = 128;
enum { CACHE_KV4 = 0, CACHE_E4M3 = 1, CACHE_I8 = 2, CACHE_E4M3_V4 = 3, CACHE_I8_V4 = 4 };

struct Pools {
    uint8_t* k; uint8_t* v;      // 4-bit records: k is the record base, v unused
    float* ks; float* vs;
    long long sp, sh, ss, csp, csh;   // strides in bytes (codes) and floats (scales)
    const int* page_table;
    int max_pages, num_pages, page_size;
    int* status;
};

struct AppendParams {
    const void* qkv;
    void* q_out;
    const unsigned long long* freqs;   // null: no rotation
    const void* positions;             // null: the cache position
    const int* cu_new;                 // null: one token per sequence
    const int* seq_lens;
    Pools c;
    long long qkv_stride;
    int T, B, Hq, Hkv, R, interleaved, pos64, q_bf16, head_splits, heads_per_split;
    double factor;
};

struct ReadParams {
    void* k_out; void* v_out;
    const int* cu;
    const int* starts;                 // null: 0
    Pools c;
    int T, B, Hkv, out_bf16, head_splits, heads_per_split;
};

// Sequence of row t: the number of sequences that end at or before it (B: behind the last).  Lanes of a row share the
// count while a few loads each do it, else they all search.  Whether the row is that sequence's is the caller's question: offsets
// that begin above 0 give the rows before them sequence 0.  An array that does not ascend gives some sequence: the row's
// position is checked before anything is stored.
template <int LPR>
__device__ __forceinline__ int sequence_of(const int* cu, int B, long long t, int l, unsigned group) {
    if (B <= 16 * LPR) {
        int n = 0;
        for (int i = l; i < B; i += LPR) n += cu[SKV_INDEX(i, B) + 1] <= t;
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) n += __shfl_xor_sync(group, n, o);
        return n;
    }
    int lo = 0, hi = B;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[SKV_INDEX(mid, B) + 1] <= t) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// x / s as correctly rounded division gives it, with r = 1 / s correctly rounded: one residual correction (Markstein's
// theorem), which holds while nothing in it under- or overflows, that is for s far from both ends of the range.
__device__ __forceinline__ float div_by(float x, float s, float r) {
    const float q = x * r;
    return fmaf(fmaf(-q, s, x), r, q);
}
__device__ __forceinline__ bool div_safe(float s) { return s > 7.9e-31f && s < 1.2e30f; }   // 2^-100 .. 2^100

__device__ __forceinline__ float bf16_bits_to_f(uint32_t b) { return __uint_as_float(b << 16); }

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& raw, float (&x)[8]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 2 && __is_same(T, __half)) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        } else {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

__device__ __forceinline__ uint32_t pack16(float a, float b, bool bf16) {
    if (bf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    return pack_half2(a, b);
}

// Eight fp32 channels of a row, quantised with one scale for LANES lanes: LANES = 4 groups of 32 (bf16 scale, 4-bit
// records), LPR: whole rows (fp32 scale).  One rule makes the scale in every format: amax times the fp32 number nearest to
// 1 / top code (7, 127, 448).  That is what torch makes of amax / 7 on the GPU, so rows quantised there and here hold the same
// codes; many values lie exactly between two codes, and which one they take follows the last bit of the scale.
// (skv_rope_quant_append divides: a scale may differ from its in the last bit, and codes of values between two then.)
template <int LANES>
__device__ __forceinline__ uint32_t abs_max_bits(const float (&x)[8], unsigned group) {
    uint32_t m = 0;   // the bits of |x| order like |x|, infinities and NaN on top
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(group, m, o));
    return m;
}

// Codes of eight quotients.  A quotient is at most its top code and a thousandth, which rounds to the top code: no clamp.  The
// rounding to whole numbers, ties to even, is the addition of 1.5 * 2^23 (+ 8, even too): the sum's low bits are the code
// (+ 8), and the eight words weighted by powers of 16, less the same sum of their constant parts, are the packed nibbles --
// half the instructions that conversions, clamps and shifts take.
__device__ __forceinline__ uint32_t nibbles8(const float (&x)[8], float s, float r) {
    uint32_t w = 0;
    if (div_safe(s)) {
#pragma unroll
        for (int i = 7; i >= 0; --i) w = w * 16u + __float_as_uint(__fadd_rn(div_by(x[i], s, r), 12582920.f));
    } else {
#pragma unroll
        for (int i = 7; i >= 0; --i) w = w * 16u + __float_as_uint(__fadd_rn(__fdiv_rn(x[i], s), 12582920.f));
    }
    return w - 0x3f400000u;                           // 0x4b400000 * 0x11111111
}

template <int D, bool IS_V>
__device__ __forceinline__ void store_kv4(const float (&x)[8], uint8_t* rec, int slot, int l, unsigned group, bool live) {
    constexpr int W = D / 32;
    const uint32_t m = abs_max_bits<4>(x, group);
    const bool finite = m < 0x7f800000u;
    const uint16_t sb = finite ? __bfloat16_as_ushort(__float2bfloat16_rn(__fmul_rn(__uint_as_float(m), 1.f / 7.f))) : (uint16_t)0x7fc0;
    const float s = bf16_bits_to_f(sb);
    // (a scale of zero or NaN: all codes zero.  Scales below the normal range hold no more than that either.)
    const uint32_t word = finite && s >= 1.1754944e-38f ? nibbles8(x, s, __frcp_rn(s)) : 0x88888888u;
    const int w = l >> 2, c = l & 3;
    if (IS_V) {
        // the lane's eight channels are value chunks g = 2c (low half) and 2c + 1; the W words of one chunk sit in the lanes
        // c, c + 4, ...: lane c gathers the low halves, lane c + 4 the high ones, and each stores 2 W bytes at once
        uint32_t part[W];
#pragma unroll
        for (int i = 0; i < W; ++i) part[i] = __shfl_sync(group, word, ((threadIdx.x & 31) & ~(D / 8 - 1)) + c + 4 * i);
        if (live && w < 2) {
            uint8_t* dst = rec + kv4_v_row<D>(slot) + (2 * c + w) * (D / 2);
            const uint32_t sel = w ? 0x7632u : 0x5410u;
            if constexpr (W == 4)
                *reinterpret_cast<uint2*>(dst) = make_uint2(__byte_perm(part[0], part[1], sel), __byte_perm(part[2], part[3], sel));
            else
                *reinterpret_cast<uint32_t*>(dst) = __byte_perm(part[0], part[1], sel);
        }
    } else if (live) {
        *reinterpret_cast<uint32_t*>(rec + kv4_place(slot) * (D / 2) + c * (D / 8) + w * 4) = word;
    }
    if (live && c == 0) *reinterpret_cast<uint16_t*>(rec + kv4_scales<D>(slot) + (IS_V ? D / 16 : 0) + 2 * w) = sb;
}

// Rows with one fp32 scale: 1 for a zero row, NaN for a row that is not finite.  BITS4: nibbles, else bytes.
template <int LPR, int CACHE, bool BITS4>
__device__ __forceinline__ void store_row(const float (&x)[8], uint8_t* row, float* scale, int l, unsigned group, bool live) {
    constexpr bool E4M3 = !BITS4 && (CACHE == CACHE_E4M3 || CACHE == CACHE_E4M3_V4);
    const uint32_t m = abs_max_bits<LPR>(x, group);
    const bool finite = m < 0x7f800000u;
    const float amax = __uint_as_float(m);
    const float top = __fmul_rn(amax, 1.f / (BITS4 ? 7.f : E4M3 ? 448.f : 127.f));
    const float s = finite ? (amax > 0.f ? top : 1.f) : __uint_as_float(0x7fc00000u);
    const float r = __frcp_rn(s);
    const bool any = finite && s >= 1.1754944e-38f;  // (a scale that is NaN, or below the normal range: all codes zero)
    if (BITS4) {
        const uint32_t word = any ? nibbles8(x, s, r) : 0x88888888u;
        if (live) *reinterpret_cast<uint32_t*>(row + l * 4) = word;
    } else {
        float q[8];
        if (div_safe(s)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = div_by(x[i], s, r);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = any ? __fdiv_rn(x[i], s) : 0.f;
        }
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (E4M3) {
                w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q[4 * i], q[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
                       ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(q[4 * i + 2], q[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16);
            } else {                                  // the low byte of a quotient + 1.5 * 2^23 is its whole number
                uint32_t c[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) c[j] = __float_as_uint(__fadd_rn(q[4 * i + j], 12582912.f));
                w[i] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
            }
        }
        if (live) *reinterpret_cast<uint2*>(row + l * 8) = make_uint2(w[0], w[1]);
    }
    if (live && l == 0) *scale = s;
}

// Page of position pos of sequence b, or -1 (no room in the page list, or a table entry outside the pool, reported)
__device__ __forceinline__ int page_of(const Pools& c, int b, long long pos, int& slot) {
    if (pos < 0 || pos >= (long long)c.max_pages * c.page_size) return -1;
    const int lp = (int)(pos / c.page_size);
    slot = (int)(pos - (long long)lp * c.page_size);
    const int page = c.page_table ? c.page_table[(long long)b * c.max_pages + SKV_INDEX(lp, c.max_pages)] : b * c.max_pages + lp;
    slot = SKV_INDEX(slot, c.page_size);
    if ((unsigned)page >= (unsigned)c.num_pages) {
        if (c.status) atomicOr(c.status, SKV_DEV_BAD_PAGE);
        return -1;
    }
    return SKV_INDEX(page, c.num_pages);
}

// 8192 tokens, 32 + 8 + 8 heads of 128 in bf16, 4-bit cache: 42.5 us (4.2 TB/s, 0.64 of a copy; 37.9 without rotation).  No one
// limit shows: issue slots are 70 % busy (163 instructions per two rows), waits are for fixed latencies, shared memory and
// instructions more than for loads, and a copy without what a block finds out first (sequence, length, page, sines) takes
// 37.3.  Query rows as four channels and their four partners, without shuffles: 45.0; with loops of their own for query rows
// and for keys and values: 43.7 at best, and narrow rows slower (5.9 -> 6.6).  U and registers of 2 | 64, 3 | 80, 4 | 96: 43.4, 42.5, 43.9;
// blocks of 64, 96, 256 threads: 44.6, 45.1, 53.6; plain loads 43.0.
template <typename T, int D, int CACHE>
__global__ void __launch_bounds__(THREADS, 6) append_tokens_kernel(const AppendParams p) {
    constexpr int LPR = D / 8, U = 3;
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    constexpr int ROWS = 32 / LPR, WARPS = THREADS / 32;
    __shared__ float2 table[ROWS * D / 2];            // (cos, sin) of the block's tokens: [token][pair]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (LPR - 1);
    // a block takes ROWS tokens and a share of the heads; every warp holds all its tokens and takes every fourth head
    const int split = (int)(blockIdx.x % (unsigned)p.head_splits);
    const long long t = (long long)(blockIdx.x / (unsigned)p.head_splits) * ROWS + lane / LPR;
    const unsigned group = 0xffffffffu;
    const bool in = t < p.T;
    const int heads = p.Hq + 2 * p.Hkv, h_begin = split * p.heads_per_split + warp;
    const int h_end = min(heads, (split + 1) * p.heads_per_split);
    const int d0 = l * 8;

    // rows are asked for before anything is known of their sequence (one behind the last reads the first row and drops it)
    const T* src = static_cast<const T*>(p.qkv) + (long long)SKV_INDEX(in ? t : 0, p.T) * p.qkv_stride + d0;
    uint4 next[U];
    auto load = [&](int h0) {
#pragma unroll
        for (int u = 0; u < U; ++u) next[u] = ld_stream16(src + (long long)SKV_INDEX(min(h0 + u * WARPS, heads - 1), heads) * D);
    };
    load(h_begin);

    int b = in ? (int)min(t, (long long)p.B) : p.B;
    long long pos = 0;
    if (p.cu_new) {
        const int s = sequence_of<LPR>(p.cu_new, p.B, in ? t : (long long)p.T, l, group);
        b = in ? s : p.B;
    }
    int page = -1, slot = 0;
    bool mine = b < p.B;                     // rows before the first sequence and behind the last are left alone
    if (mine) {
        b = SKV_INDEX(b, p.B);
        const long long i = p.cu_new ? t - p.cu_new[b] : 0;
        mine = i >= 0;
        pos = (long long)p.seq_lens[b] + i;
    }
    if (mine) {
        page = page_of(p.c, b, pos, slot);
        const int at = SKV_INDEX(t, p.T);
        if (p.positions) pos = p.pos64 ? static_cast<const long long*>(p.positions)[at]
                                       : (long long)static_cast<const int*>(p.positions)[at];
    }

    // the lane's channels: 8 pairs with a partner lane (half layout; the first half takes the sine negative), or 4 of its own
    const bool turned = p.freqs && d0 < p.R;
    float cs[8], sn[8];
    int partner = lane;
    if (p.freqs) {
        const int half = p.R / 2;
        for (int i0 = 0; i0 < ROWS * half; i0 += THREADS) {
            const int i = min(i0 + (int)threadIdx.x, ROWS * half - 1), r = i / half;
            const long long at = __shfl_sync(group, pos, r * LPR);
            table[SKV_INDEX(i, ROWS * D / 2)] = rotary_cos_sin(at, p.freqs[SKV_INDEX(i - r * half, half)], p.factor);
        }
        __syncthreads();
        if (turned) {
            const float2* f = table + (lane / LPR) * half;
            if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; ++i) { cs[i] = f[l * 4 + i].x; sn[i] = f[l * 4 + i].y; }
            } else {
                const bool first = d0 < half;
                partner = first ? lane + p.R / 16 : lane - p.R / 16;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 x = f[(first ? d0 : d0 - half) + i];
                    cs[i] = x.x;
                    sn[i] = first ? -x.y : x.y;
                }
            }
        }
    }

    __half* q_row = static_cast<__half*>(p.q_out) + t * p.Hq * D + d0;
    const bool live = mine && page >= 0;
    const long long pg = live ? page : 0;
    for (int h0 = h_begin; h0 < h_end; h0 += U * WARPS) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = next[u];
        if (h0 + U * WARPS < h_end) load(h0 + U * WARPS);   // the next rows are on their way while these are worked on
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u * WARPS;
            if (h >= h_end) break;
            float x[8];
            unpack16<T>(raw[u], x);
            if (h < p.Hq + p.Hkv) {
                if (p.interleaved) {
                    if (turned) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float a = x[2 * i], c = x[2 * i + 1];
                            rotary_turn(a, c, sn[i], cs[i], x[2 * i], x[2 * i + 1]);
                        }
                    }
                } else if (p.freqs) {
                    uint4 o;
                    o.x = __shfl_sync(group, raw[u].x, partner); o.y = __shfl_sync(group, raw[u].y, partner);
                    o.z = __shfl_sync(group, raw[u].z, partner); o.w = __shfl_sync(group, raw[u].w, partner);
                    if (turned) {
                        float y[8];
                        unpack16<T>(o, y);
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = __fadd_rn(__fmul_rn(x[i], cs[i]), __fmul_rn(y[i], sn[i]));
                    }
                }
                if (h < p.Hq) {
                    if (mine)
                        *reinterpret_cast<uint4*>(q_row + (long long)h * D) =
                            make_uint4(pack16(x[0], x[1], p.q_bf16), pack16(x[2], x[3], p.q_bf16), pack16(x[4], x[5], p.q_bf16),
                                       pack16(x[6], x[7], p.q_bf16));
                    continue;
                }
            }
            const bool is_v = h >= p.Hq + p.Hkv;
            const int hk = h - p.Hq - (is_v ? p.Hkv : 0);
            if constexpr (CACHE == CACHE_KV4) {
                uint8_t* rec = p.c.k + pg * p.c.sp + hk * p.c.sh;
                if (is_v) store_kv4<D, true>(x, rec, slot, l, group, live);
                else store_kv4<D, false>(x, rec, slot, l, group, live);
            } else {
                float* sc = (is_v ? p.c.vs : p.c.ks) + pg * p.c.csp + hk * p.c.csh + slot;
                if (is_v && (CACHE == CACHE_E4M3_V4 || CACHE == CACHE_I8_V4))
                    store_row<LPR, CACHE, true>(x, p.c.v + pg * p.c.sp + hk * p.c.sh + slot * (D / 2), sc, l, group, live);
                else
                    store_row<LPR, CACHE, false>(x, (is_v ? p.c.v : p.c.k) + pg * p.c.sp + hk * p.c.sh + slot * p.c.ss, sc, l,
                                                 group, live);
            }
        }
    }
}

// ---- read: one row group of LPR lanes per (row, share of the kv-heads)
template <int CACHE>
__device__ __forceinline__ void decode8(uint2 raw, float s, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t w = i ? raw.y : raw.x;
        if (CACHE == CACHE_E4M3 || CACHE == CACHE_E4M3_V4) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * j)), __NV_E4M3);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hr));
                x[4 * i + 2 * j] = f.x * s;
                x[4 * i + 2 * j + 1] = f.y * s;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[4 * i + j] = (float)(int)(int8_t)(w >> (8 * j)) * s;
        }
    }
}
__device__ __forceinline__ void decode4(uint32_t w, float s, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)((int)((w >> (4 * i)) & 15u) - 8) * s;
}

template <int D, int CACHE>
__global__ void __launch_bounds__(THREADS) read_tokens_kernel(const ReadParams p) {
    constexpr int LPR = D / 8;
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, l = lane & (LPR - 1);
    const unsigned warp = blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    const int split = (int)(warp % (unsigned)p.head_splits);
    const long long t = (long long)(warp / (unsigned)p.head_splits) * (32 / LPR) + lane / LPR;
    const bool in = t < p.T;
    const int s = sequence_of<LPR>(p.cu, p.B, in ? t : (long long)p.T, l, 0xffffffffu);
    if (!in || s >= p.B) return;             // rows behind the last sequence are left alone ...
    int slot = 0;
    const int start = p.starts ? p.starts[SKV_INDEX(s, p.B)] : 0;   // (asked for with the offset, not behind it)
    const long long i = t - p.cu[SKV_INDEX(s, p.B)], pos = start + i;
    if (i < 0) return;                       // ... and those before the first
    const int page = page_of(p.c, s, pos, slot);
    const long long pg = page < 0 ? 0 : page;
    const int h_end = min(p.Hkv, (split + 1) * p.heads_per_split);
    for (int h = split * p.heads_per_split; h < h_end; ++h) {
        float k[8], v[8];
        if constexpr (CACHE == CACHE_KV4) {
            const uint8_t* rec = p.c.k + pg * p.c.sp + h * p.c.sh;
            const int w = l >> 2, c = l & 3;
            const uint32_t kw = *reinterpret_cast<const uint32_t*>(rec + kv4_place(slot) * (D / 2) + c * (D / 8) + w * 4);
            const uint8_t* vr = rec + kv4_v_row<D>(slot) + 2 * c * (D / 2) + 2 * w;
            const uint32_t vw = (uint32_t)*reinterpret_cast<const uint16_t*>(vr) |
                                ((uint32_t)*reinterpret_cast<const uint16_t*>(vr + D / 2) << 16);
            const uint16_t* sc = reinterpret_cast<const uint16_t*>(rec + kv4_scales<D>(slot)) + w;
            decode4(kw, bf16_bits_to_f(sc[0]), k);
            decode4(vw, bf16_bits_to_f(sc[D / 32]), v);
        } else {
            const float ks = p.c.ks[pg * p.c.csp + h * p.c.csh + slot], vs = p.c.vs[pg * p.c.csp + h * p.c.csh + slot];
            decode8<CACHE>(*reinterpret_cast<const uint2*>(p.c.k + pg * p.c.sp + h * p.c.sh + slot * p.c.ss + l * 8), ks, k);
            if (CACHE == CACHE_E4M3_V4 || CACHE == CACHE_I8_V4)
                decode4(*reinterpret_cast<const uint32_t*>(p.c.v + pg * p.c.sp + h * p.c.sh + slot * (D / 2) + l * 4), vs, v);
            else
                decode8<CACHE>(*reinterpret_cast<const uint2*>(p.c.v + pg * p.c.sp + h * p.c.sh + slot * p.c.ss + l * 8), vs, v);
        }
        const long long o = ((long long)SKV_INDEX(t, p.T) * p.Hkv + SKV_INDEX(h, p.Hkv)) * D + l * 8;
        const bool bf = p.out_bf16;
        uint4 a = make_uint4(pack16(k[0], k[1], bf), pack16(k[2], k[3], bf), pack16(k[4], k[5], bf), pack16(k[6], k[7], bf));
        uint4 c = make_uint4(pack16(v[0], v[1], bf), pack16(v[2], v[3], bf), pack16(v[4], v[5], bf), pack16(v[6], v[7], bf));
        if (page < 0) a = c = make_uint4(0u, 0u, 0u, 0u);   // a position the cache has no page for reads as zero
        *reinterpret_cast<uint4*>(static_cast<__half*>(p.k_out) + o) = a;
        *reinterpret_cast<uint4*>(static_cast<__half*>(p.v_out) + o) = c;
    }
}

// Checks and addressing shared by the two entry points; `cache` receives the kernel's cache kind.
static int make_pools(const char* who, Pools* c, int* cache, void* k_pool, void* v_pool, float* k_scale_pool, float* v_scale_pool,
                      const int* page_table, int D, int kv_dtype, int page_size, int max_pages, int num_pages,
                      long long pool_stride_page, long long pool_stride_head, long long pool_stride_slot,
                      long long scale_stride_page, long long scale_stride_head, int* status) {
    const bool v4 = (kv_dtype & SKV_V_INT4) != 0;
    kv_dtype &= ~SKV_V_INT4;
    if (!k_pool) return fail(SKV_ERR_BAD_ARG, "%s: null pool", who);
    if (page_size <= 0 || max_pages <= 0 || num_pages <= 0) return fail(SKV_ERR_BAD_ARG, "%s: sizes must be positive", who);
    unsigned long long bits = reinterpret_cast<uintptr_t>(k_pool) | (unsigned long long)(pool_stride_page | pool_stride_head);
    if (kv_dtype == SKV_KV_INT4 && !v4) {
        if (D != 64 && D != 128) return fail(SKV_ERR_UNSUPPORTED, "%s: 4-bit caches hold head dims 64 and 128 (got %d)", who, D);
        if (page_size != KV4_PAGE) return fail(SKV_ERR_UNSUPPORTED, "%s: 4-bit page records hold 16 tokens", who);
        *cache = CACHE_KV4;
    } else {
        if (kv_dtype != SKV_KV_I8 && kv_dtype != SKV_KV_E4M3) return fail(SKV_ERR_UNSUPPORTED, "%s: kv_dtype %d", who, kv_dtype);
        if (D != 128) return fail(SKV_ERR_UNSUPPORTED, "%s: 8-bit caches hold head dim 128 (got %d)", who, D);
        if (!v_pool || !k_scale_pool || !v_scale_pool) return fail(SKV_ERR_BAD_ARG, "%s: null pool", who);
        const bool e4 = kv_dtype == SKV_KV_E4M3;
        *cache = v4 ? (e4 ? CACHE_E4M3_V4 : CACHE_I8_V4) : (e4 ? CACHE_E4M3 : CACHE_I8);
        bits |= reinterpret_cast<uintptr_t>(v_pool) | (unsigned long long)pool_stride_slot;
        if ((reinterpret_cast<uintptr_t>(k_scale_pool) | reinterpret_cast<uintptr_t>(v_scale_pool)) & 3)
            return fail(SKV_ERR_BAD_ARG, "%s: scale pools must be 4-byte aligned", who);
    }
    if (bits & 15) return fail(SKV_ERR_BAD_ARG, "%s: pools and their strides must be multiples of 16 bytes", who);
    c->k = static_cast<uint8_t*>(k_pool); c->v = static_cast<uint8_t*>(v_pool);
    c->ks = k_scale_pool; c->vs = v_scale_pool;
    c->sp = pool_stride_page; c->sh = pool_stride_head; c->ss = pool_stride_slot;
    c->csp = scale_stride_page; c->csh = scale_stride_head;
    c->page_table = page_table; c->max_pages = max_pages; c->num_pages = num_pages; c->page_size = page_size;
    c->status = status;
    return SKV_OK;
}

// A block's heads (a multiple of the four that its warps take at a time): all of them for long prompts, whose blocks are many;
// shares of them while there are fewer than four blocks an SM.
static long long split_blocks(long long tiles, int heads, int device, int* splits, int* per) {
    const long long want = (long long)sm_count(device) * 4;
    const int fours = (heads + 3) / 4;
    long long s = (want + tiles - 1) / tiles;
    s = s < 1 ? 1 : s > fours ? fours : s;
    *per = 4 * (int)((fours + s - 1) / s);
    *splits = (heads + *per - 1) / *per;
    return tiles * *splits;
}

// Heads are split over warps until the machine is full.
static long long split_heads(long long warps, int heads, int device, int* splits, int* per) {
    const long long want = (long long)sm_count(device) * 32;
    long long s = (want + warps - 1) / warps;
    s = s < 1 ? 1 : s > heads ? heads : s;
    *per = (int)((heads + s - 1) / s);
    *splits = (heads + *per - 1) / *per;
    return warps * *splits;
}

template <typename T, int D>
static auto append_kernel(int cache) {
    if constexpr (D == 64) return append_tokens_kernel<T, 64, CACHE_KV4>;
    else switch (cache) {
        case CACHE_KV4: return append_tokens_kernel<T, D, CACHE_KV4>;
        case CACHE_E4M3: return append_tokens_kernel<T, D, CACHE_E4M3>;
        case CACHE_I8: return append_tokens_kernel<T, D, CACHE_I8>;
        case CACHE_E4M3_V4: return append_tokens_kernel<T, D, CACHE_E4M3_V4>;
        default: return append_tokens_kernel<T, D, CACHE_I8_V4>;
    }
}
template <int D>
static auto read_kernel(int cache) {
    if constexpr (D == 64) return read_tokens_kernel<64, CACHE_KV4>;
    else switch (cache) {
        case CACHE_KV4: return read_tokens_kernel<D, CACHE_KV4>;
        case CACHE_E4M3: return read_tokens_kernel<D, CACHE_E4M3>;
        case CACHE_I8: return read_tokens_kernel<D, CACHE_I8>;
        case CACHE_E4M3_V4: return read_tokens_kernel<D, CACHE_E4M3_V4>;
        default: return read_tokens_kernel<D, CACHE_I8_V4>;
    }
}

}  // namespace tok
}  // namespace skv

using namespace skv;

extern "C" {

int skv_append_tokens(const void* qkv, int qkv_is_bf16, long long qkv_stride, void* q_out, int q_out_is_bf16,
                      const unsigned long long* rope_freqs, int rotary_dim, int interleaved, double rope_factor,
                      const void* positions, int positions_are_64, const int* cu_new, const int* page_table,
                      const int* seq_lens, void* k_pool, void* v_pool, float* k_scale_pool, float* v_scale_pool, int T, int B,
                      int Hq, int Hkv, int D, int kv_dtype, int page_size, int max_pages, int num_pages,
                      long long pool_stride_page, long long pool_stride_head, long long pool_stride_slot,
                      long long scale_stride_page, long long scale_stride_head, int* status, int device, void* stream) {
    if (T < 0 || B <= 0 || Hq < 0 || Hkv <= 0) return fail(SKV_ERR_BAD_ARG, "skv_append_tokens: bad sizes");
    tok::AppendParams p;
    int cache;
    const int rc = tok::make_pools("skv_append_tokens", &p.c, &cache, k_pool, v_pool, k_scale_pool, v_scale_pool, page_table, D,
                                   kv_dtype, page_size, max_pages, num_pages, pool_stride_page, pool_stride_head,
                                   pool_stride_slot, scale_stride_page, scale_stride_head, status);
    if (rc) return rc;
    if (rope_freqs && (rotary_dim <= 0 || rotary_dim > D || rotary_dim % (interleaved ? 8 : 16)))
        return fail(SKV_ERR_UNSUPPORTED, "skv_append_tokens: rotary_dim %d must be a multiple of %d up to %d", rotary_dim,
                    interleaved ? 8 : 16, D);
    if (T == 0) return SKV_OK;
    if (!qkv || !seq_lens || (Hq && !q_out)) return fail(SKV_ERR_BAD_ARG, "skv_append_tokens: null pointer");
    if (!cu_new && T != B) return fail(SKV_ERR_BAD_ARG, "skv_append_tokens: %d rows for %d sequences need cu_new", T, B);
    if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | (unsigned long long)qkv_stride * 2) & 15)
        return fail(SKV_ERR_BAD_ARG, "skv_append_tokens: rows must start on 16-byte boundaries");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(SKV_ERR_CUDA, "cannot switch to device %d", device);
    p.qkv = qkv; p.q_out = q_out; p.freqs = rope_freqs; p.positions = positions; p.cu_new = cu_new; p.seq_lens = seq_lens;
    p.qkv_stride = qkv_stride;
    p.T = T; p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.R = rotary_dim; p.interleaved = interleaved; p.pos64 = positions_are_64;
    p.q_bf16 = q_out_is_bf16; p.factor = rope_factor;
    const int rows = 256 / D;   // per block
    const long long blocks = tok::split_blocks(((long long)T + rows - 1) / rows, Hq + 2 * Hkv, device, &p.head_splits, &p.heads_per_split);
    if (blocks > 0x3fffffff) return fail(SKV_ERR_UNSUPPORTED, "skv_append_tokens: too many rows for one launch");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)blocks), block(tok::THREADS);
    if (D == 64)
        SKV_CUDA_TRY(launch_pdl(qkv_is_bf16 ? tok::append_kernel<__nv_bfloat16, 64>(cache) : tok::append_kernel<__half, 64>(cache), grid, block, 0, st, p));
    else
        SKV_CUDA_TRY(launch_pdl(qkv_is_bf16 ? tok::append_kernel<__nv_bfloat16, 128>(cache) : tok::append_kernel<__half, 128>(cache), grid, block, 0, st, p));
    SKV_CUDA_TRY(cudaGetLastError());
    return SKV_OK;
}

int skv_read_tokens(const void* k_pool, const void* v_pool, const float* k_scale_pool, const float* v_scale_pool,
                    const int* page_table, const int* cu, const int* starts, void* k_out, void* v_out, int out_is_bf16, int T,
                    int B, int Hkv, int D, int kv_dtype, int page_size, int max_pages, int num_pages,
                    long long pool_stride_page, long long pool_stride_head, long long pool_stride_slot,
                    long long scale_stride_page, long long scale_stride_head, int* status, int device, void* stream) {
    if (T < 0 || B <= 0 || Hkv <= 0) return fail(SKV_ERR_BAD_ARG, "skv_read_tokens: bad sizes");
    tok::ReadParams p;
    int cache;
    const int rc = tok::make_pools("skv_read_tokens", &p.c, &cache, const_cast<void*>(k_pool), const_cast<void*>(v_pool),
                                   const_cast<float*>(k_scale_pool), const_cast<float*>(v_scale_pool), page_table, D, kv_dtype,
                                   page_size, max_pages, num_pages, pool_stride_page, pool_stride_head, pool_stride_slot,
                                   scale_stride_page, scale_stride_head, status);
    if (rc) return rc;
    if (T == 0) return SKV_OK;
    if (!cu || !k_out || !v_out) return fail(SKV_ERR_BAD_ARG, "skv_read_tokens: null pointer");
    if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15)
        return fail(SKV_ERR_BAD_ARG, "skv_read_tokens: outputs must be 16-byte aligned");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(SKV_ERR_CUDA, "cannot switch to device %d", device);
    p.k_out = k_out; p.v_out = v_out; p.cu = cu; p.starts = starts;
    p.T = T; p.B = B; p.Hkv = Hkv; p.out_bf16 = out_is_bf16;
    const int rows = 256 / D;
    const long long warps = tok::split_heads(((long long)T + rows - 1) / rows, Hkv, device, &p.head_splits, &p.heads_per_split);
    const long long blocks = (warps + tok::THREADS / 32 - 1) / (tok::THREADS / 32);
    if (blocks > 0x3fffffff) return fail(SKV_ERR_UNSUPPORTED, "skv_read_tokens: too many rows for one launch");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)blocks), block(tok::THREADS);
    if (D == 64) SKV_CUDA_TRY(launch_pdl(tok::read_kernel<64>(cache), grid, block, 0, st, p));
    else SKV_CUDA_TRY(launch_pdl(tok::read_kernel<128>(cache), grid, block, 0, st, p));
    SKV_CUDA_TRY(cudaGetLastError());
    return SKV_OK;
}

}  // extern "C"

SKV_BOUNDS_GETTER(skv_debug_bounds_kv_tokens)
