// Rotary positions of query and key rows, and their gradient.
//
// No reference counterpart: the reference leaves the rotation to Hugging Face (benchmarks/llama_integration_benchmark.py
// :152-160); skv_rope_quant_append rotates one token per sequence on its way into the cache, rotate-half and over the
// whole head only.
//
// Pair i < R/2 of a row is (i, i + R/2) (half layout) or (2i, 2i + 1) (interleaved) and becomes
//     (x cos a - y sin a, y cos a + x sin a) * factor,   a = position * f_i;   channels from R on are copied.
// The gradient of the rotation is the same with -a (adjoint).
//
// Angles: f_i comes as the 64-bit fixed-point fraction F_i = round(f_i / (2 pi) * 2^64) of a turn per position, so
// position * F_i mod 2^64 is the angle's place in its turn, exact but for the rounding of f_i itself: far positions
// (2^20 and beyond, where a 32-bit product is off by a tenth of a radian) cost two integer multiplications and need no
// range reduction.
//
// Bound: HBM, one read and one write of every row.  A thread keeps one vector of one token's channels and takes it from U
// heads, all asked for at once; its block works out the sines and cosines of its tokens once, in shared memory, while the
// rows are on their way, and every thread takes those of its channels to registers.
#include <cuda_bf16.h>

#include "skv_common.cuh"
#include "skv_kv4.cuh"

namespace skv {
namespace rot {

constexpr int MAX_THREADS = 256;

struct Params {
    const void* src[2];         // q, k (k may be absent)
    void* dst[2];
    long long st[2], sh[2];     // element strides of token and head, source ...
    long long dt[2], dh[2];     // ... and destination
    const void* positions;
    const unsigned long long* freqs;   // [R / 2] turns per position, 64-bit fixed point
    int pos64, T, Hq, H, D, R;
    int turn_units, units;      // vectors per row: the turned ones, and with those that are copied
    int width;                  // vectors of a row that a block's threads hold at a time: units, where they fit
    int tokens, lanes;          // a block's tokens, and threads that share one vector's heads; tokens * width * lanes threads
    double factor;
    float sign;
};

// E elements of T as one access of up to 16 bytes (LOOSE: aligned to an element only)
template <typename T, int E, bool LOOSE>
struct alignas(LOOSE ? sizeof(T) : E * sizeof(T)) Vec {
    T v[E];
};

// 16-bit channels are taken from and put into their words, two at a time
template <typename T, int E>
__device__ __forceinline__ void to_floats(const T (&v)[E], float (&x)[E]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = v[i];
    } else if constexpr (E == 1) {
        x[0] = static_cast<float>(v[0]);
    } else {
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            uint32_t w;
            if constexpr (E == 2) w = (uint32_t)reinterpret_cast<const uint16_t*>(v)[0] | ((uint32_t)reinterpret_cast<const uint16_t*>(v)[1] << 16);
            else w = reinterpret_cast<const uint32_t*>(v)[i];
            if constexpr (__is_same(T, __half)) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
                x[2 * i] = f.x; x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w << 16); x[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
            }
        }
    }
}
template <typename T, int E>
__device__ __forceinline__ void from_floats(const float (&x)[E], T (&v)[E]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = x[i];
    } else if constexpr (E == 1) {
        if constexpr (__is_same(T, __half)) v[0] = __float2half_rn(x[0]);
        else v[0] = __float2bfloat16_rn(x[0]);
    } else {
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
            uint32_t w;
            if constexpr (__is_same(T, __half)) {
                w = pack_half2(x[2 * i], x[2 * i + 1]);
            } else {
                const __nv_bfloat162 f = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                w = *reinterpret_cast<const uint32_t*>(&f);
            }
            if constexpr (E == 2) {
                reinterpret_cast<uint16_t*>(v)[0] = (uint16_t)w;
                reinterpret_cast<uint16_t*>(v)[1] = (uint16_t)(w >> 16);
            } else {
                reinterpret_cast<uint32_t*>(v)[i] = w;
            }
        }
    }
}

// A unit of a row: half layout, E channels of the first half and the E that belong to them; interleaved, E channels in a row
// (E / 2 pairs); behind the turned part E channels in a row, copied.
// 64 registers, four full blocks an SM: 28.3 us for that prompt (5.9 TB/s, 0.90 of a copy), 31.0 with 80.
template <typename T, int E, bool INTER>
__global__ void __launch_bounds__(MAX_THREADS, 4) rotary_kernel(const Params p) {
    constexpr int NP = INTER ? E / 2 : E;             // pairs of a unit
    constexpr int U = INTER ? 8 : 4;                  // heads in flight per thread
    constexpr bool LOOSE = INTER && E == 2;           // channels fetched one by one: no alignment, and rows of an odd length
    using V = Vec<T, E, LOOSE>;
    extern __shared__ float2 table[];                 // (cos, sin): [token][pair of the unit][unit]
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * p.tokens, nt = min(p.tokens, p.T - t0);
    // this thread: vector `first`, `first + width`, ... of token tt, heads `lane`, `lane + lanes`, ...
    const int first = threadIdx.x % p.width, rest = threadIdx.x / p.width;
    const int lane = rest % p.lanes, tt = rest / p.lanes;
    const bool live = tt < nt;
    const long long t = SKV_INDEX(t0 + (live ? tt : 0), p.T);

    V a[U], b[U];
    auto channel = [&](int u) { return u < p.turn_units ? u * E : p.R + (u - p.turn_units) * E; };
    auto load = [&](int u, int h0) {
        const int c = SKV_INDEX(channel(u), p.D - (LOOSE ? 0 : E - 1));
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int h = min(h0 + k * p.lanes, p.H - 1), w = h >= p.Hq;   // (past the last head: that one again, not stored)
            const T* s = static_cast<const T*>(p.src[w]) + t * p.st[w] + (h - (w ? p.Hq : 0)) * p.sh[w] + c;
            if constexpr (LOOSE) {
                a[k].v[0] = s[0];
                a[k].v[1] = s[c + 1 < p.D ? 1 : 0];
            } else {
                a[k] = *reinterpret_cast<const V*>(s);
            }
            if (!INTER) b[k] = *reinterpret_cast<const V*>(u < p.turn_units ? s + p.R / 2 : s);
        }
    };
    // the block's angles: what they need is asked for first, then the rows, and the sines are worked out while those come
    const int pairs = p.turn_units * NP, angles = nt * pairs;
    auto angle = [&](int i, long long& pos, unsigned long long& f) {
        const int x = i / pairs, t = SKV_INDEX(t0 + x, p.T);
        pos = p.pos64 ? static_cast<const long long*>(p.positions)[t] : (long long)static_cast<const int*>(p.positions)[t];
        f = p.freqs[SKV_INDEX(i - x * pairs, p.R / 2)];
    };
    auto write = [&](int i, long long pos, unsigned long long f) {
        const int x = i / pairs, r = i - x * pairs;
        float2 cs = rotary_cos_sin(pos, f, p.factor);
        cs.y *= p.sign;
        table[SKV_INDEX((x * NP + r % NP) * p.turn_units + r / NP, p.tokens * NP * p.turn_units)] = cs;
    };
    {
        long long pos = 0;
        unsigned long long f = 0;
        if (threadIdx.x < angles) angle(threadIdx.x, pos, f);
        load(first, lane);
        if (threadIdx.x < angles) write(threadIdx.x, pos, f);
        for (int i = threadIdx.x + blockDim.x; i < angles; i += blockDim.x) {
            angle(i, pos, f);
            write(i, pos, f);
        }
    }
    __syncthreads();
    if (!live) return;
    for (int u = first; u < p.units; u += p.width) {
        const bool turned = u < p.turn_units;
        float cs[NP], sn[NP];
        if (turned) {
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const float2 f = table[SKV_INDEX((tt * NP + i) * p.turn_units + u, p.tokens * NP * p.turn_units)];
                cs[i] = f.x;
                sn[i] = f.y;
            }
        }
        const int c = SKV_INDEX(channel(u), p.D - (LOOSE ? 0 : E - 1));
        for (int h0 = lane; h0 < p.H; h0 += U * p.lanes) {
            if (u != first || h0 != lane) load(u, h0);
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int h = h0 + k * p.lanes;
                if (h >= p.H) break;
                V lo = a[k], hi;
                if (turned) {
                    float x[E], y[E];
                    to_floats(a[k].v, x);
                    if constexpr (INTER) {
#pragma unroll
                        for (int i = 0; i < NP; ++i) rotary_turn(x[2 * i], x[2 * i + 1], sn[i], cs[i], y[2 * i], y[2 * i + 1]);
                        from_floats(y, lo.v);
                    } else {
                        float m[E], n[E];
                        to_floats(b[k].v, y);
#pragma unroll
                        for (int i = 0; i < NP; ++i) rotary_turn(x[i], y[i], sn[i], cs[i], m[i], n[i]);
                        from_floats(m, lo.v);
                        from_floats(n, hi.v);
                    }
                }
                const int w = h >= p.Hq;
                T* d = static_cast<T*>(p.dst[w]) + t * p.dt[w] + (h - (w ? p.Hq : 0)) * p.dh[w] + c;
                if constexpr (LOOSE) {
                    d[0] = lo.v[0];
                    if (c + 1 < p.D) d[1] = lo.v[1];
                } else {
                    *reinterpret_cast<V*>(d) = lo;
                }
                if constexpr (!INTER) {
                    if (turned) *reinterpret_cast<V*>(d + p.R / 2) = hi;
                }
            }
        }
    }
}

static long long magnitude(long long x) { return x < 0 ? -x : x; }

// Whether two of the rows i * a + j * b (i < n, j < m), `width` long, share memory.
static bool rows_share(long long n, long long m, long long a, long long b, long long width) {
    a = magnitude(a); b = magnitude(b);                 // (counting i or j from the other end changes no distance)
    if ((n > 1 && a < width) || (m > 1 && b < width)) return true;
    if (n <= 1 || m <= 1 || b >= (n - 1) * a + width || a >= (m - 1) * b + width) return false;
    for (long long j = 1; j < m; ++j)                   // neither lies whole in a step of the other: the nearest steps of i to j's
        for (long long i = j * b / a; i <= j * b / a + 1; ++i)
            if (i < n && magnitude(i * a - j * b) < width) return true;
    return false;
}

// The same for a row of q (i * aq + j * bq, j < Hq) and one of k (delta + i * ak + j * bk, j < Hk).  Views whose spans meet are
// looked into where they have one token stride; others count as sharing.
static bool views_share(long long T, long long Hq, long long aq, long long bq, long long Hk, long long ak, long long bk,
                        long long delta, long long width) {
    auto low = [](long long n, long long s) { return s < 0 ? (n - 1) * s : 0; };
    auto high = [](long long n, long long s) { return s > 0 ? (n - 1) * s : 0; };
    const long long q0 = low(Hq, bq), q1 = high(Hq, bq) + width, k0 = delta + low(Hk, bk), k1 = delta + high(Hk, bk) + width;
    if (q0 + low(T, aq) >= k1 + high(T, ak) || k0 + low(T, ak) >= q1 + high(T, aq)) return false;
    if (T > 1 && aq != ak) return true;
    const long long a = T > 1 ? magnitude(aq) : 0;
    const bool apart = q0 >= k1 || k0 >= q1;            // within a token
    if (apart && (a == 0 || (q1 > k1 ? q1 : k1) - (q0 < k0 ? q0 : k0) <= a)) return false;
    for (long long j = 0; j < Hq; ++j)
        for (long long k = 0; k < Hk; ++k) {
            const long long x = magnitude(delta + k * bk - j * bq), i = a ? x / a : 0;
            if ((i < T && x - i * a < width) || (a && i + 1 < T && (i + 1) * a - x < width)) return true;
        }
    return false;
}

template <typename T, int E, bool INTER>
static int launch(Params& p, int tail, cudaStream_t st) {
    constexpr int NP = INTER ? E / 2 : E, U = INTER ? 8 : 4;
    p.turn_units = INTER ? p.R / E : p.R / 2 / E;
    p.units = p.turn_units + (tail + E - 1) / E;
    // Threads for every vector of a row, enough of them side by side that each takes at most U heads where a block can hold
    // them, and as many tokens as fill a block to about 160 threads (a prompt of 8192 tokens, 40 heads of 128 in bf16: 31.2 us
    // with 96 threads, 28.3 with 160, 36 with 256).
    p.width = p.units < MAX_THREADS ? p.units : MAX_THREADS;
    p.lanes = (p.H + U - 1) / U;
    if (p.lanes * p.width > MAX_THREADS) p.lanes = MAX_THREADS / p.width;
    p.tokens = 160 / (p.lanes * p.width);
    if (p.tokens < 1) p.tokens = 1;
    if (p.tokens > p.T) p.tokens = p.T;
    const long long blocks = ((long long)p.T + p.tokens - 1) / p.tokens;
    const size_t smem = (size_t)p.tokens * p.turn_units * NP * sizeof(float2);
    if (smem > 48 * 1024) return fail(SKV_ERR_UNSUPPORTED, "skv_rotary: rotary_dim %d is not supported", p.R);
    SKV_CUDA_TRY(launch_pdl(rotary_kernel<T, E, INTER>, dim3((unsigned)blocks), dim3(p.tokens * p.width * p.lanes), smem, st, p));
    SKV_CUDA_TRY(cudaGetLastError());
    return SKV_OK;
}

template <typename T>
static int launch_vec(int vec, Params& p, int tail, int interleaved, cudaStream_t st) {
    if (interleaved) {
        if (sizeof(T) == 2 && vec >= 8) return launch<T, sizeof(T) == 2 ? 8 : 4, true>(p, tail, st);
        if (vec >= 4) return launch<T, 4, true>(p, tail, st);
        return launch<T, 2, true>(p, tail, st);
    }
    if (sizeof(T) == 2 && vec >= 8) return launch<T, sizeof(T) == 2 ? 8 : 4, false>(p, tail, st);
    if (vec >= 4) return launch<T, 4, false>(p, tail, st);
    if (vec >= 2) return launch<T, 2, false>(p, tail, st);
    return launch<T, 1, false>(p, tail, st);
}

}  // namespace rot
}  // namespace skv

using namespace skv;

extern "C" int skv_rotary(const void* q, const void* k, void* q_out, void* k_out, int dtype, const void* positions,
                          int positions_are_64, const unsigned long long* freqs, int T, int Hq, int Hk, int D,
                          int rotary_dim, int interleaved, double rope_factor, int adjoint,
                          long long q_stride_t, long long q_stride_h, long long k_stride_t, long long k_stride_h,
                          long long q_out_stride_t, long long q_out_stride_h, long long k_out_stride_t,
                          long long k_out_stride_h, int device, void* stream) {
    if (T < 0 || Hq < 0 || Hk < 0 || Hq + Hk <= 0 || D <= 0) return fail(SKV_ERR_BAD_ARG, "skv_rotary: bad sizes");
    if (T == 0) return SKV_OK;
    if ((Hq && (!q || !q_out)) || (Hk && (!k || !k_out)) || !positions || !freqs)
        return fail(SKV_ERR_BAD_ARG, "skv_rotary: null pointer");
    if (rotary_dim <= 0 || rotary_dim > D || rotary_dim % 2)
        return fail(SKV_ERR_BAD_ARG, "skv_rotary: rotary_dim %d must be even and in 2..%d", rotary_dim, D);
    if (dtype < 0 || dtype > 2) return fail(SKV_ERR_UNSUPPORTED, "skv_rotary: dtype %d is not fp16, bf16 or fp32", dtype);
    // Rows that share memory would be turned by several threads at once: views with a repeated or shortened stride as
    // destination (an expanded or sliding view rotated in place), or heads that q and k have in common.
    const long long esz = dtype == 2 ? 4 : 2;
    if ((Hq && rot::rows_share(T, Hq, q_out_stride_t, q_out_stride_h, D)) || (Hk && rot::rows_share(T, Hk, k_out_stride_t, k_out_stride_h, D)) ||
        (Hq && Hk && rot::views_share(T, Hq, q_out_stride_t * esz, q_out_stride_h * esz, Hk, k_out_stride_t * esz, k_out_stride_h * esz,
                                      static_cast<const char*>(k_out) - static_cast<const char*>(q_out), D * esz)))
        return fail(SKV_ERR_BAD_ARG, "skv_rotary: rows of the outputs overlap");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(SKV_ERR_CUDA, "cannot switch to device %d", device);
    rot::Params p;
    p.src[0] = Hq ? q : k; p.src[1] = Hk ? k : q;
    p.dst[0] = Hq ? q_out : k_out; p.dst[1] = Hk ? k_out : q_out;
    p.st[0] = q_stride_t; p.sh[0] = q_stride_h; p.st[1] = k_stride_t; p.sh[1] = k_stride_h;
    p.dt[0] = q_out_stride_t; p.dh[0] = q_out_stride_h; p.dt[1] = k_out_stride_t; p.dh[1] = k_out_stride_h;
    p.positions = positions; p.pos64 = positions_are_64; p.freqs = freqs;
    p.T = T; p.Hq = Hq; p.H = Hq + Hk; p.D = D; p.R = rotary_dim;
    p.factor = rope_factor; p.sign = adjoint ? -1.f : 1.f;

    // The widest vector that the row's parts and every pointer and stride allow: 16 bytes where a layout is an ordinary one,
    // down to single elements for odd rotary widths or views (interleaved: to pairs, fetched one by one).
    int vec = 16 / (int)esz;
    bool same = true;   // nothing behind the rotated part to copy when a row is rotated in place
    for (int w = 0; w < 2; ++w) {
        if (!(w ? Hk : Hq)) continue;
        same = same && p.src[w] == p.dst[w] && p.st[w] == p.dt[w] && p.sh[w] == p.dh[w];
        const unsigned long long bits = (unsigned long long)(p.st[w] | p.sh[w] | p.dt[w] | p.dh[w]) * esz |
                                        reinterpret_cast<uintptr_t>(p.src[w]) | reinterpret_cast<uintptr_t>(p.dst[w]);
        if (bits % esz) return fail(SKV_ERR_BAD_ARG, "skv_rotary: pointers must be aligned to their elements");
        while (bits % (vec * esz)) vec /= 2;
    }
    const int tail = same ? 0 : D - rotary_dim;
    const int part = interleaved ? rotary_dim : rotary_dim / 2;
    while (part % vec || tail % vec) vec /= 2;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == 0) return rot::launch_vec<__half>(vec, p, tail, interleaved, st);
    if (dtype == 1) return rot::launch_vec<__nv_bfloat16>(vec, p, tail, interleaved, st);
    return rot::launch_vec<float>(vec, p, tail, interleaved, st);
}

SKV_BOUNDS_GETTER(skv_debug_bounds_rotary)
