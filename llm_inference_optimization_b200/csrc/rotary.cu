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
// range reduction.  The upper 32 bits go to sincospif.
//
// Bound: HBM, one read and one write of every row.  A thread owns VEC frequencies of one token and walks over heads, so
// that sines and cosines are computed once for the heads of its share; U rows are loaded before the first is used.
#include <cuda_bf16.h>

#include "skv_common.cuh"
#include "skv_kv4.cuh"

namespace skv {
namespace rot {

constexpr int THREADS = 128;

struct Params {
    const void* src[2];         // q, k (k may be null with heads[1] == 0)
    void* dst[2];
    long long st[2], sh[2];     // element strides of token and head, source ...
    long long dt[2], dh[2];     // ... and destination
    const void* positions;
    const unsigned long long* freqs;   // [R / 2] turns per position, 64-bit fixed point
    int pos64, T, Hq, H, R, tail_units, units, head_splits, heads_per_split;
    float factor, sign;
};

// N elements of T as one load or store of up to 16 bytes
template <typename T, int N>
struct alignas(N * sizeof(T)) Vec {
    T v[N];
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float x, float& y) { y = x; }
__device__ __forceinline__ void from_f(float x, __half& y) { y = __float2half_rn(x); }
__device__ __forceinline__ void from_f(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }

template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(THREADS) rotary_kernel(const Params p) {
    constexpr int U = sizeof(T) * VEC >= 16 ? 4 : 2;   // rows in flight
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const unsigned item = blockIdx.x * THREADS + threadIdx.x;   // (the launcher keeps the count below 2^31)
    const int unit = (int)(item % (unsigned)p.units);
    const unsigned rest = item / (unsigned)p.units;
    const int split = (int)(rest % (unsigned)p.head_splits);
    const long long t = rest / (unsigned)p.head_splits;
    if (t >= p.T) return;
    const int h_begin = split * p.heads_per_split, h_end = min(p.H, h_begin + p.heads_per_split);
    const int nrot = p.units - p.tail_units;

    if (unit >= nrot) {   // a vector of the channels behind the rotated part
        const int d = p.R + (unit - nrot) * VEC;
        for (int h = h_begin; h < h_end; ++h) {
            const int w = h >= p.Hq;
            const int hh = h - (w ? p.Hq : 0);
            *reinterpret_cast<Vec<T, VEC>*>(static_cast<T*>(p.dst[w]) + t * p.dt[w] + hh * p.dh[w] + d) =
                *reinterpret_cast<const Vec<T, VEC>*>(static_cast<const T*>(p.src[w]) + t * p.st[w] + hh * p.sh[w] + d);
        }
        return;
    }

    const long long pos = p.pos64 ? static_cast<const long long*>(p.positions)[t]
                                  : (long long)static_cast<const int*>(p.positions)[t];
    float cs[VEC], sn[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        rotary_sincos(pos, p.freqs[unit * VEC + i], sn[i], cs[i]);
        sn[i] *= p.sign * p.factor;
        cs[i] *= p.factor;
    }
    const int c0 = INTER ? unit * 2 * VEC : unit * VEC;
    const int c1 = INTER ? c0 + VEC : c0 + p.R / 2;
    for (int h0 = h_begin; h0 < h_end; h0 += U) {
        Vec<T, VEC> a[U], b[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = min(h0 + u, h_end - 1);   // (a row past the end is loaded twice and not stored)
            const int w = h >= p.Hq;
            const T* s = static_cast<const T*>(p.src[w]) + t * p.st[w] + (h - (w ? p.Hq : 0)) * p.sh[w];
            a[u] = *reinterpret_cast<const Vec<T, VEC>*>(s + c0);
            b[u] = *reinterpret_cast<const Vec<T, VEC>*>(s + c1);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + u;
            if (h >= h_end) break;
            const int w = h >= p.Hq;
            Vec<T, VEC> x, y;
            if (INTER) {   // a, b together hold 2 VEC neighbouring channels
                T e[2 * VEC], r[2 * VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) { e[i] = a[u].v[i]; e[VEC + i] = b[u].v[i]; }
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float m, n;
                    rotary_turn(to_f(e[2 * i]), to_f(e[2 * i + 1]), sn[i], cs[i], m, n);
                    from_f(m, r[2 * i]);
                    from_f(n, r[2 * i + 1]);
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) { x.v[i] = r[i]; y.v[i] = r[VEC + i]; }
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float m, n;
                    rotary_turn(to_f(a[u].v[i]), to_f(b[u].v[i]), sn[i], cs[i], m, n);
                    from_f(m, x.v[i]);
                    from_f(n, y.v[i]);
                }
            }
            T* d = static_cast<T*>(p.dst[w]) + t * p.dt[w] + (h - (w ? p.Hq : 0)) * p.dh[w];
            *reinterpret_cast<Vec<T, VEC>*>(d + c0) = x;
            *reinterpret_cast<Vec<T, VEC>*>(d + c1) = y;
        }
    }
}

template <typename T, int VEC>
static int launch(const Params& p, int interleaved, cudaStream_t st) {
    const long long threads = (long long)p.T * p.units * p.head_splits;
    const long long blocks = (threads + THREADS - 1) / THREADS;
    if (threads > 0x7fffff00ll) return fail(SKV_ERR_UNSUPPORTED, "skv_rotary: too many rows for one launch");
    SKV_CUDA_TRY(launch_pdl(interleaved ? rotary_kernel<T, VEC, true> : rotary_kernel<T, VEC, false>, dim3((unsigned)blocks),
                            dim3(THREADS), 0, st, p));
    SKV_CUDA_TRY(cudaGetLastError());
    return SKV_OK;
}

template <typename T>
static int launch_vec(int vec, const Params& p, int interleaved, cudaStream_t st) {
    switch (vec) {
        case 8: if constexpr (sizeof(T) == 2) return launch<T, 8>(p, interleaved, st);
        case 4: return launch<T, 4>(p, interleaved, st);
        case 2: return launch<T, 2>(p, interleaved, st);
        default: return launch<T, 1>(p, interleaved, st);
    }
}

}  // namespace rot
}  // namespace skv

using namespace skv;

extern "C" int skv_rotary(const void* q, const void* k, void* q_out, void* k_out, int dtype, const void* positions,
                          int positions_are_64, const unsigned long long* freqs, int T, int Hq, int Hk, int D,
                          int rotary_dim, int interleaved, float factor, int adjoint,
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
    DeviceGuard guard(device);
    if (!guard.ok) return fail(SKV_ERR_CUDA, "cannot switch to device %d", device);
    rot::Params p;
    p.src[0] = Hq ? q : k; p.src[1] = Hk ? k : q;
    p.dst[0] = Hq ? q_out : k_out; p.dst[1] = Hk ? k_out : q_out;
    p.st[0] = q_stride_t; p.sh[0] = q_stride_h; p.st[1] = k_stride_t; p.sh[1] = k_stride_h;
    p.dt[0] = q_out_stride_t; p.dh[0] = q_out_stride_h; p.dt[1] = k_out_stride_t; p.dh[1] = k_out_stride_h;
    p.positions = positions; p.pos64 = positions_are_64; p.freqs = freqs;
    p.T = T; p.Hq = Hq; p.H = Hq + Hk; p.R = rotary_dim;
    p.factor = factor; p.sign = adjoint ? -1.f : 1.f;

    // The widest vector that the row's two halves, its tail and every pointer and stride allow: 16 bytes where a layout
    // is an ordinary one, down to single elements for odd rotary widths or views.
    const int esz = dtype == 2 ? 4 : 2;
    int vec = 16 / esz;
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
    while ((rotary_dim / 2) % vec || tail % vec || (tail && rotary_dim % vec)) vec /= 2;
    p.tail_units = tail / vec;
    p.units = rotary_dim / 2 / vec + p.tail_units;
    // Heads are split over threads until the machine is full (eight blocks of 128 threads an SM hold the loads that
    // cover HBM's latency): a prompt's thread walks over many heads and pays for its sines once, a decode step gives
    // every head a thread of its own.
    const long long want = (long long)sm_count(device) * 1024;
    long long splits = (want + (long long)T * p.units - 1) / ((long long)T * p.units);
    splits = splits < 1 ? 1 : splits > p.H ? p.H : splits;
    p.heads_per_split = (int)((p.H + splits - 1) / splits);
    p.head_splits = (p.H + p.heads_per_split - 1) / p.heads_per_split;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == 0) return rot::launch_vec<__half>(vec, p, interleaved, st);
    if (dtype == 1) return rot::launch_vec<__nv_bfloat16>(vec, p, interleaved, st);
    return rot::launch_vec<float>(vec, p, interleaved, st);
}
