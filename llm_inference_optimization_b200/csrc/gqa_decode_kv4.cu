// Dense GQA attention over a paged cache whose keys AND values are held in 4 bits (page records of skv_kv4.cuh), for one
// or more query tokens per sequence, causal among themselves (the last query sees every token of the sequence).
//
// No reference counterpart (the reference reads an unpaged fp16 cache, csrc/kernels/gqa_decode.cu:84-90).
//   s[t]  = scale * sum_w ks[t,w] * sum_{d in group w} q_d kc[t,d]       t < len - n + i + 1 for query i of n
//   out_d = sum_t softmax(s)[t] * vs[t,d/32] * vc[t,d]                   no visible token: 0
//
// What bounds it: HBM delivers a 16-token record (2304 bytes at D = 128) to an SM every ~100 cycles, in which the SM has 400
// issue slots, 200 of them for logic operations: a 4-bit stream is as much about the instructions per record as about the
// bytes.  Hence:
//   * No shared-memory shuffling: a record is stored in fragment order, so a lane fetches its 64 key codes, its 64 value
//     codes and the scales of its two tokens with two 16-byte loads each.
//   * No conversion of codes: a nibble u masked out of its word IS the fp16 number u * 2^-24 (bits 0-3) or u * 2^-20
//     (bits 4-7), subnormal and exact, and products with it are exact in the fp32 accumulator: 5 logic operations for 8
//     codes.  The factor 16 between the two kinds is put into the query (its own exponent is normalised first) and, for
//     values, divided out of the rows of O at the end.  Codes are u - 8: the 8 is taken out of the scores by starting the
//     accumulators at -8 sum(q) and out of O with sum(p), which one product with a tile of ones per group yields.
//   * ks multiplies the fp32 partial scores of its group; vs is folded into the weights before they are rounded to fp16.
//     So that neither small nor large value scales under- or overflow there, the running maximum is taken over
//     s + (a bound of log2 vs), and the weights, at most 1, carry a factor 2^14.  (One rounding to 11 bits per weight.)
//   * Tokens on the M side of both products (S^T = K Q^T, O^T = V^T P^T), up to 8 NT columns (query token, head) on the
//     N side; P goes from the one layout to the other by movmatrix.
//
// Streaming: every warp is on its own -- it copies records to a ring of its own with cp.async (16 bytes per lane and
// request: a record is five requests of a warp), keeps its own softmax state, and meets the others only at the end of a
// segment.  No producer warps and no barriers in the loop.
//
// Work split: the host does not know the lengths.  Work is counted in records over (kv-head, sequence, chunk of columns)
// in this order and cut into equal runs, one for each CTA of ONE resident wave; a CTA finds its run with a scan of the
// lengths and walks over the items in it.  An item that spans CTAs is summed by the last of them to finish (a ticket per
// first CTA), in the order of the sequence: results do not depend on timing.
#include <cuda_bf16.h>

#include "skv_common.cuh"
#include "skv_kv4.cuh"

namespace skv {
namespace kv4 {

constexpr int NW = 8;                 // warps per CTA
constexpr int THREADS = NW * 32;
constexpr int MIN_UNITS = 16;         // records per CTA at least: shorter runs are all start and end
constexpr size_t TICKET_OFF = 256, PARTIAL_OFF = 8192;
constexpr int MAX_GRID = 320;         // CTAs of one wave (a combine keeps this many (max, sum) pairs in registers)
static_assert(MAX_GRID * 4 <= PARTIAL_OFF - TICKET_OFF, "tickets");

template <int D, int NT> struct Shape {
    static constexpr int W = D / 32;                     // scale groups per row
    static constexpr int REC = kv4_record_bytes<D>();
    static constexpr int STAGES = NT == 1 ? 4 : 5;
    static constexpr int CTAS_PER_SM = NT == 1 ? 2 : 1;
    static constexpr int ROW = D + 4;                    // merge rows, padded: 16-byte stores of a warp spread over the banks
    static constexpr int RING = NW * STAGES * REC;
    static constexpr int MERGE = NW * 8 * ROW * 4;       // one n-tile (8 columns) at a time
    static constexpr int ML = NW * 8 * NT * 8;           // (max, sum) per warp and column
    static constexpr size_t SMEM = RING + MERGE + ML + 16;
    static_assert(MAX_GRID / (NT == 1 ? 1 : 2) * 8 * NT * 4 + 16 * 4 + THREADS * 16 + 16 <= MERGE, "combine's scratch");
};

struct Params {
    const void* q;
    void* out;
    const uint8_t* pool;
    long long sp, sh;            // record strides in bytes: page, head
    const int* page_table;       // null: page = b * max_pages + i
    const int* seq_lens;         // null: N
    const int* cu_q;             // null: one query token per sequence
    float* partial_o;            // [2 * CTAs][8 NT][D]
    float* partial_ml;           // [2 * CTAs][8 NT][2]
    int* tickets;                // [CTAs]
    int* status;
    int B, T, N, Hq, Hkv, G, max_pages, num_pages, q_bf16, out_bf16;
    float scale_log2;
};

// One sequence as the work list counts it
struct Seq {
    int q0, nq, len, chunks, recs;
};
template <int NC>
__device__ __forceinline__ Seq sequence(const Params& p, int b) {
    Seq s;
    s.q0 = p.cu_q ? min(max(p.cu_q[b], 0), p.T) : b;
    s.nq = p.cu_q ? min(max(p.cu_q[b + 1], s.q0), p.T) - s.q0 : 1;
    s.len = p.seq_lens ? min(max(p.seq_lens[b], 0), p.N) : p.N;
    s.chunks = (int)(((long long)s.nq * p.G + NC - 1) / NC);
    s.recs = max(1, (s.len + 15) >> 4);      // (an empty sequence still writes zeros)
    return s;
}

struct Segment {
    int h, b, chunk, r0, r1;     // records [r0, r1) of the item
    Seq s;
    bool whole;                  // the item lies in this CTA
    int c_first, c_last;         // CTAs that share it, else
};

__device__ __forceinline__ void mma_f16_c(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}

template <int BYTES>
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&r)[BYTES / 4]) {
    if constexpr (BYTES == 16)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
    else
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
}

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// group w of a row's scales, held as pairs in words
template <int N> __device__ __forceinline__ float group_scale(const uint32_t (&s)[N], int first, int w) {
    return (w & 1) ? bf_hi(s[first + (w >> 1)]) : bf_lo(s[first + (w >> 1)]);
}
// e with max(vs) < 2^e, within what keeps the sums of weights in range
template <int D> __device__ __forceinline__ float scale_bound(const uint32_t (&s)[D / 32]) {
    uint32_t m = s[D / 64];
    if (D == 128) m = __vmaxu2(m, s[D / 64 + 1]);
    m = max(m & 0x7fff0000u, (m << 16) & 0x7fff0000u);
    const float e = __uint_as_float((m >> 23) | 0x4b000000u) - (8388608.f + 126.f);   // exponent field -> float
    return fminf(fmaxf(e, -60.f), 100.f);
}

// Column `col` of the item's list (query token col / G, head col % G), channels d .. d + 3
__device__ __forceinline__ void store_out(const Params& p, const Segment& x, int D, int col, int d, float4 v, float L) {
    const float inv = L == 0.f ? 0.f : 1.f / L;        // nothing visible: zeros; a NaN stays one
    const long long at = ((long long)(x.s.q0 + col / p.G) * p.Hq + x.h * p.G + col % p.G) * D + d;
    uint2 r;
    if (p.out_bf16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x * inv, v.y * inv), b = __floats2bfloat162_rn(v.z * inv, v.w * inv);
        r = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        r = make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
    }
    *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) = r;
}

// Sum of an item's n partial results, by the whole CTA.  scratch: n * cols weights, 16 floats, THREADS * 4 floats.  The
// threads are split over the partials where the columns leave them free; every sum has one order, whoever runs it.
template <int D, int NC>
__device__ __forceinline__ void combine(const Params& p, const Segment& x, int n, int cols, int col0, float* scratch) {
    constexpr int REGS = (MAX_GRID + 31) / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* weight = scratch;                            // [n][cols]
    float* sums = scratch + ((n * cols + 3) & ~3);      // [cols]
    float4* part = reinterpret_cast<float4*>(sums + 16);
    auto slot = [&](int i) { return 2ll * (x.c_first + i) + (i == 0 ? 1 : 0); };
    for (int c = warp; c < cols; c += NW) {
        float2 ml[REGS];
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < REGS; ++i) {
            const int k = lane + 32 * i;
            ml[i] = make_float2(-INFINITY, 0.f);
            if (k < n) ml[i] = __ldcg(reinterpret_cast<const float2*>(p.partial_ml + (slot(k) * NC + c) * 2));
        }
#pragma unroll
        for (int i = 0; i < REGS; ++i) M = fmaxf(M, ml[i].x);
        M = warp_max(M);
        const float ref = M == -INFINITY ? 0.f : M;
        float L = 0.f;
#pragma unroll
        for (int i = 0; i < REGS; ++i) {
            const int k = lane + 32 * i;
            if (k < n) {
                const float w = fast_exp2(ml[i].x - ref);
                weight[k * cols + c] = w;
                L = fmaf(ml[i].y, w, L);
            }
        }
        L = warp_sum(L);
        if (lane == 0) sums[c] = L;
    }
    __syncthreads();
    const int places = cols * (D / 4);
    const int subs = max(1, THREADS / places);
    constexpr int U = 8;                                // partial rows in flight per thread
    for (int i0 = threadIdx.x; i0 < places * subs; i0 += THREADS) {
        const int sub = i0 / places, pos = i0 - sub * places;
        const int c = pos / (D / 4), d = pos % (D / 4) * 4;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = sub; k0 < n; k0 += U * subs) {
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)                 // (past the end: the last row again, with weight zero)
                v[u] = __ldcg(reinterpret_cast<const float4*>(p.partial_o + (slot(min(k0 + u * subs, n - 1)) * NC + c) * D + d));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = k0 + u * subs;
                if (k >= n) break;
                const float w = weight[k * cols + c];
                acc.x = fmaf(v[u].x, w, acc.x); acc.y = fmaf(v[u].y, w, acc.y);
                acc.z = fmaf(v[u].z, w, acc.z); acc.w = fmaf(v[u].w, w, acc.w);
            }
        }
        if (subs == 1) store_out(p, x, D, col0 + c, d, acc, sums[c]);
        else part[i0] = acc;
    }
    if (subs > 1) {
        __syncthreads();
        for (int pos = threadIdx.x; pos < places; pos += THREADS) {
            float4 acc = part[pos];
            for (int k = 1; k < subs; ++k) {
                const float4 v = part[k * places + pos];
                acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
            }
            const int c = pos / (D / 4);
            store_out(p, x, D, col0 + c, pos % (D / 4) * 4, acc, sums[c]);
        }
    }
}

template <int D, int NT>
__global__ void __launch_bounds__(THREADS, (Shape<D, NT>::CTAS_PER_SM)) gqa_decode_kv4_kernel(const Params p) {
    using S = Shape<D, NT>;
    constexpr int W = S::W, NC = 8 * NT, REC = S::REC, STAGES = S::STAGES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tq = lane & 3;
    extern __shared__ __align__(16) uint8_t smem[];
    float* merge = reinterpret_cast<float*>(smem + S::RING);
    float2* merge_ml = reinterpret_cast<float2*>(smem + S::RING + S::MERGE);       // [NW][NC]
    int* flag = reinterpret_cast<int*>(smem + S::RING + S::MERGE + S::ML);
    const uint32_t ring = smem_u32(smem) + warp * (STAGES * REC);

    pdl_wait_prior_grids();
    pdl_launch_dependents();

    // ---- this CTA's run of the work list (every warp finds it for itself)
    long long per_head = 0;
    for (int b = lane; b < p.B; b += 32) {
        const Seq s = sequence<NC>(p, b);
        per_head += (long long)s.chunks * s.recs;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) per_head += __shfl_xor_sync(0xffffffffu, per_head, o);
    const long long total = per_head * p.Hkv;
    const long long run = max((total + gridDim.x - 1) / gridDim.x, (long long)MIN_UNITS);
    long long at = run * blockIdx.x;                  // position in the list
    const long long end = min(at + run, total);
    if (at >= end) return;

    Segment sg;
    sg.h = (int)(at / per_head);
    long long rest = at - sg.h * per_head;
    sg.b = -1;
    for (int b0 = 0; b0 < p.B; b0 += 32) {            // find the sequence: a warp-wide prefix sum of 32 at a time
        long long mine = 0;
        if (b0 + lane < p.B) {
            const Seq s = sequence<NC>(p, b0 + lane);
            mine = (long long)s.chunks * s.recs;
        }
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned past = __ballot_sync(0xffffffffu, upto > rest);
        if (past) {
            const int l = __ffs(past) - 1;
            sg.b = b0 + l;
            rest -= __shfl_sync(0xffffffffu, upto - mine, l);
            break;
        }
        rest -= __shfl_sync(0xffffffffu, upto, 31);
    }
    if (sg.b < 0) return;                             // (only if the lengths changed under the kernel)
    sg.s = sequence<NC>(p, sg.b);
    sg.chunk = (int)(rest / sg.s.recs);
    sg.r0 = (int)(rest - (long long)sg.chunk * sg.s.recs);

    auto finish_segment = [&]() {                     // r1 and who shares the item, from (b, chunk, r0) at list position `at`
        sg.r1 = (int)min((long long)sg.s.recs, sg.r0 + (end - at));
        sg.whole = sg.r0 == 0 && sg.r1 == sg.s.recs;
        sg.c_first = sg.c_last = blockIdx.x;
        if (!sg.whole) {
            sg.c_first = (int)((at - sg.r0) / run);
            sg.c_last = (int)((at - sg.r0 + sg.s.recs - 1) / run);
        }
    };
    finish_segment();

    // ---- streaming: this warp's records of a segment are r0 + warp, r0 + warp + NW, ...
    int n_rec = 0, page_now = 0, page_next = 0;
    bool bad_page = false;
    auto load_page = [&](const Segment& x, int k) {   // page of this warp's k-th record
        const int r = x.r0 + warp + k * NW;
        int page = 0;
        if (k < n_rec)
            page = p.page_table ? __ldg(p.page_table + (long long)x.b * p.max_pages + r) : x.b * p.max_pages + r;
        return checked_page(page, p.num_pages, bad_page);
    };
    auto issue = [&](const Segment& x, int k) {
        if ((k & 31) == 0) {                          // pages of the next 32 records, one per lane, fetched 32 ahead
            page_now = k ? page_next : load_page(x, lane);
            page_next = load_page(x, k + 32 + lane);
        }
        const int page = __shfl_sync(0xffffffffu, page_now, k & 31);
        if (k < n_rec) {
            const uint8_t* src = p.pool + SKV_INDEX(page, p.num_pages) * p.sp + x.h * p.sh + lane * 16;
            const uint32_t dst = ring + (k % STAGES) * REC + lane * 16;
#pragma unroll
            for (int i = 0; i < REC / 512; ++i) cp_async16(dst + i * 512, src + i * 512);
            if (lane < REC % 512 / 16) cp_async16(dst + REC / 512 * 512, src + REC / 512 * 512);
        }
        cp_async_commit();
    };
    // the last token that any column of the item sees bounds the records that are read
    auto records = [&](const Segment& x) {
        const int cols = x.s.nq * p.G;
        const int i_last = (min(cols, (x.chunk + 1) * NC) - 1) / p.G;
        const int seen = max(0, x.s.len - x.s.nq + i_last + 1);
        const int r1 = min(x.r1, (seen + 15) >> 4);
        return max(0, (r1 - x.r0 - warp + NW - 1) / NW);
    };
    auto begin = [&](const Segment& x) {
        n_rec = records(x);
#pragma unroll
        for (int k = 0; k < STAGES - 1; ++k) issue(x, k);
    };
    begin(sg);

    for (;;) {
        // ---- query columns of this item
        const int col0 = sg.chunk * NC;               // first column: query token col0 / G, head col0 % G of the group
        const int cols = min(sg.s.nq * p.G - col0, NC);
        uint32_t qb[NT][W][4];
        float init[NT][W][2], factor[NT][2];
        int limit[NT][2];                             // tokens that columns 2tq, 2tq + 1 see
        int limit_min = sg.s.len - sg.s.nq + col0 / p.G + 1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int c = nt * 8 + g;
            const int qi = (col0 + c) / p.G, hj = (col0 + c) % p.G;
            const long long row = ((long long)(sg.s.q0 + qi) * p.Hq + sg.h * p.G + hj) * D;
            float x[W][8];
            float amax = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                uint4 raw = make_uint4(0u, 0u, 0u, 0u);
                if (c < cols) raw = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p.q) + row + w * 32 + tq * 8);
                if (p.q_bf16) {
                    const uint32_t v[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) { x[w][2 * i] = bf_lo(v[i]); x[w][2 * i + 1] = bf_hi(v[i]); }
                } else {
                    unpack8(raw, x[w]);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[w][i]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // the column's own exponent is taken out, exactly: its largest channel lies in [2^10, 2^11), sixteen times which
            // fp16 still holds; channels below 2^-25 of it round
            const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127, -110), 127);
            const float up = __uint_as_float((uint32_t)(137 - e) << 23);
            float sum[W];
#pragma unroll
            for (int w = 0; w < W; ++w) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {          // nibbles i and i + 4; even i are masked out of bits 0-3, odd out of 4-7
                    const float k = (i & 1) ? up : up * 16.f;
                    qb[nt][w][i] = pack_half2(x[w][i] * k, x[w][i + 4] * k);
                }
                float a = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qb[nt][w][i]));
                    a += (f.x + f.y) * ((i & 1) ? 1.f : 0.0625f);
                }
                a += __shfl_xor_sync(0xffffffffu, a, 1);
                a += __shfl_xor_sync(0xffffffffu, a, 2);
                sum[w] = a * -7.62939453125e-06f;       // -8 * 2^-20
            }
            const float f = p.scale_log2 * __uint_as_float((uint32_t)min(max(e + 137, 1), 254) << 23);   // 2^20 / up
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int from = (2 * tq + j) * 4;
                factor[nt][j] = __shfl_sync(0xffffffffu, f, from);
#pragma unroll
                for (int w = 0; w < W; ++w) init[nt][w][j] = __shfl_sync(0xffffffffu, sum[w], from);
                const int cj = nt * 8 + 2 * tq + j;
                limit[nt][j] = cj < cols ? sg.s.len - sg.s.nq + (col0 + cj) / p.G + 1 : sg.s.len;
            }
        }

        // o[nt][2w + m][j], [j + 2]: channels 32w + 4g + 2m, + 1 of column 8nt + 2tq + j
        float o[NT][2 * W][4], psum[NT][W][4], mrun[NT][2], lrun[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2 * W; ++c) o[nt][c][0] = o[nt][c][1] = o[nt][c][2] = o[nt][c][3] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) psum[nt][w][0] = psum[nt][w][1] = psum[nt][w][2] = psum[nt][w][3] = 0.f;
            mrun[nt][0] = mrun[nt][1] = -INFINITY;
            lrun[nt][0] = lrun[nt][1] = 0.f;
        }

        const int n_mine = n_rec;
        const int tok_a = 4 * (g >> 1) + (g & 1);      // rows g and g + 8 of the score tile are tokens tok_a and tok_a + 2
        for (int k = 0; k < n_mine; ++k) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();                              // record k is here, and every lane is done with record k - 1
            issue(sg, k + STAGES - 1);
            const uint32_t rec = ring + (k % STAGES) * REC;
            const int tok0 = (sg.r0 + warp + k * NW) * 16;

            // scores: rows g, g + 8 = places g, g + 8 of the record
            uint32_t ka[W], kb[W], sa[W], sb[W];       // sa, sb: W key scales, then W value scales, two a word
            lds<D / 8>(rec + g * (D / 2) + tq * (D / 8), ka);
            lds<D / 8>(rec + (g + 8) * (D / 2) + tq * (D / 8), kb);
            lds<D / 8>(rec + 16 * D + g * (D / 8), sa);
            lds<D / 8>(rec + 16 * D + (g + 8) * (D / 8), sb);
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const uint32_t a8 = ka[w] >> 8, b8 = kb[w] >> 8;
                const uint32_t m0[4] = {ka[w] & 0x000f000fu, kb[w] & 0x000f000fu, ka[w] & 0x00f000f0u, kb[w] & 0x00f000f0u};
                const uint32_t m1[4] = {a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u, b8 & 0x00f000f0u};
                const float ska = group_scale(sa, 0, w), skb = group_scale(sb, 0, w);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float acc[4];
                    mma_f16_c(acc, m0, qb[nt][w][0], qb[nt][w][1], init[nt][w][0], init[nt][w][1]);
                    mma_f16(acc, m1, qb[nt][w][2], qb[nt][w][3]);
                    s[nt][0] = fmaf(acc[0], ska, s[nt][0]);
                    s[nt][1] = fmaf(acc[1], ska, s[nt][1]);
                    s[nt][2] = fmaf(acc[2], skb, s[nt][2]);
                    s[nt][3] = fmaf(acc[3], skb, s[nt][3]);
                }
            }
            const bool masked = tok0 + 16 > limit_min;
            const int ta = tok0 + tok_a, tb = ta + 2;
            const float ea = scale_bound<D>(sa), eb = scale_bound<D>(sb);
            float mnew[NT][2];
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[nt][j] *= factor[nt][j & 1];
                if (masked) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if ((j < 2 ? ta : tb) >= limit[nt][j & 1]) s[nt][j] = -INFINITY;
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {          // maximum over the 16 tokens: two rows of this lane, then the lanes g
                    float mx = fmaxf(s[nt][j] + ea, s[nt][j + 2] + eb);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    mnew[nt][j] = fmaxf(mrun[nt][j], mx);
                    grow |= mnew[nt][j] > mrun[nt][j];
                }
            }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        // (a column that has seen nothing yet: exp2(-inf) = 0 times zeros)
                        const float c = fast_exp2(mrun[nt][j] - (mnew[nt][j] == -INFINITY ? 0.f : mnew[nt][j]));
                        lrun[nt][j] *= c;
#pragma unroll
                        for (int i = 0; i < 2 * W; ++i) { o[nt][i][j] *= c; o[nt][i][j + 2] *= c; }
#pragma unroll
                        for (int w = 0; w < W; ++w) { psum[nt][w][j] *= c; psum[nt][w][j + 2] *= c; }
                        mrun[nt][j] = mnew[nt][j];
                    }
            }
            float pr[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float m = mrun[nt][j & 1] == -INFINITY ? 0.f : mrun[nt][j & 1];
                    pr[nt][j] = fast_exp2(s[nt][j] - m);
                }
                lrun[nt][0] += pr[nt][0] + pr[nt][2];
                lrun[nt][1] += pr[nt][1] + pr[nt][3];
            }

            // values: plane j holds tokens 4tq + 2j and + 1 of the lane's channels, matching P's rows after the move
            uint32_t va[W], vb[W];
            lds<D / 8>(rec + 8 * D + lane * (D / 8), va);
            lds<D / 8>(rec + 12 * D + lane * (D / 8), vb);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const uint32_t sel = (w & 1) ? 0x7632u : 0x5410u;
                const uint32_t x = __byte_perm(va[w >> 1], va[W / 2 + (w >> 1)], sel);
                const uint32_t y = __byte_perm(vb[w >> 1], vb[W / 2 + (w >> 1)], sel);
                const uint32_t x8 = x >> 8, y8 = y >> 8;
                const uint32_t m0[4] = {x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u};
                const uint32_t m1[4] = {x8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x000f000fu, y8 & 0x00f000f0u};
                const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
                const float sva = group_scale(sa, W / 2, w) * 16384.f, svb = group_scale(sb, W / 2, w) * 16384.f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float z[4] = {pr[nt][0] * sva, pr[nt][1] * sva, pr[nt][2] * svb, pr[nt][3] * svb};
                    if (masked) {                      // a masked token's scale may be anything, NaN included
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if ((j < 2 ? ta : tb) >= limit[nt][j & 1]) z[j] = 0.f;
                    }
                    const uint32_t b0 = movmatrix_trans(pack_half2(z[0], z[1]));
                    const uint32_t b1 = movmatrix_trans(pack_half2(z[2], z[3]));
                    mma_f16(o[nt][2 * w], m0, b0, b1);
                    mma_f16(o[nt][2 * w + 1], m1, b0, b1);
                    mma_f16(psum[nt][w], ones, b0, b1);
                }
            }
        }
        cp_async_wait<0>();
        __syncwarp();

        // ---- the next segment's first records are on their way while this one is written
        const Segment done = sg;
        at += sg.r1 - sg.r0;
        bool more = at < end;
        if (more) {
            sg.r0 = 0;
            if (++sg.chunk >= sg.s.chunks) {
                sg.chunk = 0;
                do {
                    if (++sg.b == p.B) { sg.b = 0; ++sg.h; }
                    sg.s = sequence<NC>(p, sg.b);
                } while (sg.s.chunks == 0 && sg.h < p.Hkv);
                more = sg.h < p.Hkv;                   // (`at` < end, so it is, while the lengths stay as they are)
            }
        }
        if (more) {
            finish_segment();
            begin(sg);
        }

        // ---- merge the warps, a tile of 8 columns at a time
        const long long slot = 2ll * blockIdx.x + (done.r0 == 0 ? 1 : 0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = 2 * tq + j;
                float l = lrun[nt][j];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (g == 0) merge_ml[warp * 8 + c] = make_float2(mrun[nt][j], l);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    // rows g hold sum p u 2^-24, rows g + 8 sum p u 2^-20; u = code + 8; p carries 2^14
                    const float b0 = 8.f * psum[nt][w][j], b1 = 8.f * psum[nt][w][j + 2];
                    float4 v;
                    v.x = (o[nt][2 * w][j] * 16777216.f - b0) * 6.103515625e-05f;
                    v.y = (o[nt][2 * w][j + 2] * 1048576.f - b1) * 6.103515625e-05f;
                    v.z = (o[nt][2 * w + 1][j] * 16777216.f - b0) * 6.103515625e-05f;
                    v.w = (o[nt][2 * w + 1][j + 2] * 1048576.f - b1) * 6.103515625e-05f;
                    *reinterpret_cast<float4*>(merge + (warp * 8 + c) * S::ROW + 32 * w + 4 * g) = v;
                }
            }
            __syncthreads();
            const int n_cols = min(cols - nt * 8, 8);
            for (int i = threadIdx.x; i < n_cols * (D / 4); i += THREADS) {
                const int c = i / (D / 4), d = i % (D / 4) * 4;
                float2 ml[NW];
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    ml[w] = merge_ml[w * 8 + c];
                    M = fmaxf(M, ml[w].x);
                }
                const float ref = M == -INFINITY ? 0.f : M;
                float L = 0.f;
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const float wt = fast_exp2(ml[w].x - ref);
                    const float4 v = *reinterpret_cast<const float4*>(merge + (w * 8 + c) * S::ROW + d);
                    L = fmaf(ml[w].y, wt, L);
                    acc.x = fmaf(v.x, wt, acc.x); acc.y = fmaf(v.y, wt, acc.y);
                    acc.z = fmaf(v.z, wt, acc.z); acc.w = fmaf(v.w, wt, acc.w);
                }
                const int col = nt * 8 + c;
                if (done.whole) {
                    store_out(p, done, D, col0 + col, d, acc, L);
                } else {
                    *reinterpret_cast<float4*>(p.partial_o + (slot * NC + col) * D + d) = acc;
                    if (d == 0) *reinterpret_cast<float2*>(p.partial_ml + (slot * NC + col) * 2) = make_float2(M, L);
                }
            }
            __syncthreads();
        }

        // ---- an item that spans CTAs: the last one to arrive adds up
        if (!done.whole) {
            const int n = done.c_last - done.c_first + 1;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                const int last = atomicAdd(&p.tickets[done.c_first], 1) == n - 1;
                if (last) p.tickets[done.c_first] = 0;  // ready for the next launch on this workspace
                *flag = last;
            }
            __syncthreads();
            if (*flag) {
                __threadfence();
                combine<D, NC>(p, done, n, cols, col0, merge);
            }
            __syncthreads();
        }
        if (!more) break;
    }
    report_bad_page(bad_page, p.status);
}

template <int D, int NT>
static int launch(const Params& p, void* workspace, int device, cudaStream_t stream) {
    using S = Shape<D, NT>;
    constexpr int NC = 8 * NT;
    static bool configured[64] = {};
    if (device >= 64 || !configured[device]) {
        SKV_CUDA_TRY(cudaFuncSetAttribute(gqa_decode_kv4_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM));
        if (device < 64) configured[device] = true;
    }
    // no more CTAs than the longest possible work gives MIN_UNITS records each
    const long long chunks = ((long long)p.T * p.G + NC - 1) / NC + (p.cu_q ? p.B : 0);
    const long long units = p.Hkv * (p.cu_q ? chunks : (long long)p.B * ((p.G + NC - 1) / NC)) * (((long long)p.N + 15) / 16);
    long long grid = (long long)sm_count(device) * S::CTAS_PER_SM;
    if (grid > MAX_GRID / (NT == 1 ? 1 : 2)) grid = MAX_GRID / (NT == 1 ? 1 : 2);
    if (grid > (units + MIN_UNITS - 1) / MIN_UNITS) grid = (units + MIN_UNITS - 1) / MIN_UNITS;
    Params q = p;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    q.status = reinterpret_cast<int*>(ws);
    q.tickets = reinterpret_cast<int*>(ws + TICKET_OFF);
    q.partial_ml = reinterpret_cast<float*>(ws + PARTIAL_OFF);
    q.partial_o = q.partial_ml + 2ll * MAX_GRID * 8 * 2;        // (NT = 2 has half the CTAs and twice the columns)
    SKV_CUDA_TRY(launch_pdl(gqa_decode_kv4_kernel<D, NT>, dim3((unsigned)grid), dim3(THREADS), S::SMEM, stream, q));
    SKV_CUDA_TRY(cudaGetLastError());
    return SKV_OK;
}

static size_t workspace_bytes(int D) { return PARTIAL_OFF + 2ull * MAX_GRID * 8 * (2 + D) * 4; }

}  // namespace kv4
}  // namespace skv

using namespace skv;

extern "C" {

size_t skv_gqa_decode_kv4_workspace_bytes(int D) { return D == 64 || D == 128 ? kv4::workspace_bytes(D) : 0; }

int skv_gqa_decode_kv4(const void* q, int q_is_bf16, const void* pool, const int* page_table, const int* seq_lens,
                       const int* cu_q, void* out, int out_is_bf16, void* workspace, size_t workspace_bytes, int T, int B, int N,
                       int Hq, int Hkv, int D, int max_pages, int num_pages, long long pool_stride_page,
                       long long pool_stride_head, float scale, int device, void* stream) {
    if (!pool) return fail(SKV_ERR_BAD_ARG, "skv_gqa_decode_kv4: null pool");
    if (T < 0 || B <= 0 || N <= 0 || Hq <= 0 || Hkv <= 0 || num_pages <= 0 || max_pages <= 0)
        return fail(SKV_ERR_BAD_ARG, "skv_gqa_decode_kv4: sizes must be positive");
    if (Hq % Hkv != 0) return fail(SKV_ERR_BAD_ARG, "Hq=%d must be divisible by Hkv=%d", Hq, Hkv);
    if (D != 64 && D != 128) return fail(SKV_ERR_UNSUPPORTED, "4-bit KV decode supports head dims 64 and 128 (got %d)", D);
    if ((long long)max_pages * KV4_PAGE < N) return fail(SKV_ERR_BAD_ARG, "max_pages * 16 < N");
    if (N > 0x7fffffff - KV4_PAGE) return fail(SKV_ERR_UNSUPPORTED, "sequences of %d tokens are not supported", N);
    if (!(scale > 0.f)) return fail(SKV_ERR_BAD_ARG, "softmax scale must be positive");
    if (T == 0) return SKV_OK;
    if (!q || !out) return fail(SKV_ERR_BAD_ARG, "skv_gqa_decode_kv4: null tensor pointer");
    if (!cu_q && T != B) return fail(SKV_ERR_BAD_ARG, "skv_gqa_decode_kv4: %d query rows for %d sequences need cu_q", T, B);
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(pool) |
         (unsigned long long)pool_stride_page | (unsigned long long)pool_stride_head) & 15)
        return fail(SKV_ERR_BAD_ARG, "q, out, the pool and its strides must be multiples of 16 bytes");
    if ((long long)T * (Hq / Hkv) > 0x7fffffffll - 16) return fail(SKV_ERR_UNSUPPORTED, "too many query rows");
    if (!workspace || workspace_bytes < kv4::workspace_bytes(D))
        return fail(SKV_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, kv4::workspace_bytes(D));
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(SKV_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(SKV_ERR_CUDA, "cannot switch to device %d", device);
    kv4::Params p = {};
    p.q = q; p.out = out; p.pool = static_cast<const uint8_t*>(pool);
    p.sp = pool_stride_page; p.sh = pool_stride_head;
    p.page_table = page_table; p.seq_lens = seq_lens; p.cu_q = cu_q;
    p.B = B; p.T = T; p.N = N; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv;
    p.max_pages = max_pages; p.num_pages = num_pages; p.q_bf16 = q_is_bf16; p.out_bf16 = out_is_bf16;
    p.scale_log2 = scale * 1.4426950408889634f;
    // columns per pass over the cache: 8, or 16 where the (query token, head) pairs of a sequence fill more than 8
    const bool wide = (long long)p.G * ((T + B - 1) / B) > 8;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (D == 128) return wide ? kv4::launch<128, 2>(p, workspace, device, st) : kv4::launch<128, 1>(p, workspace, device, st);
    return wide ? kv4::launch<64, 2>(p, workspace, device, st) : kv4::launch<64, 1>(p, workspace, device, st);
}

}  // extern "C"

SKV_BOUNDS_GETTER(skv_debug_bounds_gqa_decode_kv4)
