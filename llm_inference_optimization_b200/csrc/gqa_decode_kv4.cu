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
//     accumulators at -8 ks sum(q), a small product of its own, and out of the value codes by an exact packed addition.
//   * ks multiplies the fp32 partial scores of its group; vs is folded into the weights before they are rounded to fp16 (one
//     rounding of each product of weight and scale).  vs is taken relative to a power of two of its group of 32 channels,
//     which follows the largest scale seen there; the reference that scores are taken against before exp2 only has to keep
//     the weights within fp16 and follows their running maximum in jumps of several powers of two.  So a record costs one vote
//     where exact running maxima cost shuffles and a rescaling of O.
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
//
// Measured (D = 128, 8 kv-heads of 4 heads, one query each): 4 sequences of 65536 tokens 64.7 us, 4.7 TB/s, 0.71 of a copy (the
// stream alone, without the arithmetic, takes 52.5); 16 ragged sequences of 0 .. 32000 tokens 55.8 us; one of 4093 tokens
// 12.0 us, all of it start, merge and sum.  ncu: 318 instructions a record, issue slots 63 % busy, logic pipe 55 %, tensor pipe
// 27 %.  (A power of two for each group of 32 channels instead of one bound for all, and scores far from zero, cost 2 %.)
#include <cuda_bf16.h>

#include "skv_common.cuh"
#include "skv_kv4.cuh"

namespace skv {
namespace kv4 {

// Weights are kept below 2^WEIGHT_MAX and are at most 2^WEIGHT_AIM when their reference has just moved: four powers of two
// before it moves again.  Value scales relative to their group's power of two lie below 2 (below 3.99 for bf16's topmost
// exponent), so products stay below fp16's 65504; when the power has just moved, below 2^(1 - SCALE_ROOM): the next larger
// scales find room (0, 1, 2: 70.1, 68.7, 68.5 us for 4 sequences of 65536 tokens, 67.9 with one power for all groups and
// weights together).  A product has eleven bits down to 2^-22 of the largest weight times the largest scale of the same group
// that the warp has seen, and is off by at most 2^-33 of that below (2^-25, half of fp16's smallest step, against 2^(10 - 2)).
constexpr float WEIGHT_MAX = 14.f, WEIGHT_AIM = 10.f;
constexpr int SCALE_ROOM = 2;
constexpr float BIG_SCORE = 1048576.f;   // a step of fp32 is an eighth there
constexpr uint32_t MOVE = 0x40004000u;   // bit 14 of a bf16 number, twice: 2 and more
// Sums leave the registers times 2^SUMS_DOWN: 2^14 * 2^16 tokens * 8 * the largest bf16 number times 2^-40 is within fp32.
constexpr int SUMS_DOWN = -40;
constexpr float NOTHING = -3e38f;     // reference of a column that has seen no token, near the lowest number: scores lie above it
constexpr int MIN_UNITS = 16;         // records per CTA at least: shorter runs are all start and end
constexpr size_t TICKET_OFF = 256, PARTIAL_OFF = 8192;
constexpr int MAX_GRID = 160;         // CTAs of one wave (a combine keeps this many (max, sum) pairs in a warp's registers)
static_assert(MAX_GRID * 4 <= PARTIAL_OFF - TICKET_OFF, "tickets");

template <int D, int NT> struct Shape {
    // Warps of a CTA, one CTA an SM: 16 at 128 registers, 8 at 256.  (Two CTAs of 8: the one that came first on its SM ended
    // at 50 us of 4 sequences of 65536 tokens, the other at 62; 16 warps of one end within 3 us of one another, at 60.)
    static constexpr int NW = NT == 1 ? 16 : 8;
    // What starting an item costs a CTA, in records its warps could have read: query, first loads, merge.  (Without it CTAs
    // with several items end last: 16 ragged sequences 67.7 us with 0, 64.1 with a third, 62.4 with this, 62.5 with four
    // thirds at the time it was brought in.)
    static constexpr int SETUP = 6 * NW;
    static constexpr int THREADS = NW * 32;
    static constexpr int W = D / 32;                     // scale groups per row
    static constexpr int REC = kv4_record_bytes<D>();
    static constexpr int STAGES = NT == 1 ? 3 : 5;       // records in a warp's ring: 111 | 92 KB of a CTA at D = 128
    static constexpr int ROW = D + 4;                    // rows of sums, padded: 16-byte stores of a warp spread over the banks
    static constexpr int RING = NW * STAGES * REC;
    static constexpr int SCRATCH = MAX_GRID * 8 * NT * 4 + 16 * 4 + THREADS * 16 + 16;   // what combine() needs
    static constexpr int TILE = NW * 8 * NT * ROW * 4;   // the sums of every warp
    static constexpr int MERGE = TILE > SCRATCH ? TILE : SCRATCH;
    static constexpr int ML = NW * 8 * NT * 8;           // (max, sum) per warp and column
    static constexpr int QUERY = NT * (W * 512 + 32 * 12);   // the item's columns as operands, and 12 bytes per lane
    static constexpr size_t SMEM = RING + MERGE + ML + 2 * QUERY + 128;
};

struct Params {
    const void* q;
    void* out;
    const uint8_t* pool;
    uint32_t sp;                 // record strides in bytes: page (below 4 GB: one multiply-add makes an address), head
    long long sh;
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
    b = SKV_INDEX(b, p.B);
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

// products that start from zero
__device__ __forceinline__ void mma_f16_0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16_0(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// -136 and -128 times 2^-24, twice: what a byte of value codes, and its upper nibble in place, hold too much
constexpr uint32_t MINUS_136 = 0x80888088u, MINUS_128 = 0x80808080u;
__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("add.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// cp.async, or zeros
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool p) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(p ? 16 : 0) : "memory");
}
// cp.async under a predicate, without a branch
__device__ __forceinline__ void cp_async16_if(uint32_t dst, const void* src, bool p) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p cp.async.cg.shared.global [%0], [%1], 16;\n\t}"
                 ::"r"(dst), "l"(src), "r"((int)p) : "memory");
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
template <bool V> struct Constant { static constexpr bool value = V; };

// The power of two that a group's value scales are multiplied by, a bf16 number of field 254 - e for scales of fields up to e
// (fields with the bias 127, e = 0 .. 253: 2^-127 is no normal number, so the topmost field counts as the one below it).
constexpr uint32_t DOWN_NONE = 254u << 7;             // no scale yet, or numbers below the normal range: 2^127
template <int N> __device__ __forceinline__ int exponent_of(const uint32_t (&down)[N], int w) {
    return 254 - (int)(down[w >> 1] >> ((w & 1) * 16 + 7) & 0xffu);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ constexpr float exp2_of(int e) {
    float x = 1.f;
    for (int i = 0; i < (e < 0 ? -e : e); ++i) x *= e < 0 ? 0.5f : 2.f;
    return x;
}

// Column `col` of the item's list (query token col / G, head col % G), channels d .. d + 3
__device__ __forceinline__ void store_out(const Params& p, const Segment& x, int D, int col, int d, float4 v, float L) {
    const float inv = L == 0.f ? 0.f : 1.f / L;        // nothing visible: zeros; a NaN stays one
    const long long at = ((long long)SKV_INDEX(x.s.q0 + col / p.G, p.T) * p.Hq + SKV_INDEX(x.h * p.G + col % p.G, p.Hq)) * D + SKV_INDEX(d, D - 3);
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
template <int D, int NC, int THREADS>
__device__ __forceinline__ void combine(const Params& p, const Segment& x, int n, int cols, int col0, float* scratch) {
    constexpr int REGS = (MAX_GRID + 31) / 32;
    constexpr int NW = THREADS / 32;
    constexpr int U = 4;                                // partial rows in flight per thread (more would cost the loop registers)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* weight = scratch;                            // [n][cols]
    float* sums = scratch + ((n * cols + 3) & ~3);      // [cols]
    float4* part = reinterpret_cast<float4*>(sums + 16);
    const int places = cols * (D / 4);
    const int subs = max(1, THREADS / places);
    // the k-th partial row of thread i: the same for all but the first CTA, whose slot is its second
    auto row = [&](int i, int k) {
        const int pos = i % places;
        const long long slot = 2ll * SKV_INDEX(x.c_first + k, (int)gridDim.x) + (k == 0 ? 1 : 0);
        return p.partial_o + (slot * NC + pos / (D / 4)) * D + pos % (D / 4) * 4;
    };
    float4 v[U];                                        // asked for before the weights are known (past the end: the last row again)
    if (threadIdx.x < places * subs) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            v[u] = __ldcg(reinterpret_cast<const float4*>(row(threadIdx.x, min(threadIdx.x / places + u * subs, n - 1))));
    }
    for (int c = warp; c < cols; c += NW) {
        float2 ml[REGS];
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < REGS; ++i) {
            const int k = lane + 32 * i;
            ml[i] = make_float2(-INFINITY, 0.f);
            if (k < n) ml[i] = __ldcg(reinterpret_cast<const float2*>(p.partial_ml + ((2ll * SKV_INDEX(x.c_first + k, (int)gridDim.x) + (k == 0 ? 1 : 0)) * NC + c) * 2));
        }
#pragma unroll
        for (int i = 0; i < REGS; ++i) M = fmaxf(M, ml[i].x);
        M = warp_max(M);
        float L = 0.f;
#pragma unroll
        for (int i = 0; i < REGS; ++i) {
            const int k = lane + 32 * i;
            if (k < n) {
                const float w = fast_exp2(ml[i].x - M);
                weight[SKV_INDEX(k * cols + c, MAX_GRID * NC)] = w;
                L = fmaf(ml[i].y, w, L);
            }
        }
        L = warp_sum(L);
        if (lane == 0) sums[c] = L;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < places * subs; i += THREADS) {
        const int sub = i / places, c = i % places / (D / 4);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = sub; k0 < n; k0 += U * subs) {
            if (i != threadIdx.x || k0 != sub) {
#pragma unroll
                for (int u = 0; u < U; ++u) v[u] = __ldcg(reinterpret_cast<const float4*>(row(i, min(k0 + u * subs, n - 1))));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = k0 + u * subs;
                const float w = k < n ? weight[k * cols + c] : 0.f;
                if (k < n) {
                    acc.x = fmaf(v[u].x, w, acc.x); acc.y = fmaf(v[u].y, w, acc.y);
                    acc.z = fmaf(v[u].z, w, acc.z); acc.w = fmaf(v[u].w, w, acc.w);
                }
            }
        }
        if (subs == 1) store_out(p, x, D, col0 + c, i % (D / 4) * 4, acc, sums[c]);
        else part[i] = acc;
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
__global__ void __launch_bounds__((Shape<D, NT>::THREADS), 1) gqa_decode_kv4_kernel(const Params p) {
    using S = Shape<D, NT>;
    constexpr int W = S::W, NC = 8 * NT, REC = S::REC, STAGES = S::STAGES, NW = S::NW, THREADS = S::THREADS;
    constexpr int SETUP = S::SETUP;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, tq = lane & 3;
    extern __shared__ __align__(16) uint8_t smem[];
    float* merge = reinterpret_cast<float*>(smem + S::RING);
    float2* merge_ml = reinterpret_cast<float2*>(smem + S::RING + S::MERGE);       // [NW][NC]
    uint8_t* query = smem + S::RING + S::MERGE + S::ML;                             // two of them, for items in turn
    // What only the change from one item to the next needs lives in shared memory: the loop below needs the registers.
    struct State {
        Segment sg;
        int last;
        long long at, end, run;                       // list position behind sg, end of this CTA's run, length of a run
    };
    static_assert(sizeof(State) <= 128, "state");
    State* state = reinterpret_cast<State*>(query + 2 * S::QUERY);
    const uint32_t ring = smem_u32(smem) + warp * (STAGES * REC);

    pdl_wait_prior_grids();
    pdl_launch_dependents();

    // ---- this CTA's run of the work list (every warp finds it for itself).  An item counts SETUP units for starting it and
    // one for each record; positions fit 32 bits but for work of days, whose runs are found in 64.
    auto units = [&](int b) {                         // of sequence b + lane of a kv-head
        if (b + lane >= p.B) return 0ll;
        const Seq s = sequence<NC>(p, b + lane);
        return (long long)s.chunks * (SETUP + s.recs);
    };
    auto prefix = [&](long long v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long w = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += w;
        }
        return v;
    };
    long long mine = units(0), upto = prefix(mine);   // the first 32 sequences, of most calls all: counted once
    long long per_head = 0;
    for (int b0 = 32; b0 < p.B; b0 += 32) per_head += units(b0);
    if (p.B > 32) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) per_head += __shfl_xor_sync(0xffffffffu, per_head, o);
    }
    per_head += __shfl_sync(0xffffffffu, upto, 31);
    const long long total = per_head * p.Hkv;
    const bool small = total < 0x40000000ll;
    auto divide = [&](long long a, long long b) { return small ? (long long)((uint32_t)a / (uint32_t)b) : a / b; };
    // the item at (h, b, chunk) of sg, from `place` on (its position in the item: SETUP + record), at list position `at`, which
    // moves behind what is taken: false if the run ends before the first record
    auto take = [&](Segment& sg, long long& at, int place, long long end, long long run) {
        sg.r0 = max(place - SETUP, 0);
        const long long stop = min((long long)(SETUP + sg.s.recs), place + (end - at));
        sg.r1 = (int)max(stop - SETUP, 0ll);
        sg.whole = sg.r0 == 0 && sg.r1 == sg.s.recs;
        sg.c_first = sg.c_last = blockIdx.x;
        if (!sg.whole) {                              // the CTAs that hold its first and last record
            sg.c_first = (int)divide(at - place + SETUP, run);
            sg.c_last = (int)divide(at - place + SETUP + sg.s.recs - 1, run);
        }
        at += stop - place;
        return sg.r1 > sg.r0;
    };

    Segment first;
    {
        const long long run = max(divide(total + gridDim.x - 1, gridDim.x), (long long)MIN_UNITS);
        long long at = run * blockIdx.x;
        const long long end = min(at + run, total);
        if (at >= end) return;
        Segment& sg = first;
        sg.h = (int)divide(at, per_head);
        long long rest = at - sg.h * per_head;
        sg.b = -1;
        for (int b0 = 0; b0 < p.B; b0 += 32) {        // find the sequence: a warp-wide prefix sum of 32 at a time
            if (b0 > 0) {
                mine = units(b0);
                upto = prefix(mine);
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
        if (sg.b < 0) return;                         // (only if the lengths changed under the kernel)
        sg.s = sequence<NC>(p, sg.b);
        sg.chunk = (int)divide(rest, SETUP + sg.s.recs);
        const int place = (int)(rest - (long long)sg.chunk * (SETUP + sg.s.recs));
        if (!take(sg, at, place, end, run)) return;   // (a run that ends inside its first item's setup holds nothing)
        if (threadIdx.x == 0) { state->sg = sg; state->at = at; state->end = end; state->run = run; }
    }

    // ---- streaming: this warp's k-th record of a segment is r_first + k NW
    int n_rec = 0, rec_end = 0, r_first = 0, seq = 0;   // records of this warp; end of the records read; its first one; sequence
    int in_off = 0;                                   // ring offset of the next copy
    int page_now = 0, page_next = 0;
    const uint8_t* head_base = nullptr;               // this lane's 16 bytes of the kv-head's record in page 0
    bool bad_page = false;
    auto load_page = [&](int r) {
        int page = 0;
        if (r < rec_end)
            page = p.page_table ? __ldg(p.page_table + (long long)SKV_INDEX(seq, p.B) * p.max_pages + SKV_INDEX(r, p.max_pages)) : seq * p.max_pages + r;
        return checked_page(page, p.num_pages, bad_page);
    };
    auto issue = [&](int k, auto certain_constant) {  // (certain: the caller knows that record k exists)
        constexpr bool CERTAIN = decltype(certain_constant)::value;
        if ((k & 31) == 0) {                          // pages of the next 32 records, one per lane, fetched 32 ahead
            const int r = r_first + (k + lane) * NW;
            page_now = k ? page_next : load_page(r);
            page_next = load_page(r + 32 * NW);
        }
        const int page = __shfl_sync(0xffffffffu, page_now, k & 31);
        if (CERTAIN || k < n_rec) {
            const uint8_t* src = head_base + (unsigned long long)(uint32_t)SKV_INDEX(page, p.num_pages) * p.sp;
            const uint32_t dst = ring + SKV_INDEX(in_off, (STAGES - 1) * REC + 1) + lane * 16;
#pragma unroll
            for (int i = 0; i < REC / 512; ++i) cp_async16(dst + i * 512, src + i * 512);
            cp_async16_if(dst + REC / 512 * 512, src + REC / 512 * 512, lane < REC % 512 / 16);
        }
        cp_async_commit();
        in_off = in_off == (STAGES - 1) * REC ? 0 : in_off + REC;
    };
    // first copies of a segment, its query rows (as they are, to where the operands made of them will lie) ahead of the records
    auto begin = [&](const Segment& x, uint8_t* q_to) {
        const int total_cols = x.s.nq * p.G;
        if (warp < NT) {
            const int c = x.chunk * NC + warp * 8 + g;
            const bool in = c < total_cols;
            const long long row = in ? ((long long)SKV_INDEX(x.s.q0 + c / p.G, p.T) * p.Hq + SKV_INDEX(x.h * p.G + c % p.G, p.Hq)) * D : 0;
#pragma unroll
            for (int w = 0; w < W; ++w)
                cp_async16_or_zero(smem_u32(q_to) + ((warp * W + w) * 32 + lane) * 16, static_cast<const __half*>(p.q) + row + w * 32 + tq * 8, in);
        }
        // the last token that any column of the item sees bounds the records that are read
        const int i_last = (min(total_cols, (x.chunk + 1) * NC) - 1) / p.G;
        const int seen = max(0, x.s.len - x.s.nq + i_last + 1);
        seq = x.b;
        rec_end = min(x.r1, (seen + 15) >> 4);
        r_first = x.r0 + warp;
        n_rec = max(0, (rec_end - r_first + NW - 1) / NW);
        in_off = 0;
        head_base = p.pool + x.h * p.sh + lane * 16;
#pragma unroll
        for (int k = 0; k < STAGES - 1; ++k) issue(k, Constant<false>{});
    };
    begin(first, query);

    for (int item = 0;; ++item) {
        // ---- query columns of this item, as operands in shared memory, made by one warp per n-tile: [n-tile][group][lane] 16
        // bytes, then two words of the bias operand and the factor of column g per lane
        uint8_t* q_here = query + (item & 1) * S::QUERY;
        const uint32_t q_ops = smem_u32(q_here);
        uint32_t* q_words = reinterpret_cast<uint32_t*>(q_here + NT * W * 512);       // [n-tile][3][32]
        if (warp < NT) {
            const int nt = warp;
            cp_async_wait<STAGES - 2>();
            float x[W][8];
            float amax = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const uint4 raw = *reinterpret_cast<const uint4*>(q_here + ((nt * W + w) * 32 + lane) * 16);
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
                uint32_t b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {          // nibbles i and i + 4; even i are masked out of bits 0-3, odd out of 4-7
                    const float k = (i & 1) ? up : up * 16.f;
                    b[i] = pack_half2(x[w][i] * k, x[w][i + 4] * k);
                }
                *reinterpret_cast<uint4*>(q_here + ((nt * W + w) * 32 + lane) * 16) = make_uint4(b[0], b[1], b[2], b[3]);
                float a = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&b[i]));
                    a += (f.x + f.y) * ((i & 1) ? 1.f : 0.0625f);
                }
                a += __shfl_xor_sync(0xffffffffu, a, 1);
                a += __shfl_xor_sync(0xffffffffu, a, 2);
                sum[w] = a * -7.62939453125e-06f;       // -8 * 2^-20
            }
            // the bias of a column's scores, sum_w ks_w sum[w], is a product of its own over the groups, the sums split into three
            // bf16 terms (24 bits): k index 2 tq + {0, 1} (+ 8) is group 2 (tq & 1) + {0, 1} (D = 64: {0, 1}) of term tq >> 1 (+ 2)
            uint32_t term[3][W / 2];
#pragma unroll
            for (int i = 0; i < 3; ++i)
#pragma unroll
                for (int w = 0; w < W; w += 2) {
                    term[i][w / 2] = pack_bf16(sum[w], sum[w + 1]);
                    sum[w] -= bf_lo(term[i][w / 2]);
                    sum[w + 1] -= bf_hi(term[i][w / 2]);
                }
            uint32_t b0, b1 = 0u;
            if constexpr (W == 4) {
                b0 = (tq & 1) ? (tq < 2 ? term[0][1] : term[1][1]) : (tq < 2 ? term[0][0] : term[1][0]);
                b1 = tq == 0 ? term[2][0] : tq == 1 ? term[2][1] : 0u;
            } else {
                b0 = tq == 0 ? term[0][0] : tq == 1 ? term[1][0] : tq == 2 ? term[2][0] : 0u;
            }
            q_words[(nt * 3 + 0) * 32 + lane] = b0;
            q_words[(nt * 3 + 1) * 32 + lane] = b1;
            q_words[(nt * 3 + 2) * 32 + lane] =         // 2^20 / up, which may pass fp32's range by itself, and the softmax scale
                __float_as_uint(p.scale_log2 * __uint_as_float((uint32_t)(e + 121) << 23) * 65536.f);
        }
        __syncthreads();
        uint32_t qbias[NT][2];
        float factor[NT][2];
        int limit[NT][2];                             // end of the tokens of this segment that columns 2tq, 2tq + 1 see
        int n_full, end_tok;                          // this warp's records that every column sees whole; end of the tokens that are here
        {
            const int len = state->sg.s.len, r1 = state->sg.r1, col0 = state->sg.chunk * NC;
            const int before = len - state->sg.s.nq + 1;   // query token i sees before + i tokens
            const int cols = min(state->sg.s.nq * p.G - col0, NC);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    qbias[nt][j] = q_words[(nt * 3 + j) * 32 + lane];
                    factor[nt][j] = __uint_as_float(q_words[(nt * 3 + 2) * 32 + (2 * tq + j) * 4]);
                    const int cj = nt * 8 + 2 * tq + j;
                    limit[nt][j] = min(cj < cols ? before + (col0 + cj) / p.G : len, r1 * 16);
                }
            const int all = max(0, min(before + col0 / p.G, r1 * 16));
            n_full = min(n_rec, max(0, (all / 16 - r_first + NW - 1) / NW));
            end_tok = min(len, rec_end * 16);
        }

        // o[nt][2w + m][j], [j + 2]: channels 32w + 4g + 2m, + 1 of column 8nt + 2tq + j
        float o[NT][2 * W][4], ref[NT][2], lrun[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2 * W; ++c) o[nt][c][0] = o[nt][c][1] = o[nt][c][2] = o[nt][c][3] = 0.f;
            ref[nt][0] = ref[nt][1] = NOTHING;
            lrun[nt][0] = lrun[nt][1] = 0.f;
        }
        uint32_t vdown[W / 2];                         // the groups' powers of two, two a word: no scale of this warp so far reaches 2 times it
#pragma unroll
        for (int i = 0; i < W / 2; ++i) vdown[i] = DOWN_NONE | DOWN_NONE << 16;

        uint32_t big = 0u;                             // MOVE: a reference of this warp is far from zero
        const int tok_a = 4 * (g >> 1) + (g & 1);      // rows g and g + 8 of the score tile are tokens tok_a and tok_a + 2
        int out_off = 0;                               // ring offset of the record that is worked on
        auto record = [&](int k, auto masked_constant) {
            constexpr bool MASKED = decltype(masked_constant)::value;
            cp_async_wait<STAGES - 2>();
            __syncwarp();                              // record k is here, and every lane is done with record k - 1
            issue(k + STAGES - 1, Constant<!MASKED>{});
            const uint32_t rec = ring + SKV_INDEX(out_off, (STAGES - 1) * REC + 1);
            out_off = out_off == (STAGES - 1) * REC ? 0 : out_off + REC;
            const int t0 = (r_first + k * NW) * 16 + tok_a;   // this lane's tokens: t0, t0 + 2
            auto hidden = [&](int j, int nt) { return t0 + (j & 2) >= limit[nt][j & 1]; };

            // scores: rows g, g + 8 = places g, g + 8 of the record
            float s[NT][4];
            uint32_t va_scale[W / 2], vb_scale[W / 2]; // value scales of the lane's two tokens
            {
                uint32_t ka[W], kb[W], sa[W], sb[W];   // sa, sb: W key scales, then W value scales, two a word
                lds<D / 8>(rec + lane * (D / 8), ka);
                lds<D / 8>(rec + 4 * D + lane * (D / 8), kb);
                lds<D / 8>(rec + 16 * D + g * (D / 8), sa);
                lds<D / 8>(rec + 17 * D + g * (D / 8), sb);
                const uint32_t ba = W == 4 && (tq & 1) ? sa[1] : sa[0], bb = W == 4 && (tq & 1) ? sb[1] : sb[0];
                const uint32_t bias[4] = {ba, bb, ba, bb};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma_bf16_0(s[nt], bias, qbias[nt][0], qbias[nt][1]);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t a8 = ka[w] >> 8, b8 = kb[w] >> 8;
                    const uint32_t m0[4] = {ka[w] & 0x000f000fu, kb[w] & 0x000f000fu, ka[w] & 0x00f000f0u, kb[w] & 0x00f000f0u};
                    const uint32_t m1[4] = {a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u, b8 & 0x00f000f0u};
                    const float ska = group_scale(sa, 0, w), skb = group_scale(sb, 0, w);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        uint32_t qb[4];
                        lds<16>(q_ops + ((nt * W + w) * 32 + lane) * 16, qb);
                        float acc[4];
                        mma_f16_0(acc, m0, qb[0], qb[1]);
                        mma_f16(acc, m1, qb[2], qb[3]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[nt][j] = fmaf(acc[j], j < 2 ? ska : skb, s[nt][j]);
                    }
                }
#pragma unroll
                for (int i = 0; i < W / 2; ++i) { va_scale[i] = sa[W / 2 + i]; vb_scale[i] = sb[W / 2 + i]; }
            }
            if (MASKED) {                              // scales behind the end may hold anything
#pragma unroll
                for (int i = 0; i < W / 2; ++i) {
                    if (t0 >= end_tok) va_scale[i] = 0u;
                    if (t0 + 2 >= end_tok) vb_scale[i] = 0u;
                }
            }
            // Weights are exp2(s - ref), ref any number that keeps them in fp16's range, value scales are taken relative to their
            // group's power of two: both move only when a score or a scale leaves the room there is, seldom after the first record.
            uint32_t large = big;
            float t[NT][4], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < W / 2; ++i) {
                va_scale[i] = mul_bf16x2(va_scale[i], vdown[i]);
                vb_scale[i] = mul_bf16x2(vb_scale[i], vdown[i]);
                large |= va_scale[i] | vb_scale[i];
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    t[nt][j] = fmaf(s[nt][j], factor[nt][j & 1], -ref[nt][j & 1]);
                    if (MASKED && hidden(j, nt)) t[nt][j] = -INFINITY;
                    top = fmaxf(top, t[nt][j]);
                }
            if (__any_sync(0xffffffffu, top > WEIGHT_MAX || (large & MOVE) != 0u)) {
                // the largest exponent of each group's value scales so far (a scale that is NaN or infinite is for those who see
                // it, not for the bound); the scales themselves are fetched once more
                uint32_t ra[W], rb[W];
                lds<D / 8>(rec + 16 * D + g * (D / 8), ra);
                lds<D / 8>(rec + 17 * D + g * (D / 8), rb);
                unsigned e[W];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const int half = (w & 1) * 16;
                    const uint32_t xa = MASKED && t0 >= end_tok ? 0u : ra[W / 2 + (w >> 1)] >> half & 0xffffu;
                    const uint32_t xb = MASKED && t0 + 2 >= end_tok ? 0u : rb[W / 2 + (w >> 1)] >> half & 0xffffu;
                    e[w] = max(xa < 0x7f80u ? xa >> 7 : 0u, xb < 0x7f80u ? xb >> 7 : 0u);
                }
#pragma unroll
                for (int w = 0; w < W; ++w) e[w] = __reduce_max_sync(0xffffffffu, e[w]);   // (one behind the other, no branch between)
                float fall[W];                         // what O of a group that grows is multiplied by, exactly while nothing underflows
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const int half = (w & 1) * 16, old = exponent_of(vdown, w);
                    const int now = (int)e[w] > old ? min((int)e[w] + SCALE_ROOM, 253) : old;
                    fall[w] = now - old < 127 ? __uint_as_float((uint32_t)(127 - now + old) << 23) : 0.f;
                    vdown[w >> 1] = (vdown[w >> 1] & (0xffff0000u >> half)) | (uint32_t)(254 - now) << (7 + half);
                }
#pragma unroll
                for (int i = 0; i < W / 2; ++i) {
                    va_scale[i] = mul_bf16x2(MASKED && t0 >= end_tok ? 0u : ra[W / 2 + i], vdown[i]);
                    vb_scale[i] = mul_bf16x2(MASKED && t0 + 2 >= end_tok ? 0u : rb[W / 2 + i], vdown[i]);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        // the column's largest score (from the score itself: t has lost it against NOTHING); far from zero scores
                        // and references are rounded alike, or t would be off by as much as a step of the score
                        if (big) {
#pragma unroll
                            for (int i = j; i < 4; i += 2)
                                if (!MASKED || !hidden(i, nt)) t[nt][i] = __fsub_rn(__fmul_rn(s[nt][i], factor[nt][j]), ref[nt][j]);
                        }
                        float sx = -INFINITY, tx = fmaxf(t[nt][j], t[nt][j + 2]);
#pragma unroll
                        for (int i = j; i < 4; i += 2)
                            if (!MASKED || !hidden(i, nt)) sx = fmaxf(sx, s[nt][i] * factor[nt][j]);
#pragma unroll
                        for (int x = 4; x < 32; x *= 2) {
                            sx = fmaxf(sx, __shfl_xor_sync(0xffffffffu, sx, x));
                            tx = fmaxf(tx, __shfl_xor_sync(0xffffffffu, tx, x));
                        }
                        float c = 1.f;
                        if (tx > WEIGHT_MAX) {         // (the same for all lanes of a column)
                            const float moved = __fsub_ru(sx, WEIGHT_AIM);
                            if (fabsf(moved) >= BIG_SCORE) big = MOVE;
                            c = fast_exp2(ref[nt][j] - moved);
                            ref[nt][j] = moved;
                            lrun[nt][j] *= c;
#pragma unroll
                            for (int i = j; i < 4; i += 2) {
                                t[nt][i] = big ? __fsub_rn(__fmul_rn(s[nt][i], factor[nt][j]), moved) : fmaf(s[nt][i], factor[nt][j], -moved);
                                if (MASKED && hidden(i, nt)) t[nt][i] = -INFINITY;
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 2 * W; ++i) { o[nt][i][j] *= c * fall[i >> 1]; o[nt][i][j + 2] *= c * fall[i >> 1]; }
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < 4; ++j) t[nt][j] = fast_exp2(t[nt][j]);
                lrun[nt][0] += t[nt][0] + t[nt][2];
                lrun[nt][1] += t[nt][1] + t[nt][3];
            }

            // values: plane j holds tokens 4tq + 2j and + 1 of the lane's channels, matching the weights' rows after their move.
            // Rows g take a whole byte, even channel + 16 odd channel, rows g + 8 the odd channel in its place: one logic operation
            // less than two nibbles cost, and the difference of the rows is the even channel.  The 8 of the codes is taken out here,
            // exactly (a packed addition of whole multiples of 2^-24; measured 10 % faster than taking it out of O by products).
            uint32_t va[W], vb[W];
            lds<D / 8>(rec + 8 * D + lane * (D / 8), va);
            lds<D / 8>(rec + 12 * D + lane * (D / 8), vb);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const uint32_t sel = (w & 1) ? 0x7632u : 0x5410u;
                const uint32_t x = __byte_perm(va[w >> 1], va[W / 2 + (w >> 1)], sel);
                const uint32_t y = __byte_perm(vb[w >> 1], vb[W / 2 + (w >> 1)], sel);
                const uint32_t x8 = __byte_perm(x, 0u, 0x4341u), y8 = __byte_perm(y, 0u, 0x4341u);
                const uint32_t m0[4] = {add_f16x2(x & 0x00ff00ffu, MINUS_136), add_f16x2(x & 0x00f000f0u, MINUS_128),
                                        add_f16x2(y & 0x00ff00ffu, MINUS_136), add_f16x2(y & 0x00f000f0u, MINUS_128)};
                const uint32_t m1[4] = {add_f16x2(x8, MINUS_136), add_f16x2(x8 & 0x00f000f0u, MINUS_128),
                                        add_f16x2(y8, MINUS_136), add_f16x2(y8 & 0x00f000f0u, MINUS_128)};
                const float sva = group_scale(va_scale, 0, w), svb = group_scale(vb_scale, 0, w);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float z[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        z[j] = t[nt][j] * (j < 2 ? sva : svb);
                        if (MASKED && hidden(j, nt)) z[j] = 0.f;   // a live token's NaN is not for columns that do not see it
                    }
                    const uint32_t b0 = movmatrix_trans(pack_half2(z[0], z[1]));
                    const uint32_t b1 = movmatrix_trans(pack_half2(z[2], z[3]));
                    mma_f16(o[nt][2 * w], m0, b0, b1);
                    mma_f16(o[nt][2 * w + 1], m1, b0, b1);
                }
            }
        };
        // Records that every column sees whole, with another to fetch behind them; then those at the end.
        const int n_mine = n_rec;
        int k = 0;
        for (; k < min(n_full, n_mine - (STAGES - 1)); ++k) record(k, Constant<false>{});
        for (; k < n_mine; ++k) record(k, Constant<true>{});
        cp_async_wait<0>();
        __syncwarp();

        // ---- this warp's sums to shared memory (their registers are free then for what follows)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int c = nt * 8 + 2 * tq + j;
                float l = lrun[nt][j];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (g == 0) merge_ml[warp * NC + c] = make_float2(ref[nt][j], l * exp2_of(SUMS_DOWN));
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    // rows g hold (even + 16 odd) 2^-24, rows g + 8 odd 2^-20, both less the group's power of two
                    const int e = exponent_of(vdown, w);
                    const float up = __uint_as_float(e ? (uint32_t)e << 23 : 0x400000u);   // 2^(e - 127)
                    float4 v;
                    const float odd = up * exp2_of(20 + SUMS_DOWN), even = up * exp2_of(24 + SUMS_DOWN);
                    v.x = (o[nt][2 * w][j] - o[nt][2 * w][j + 2]) * even;
                    v.y = o[nt][2 * w][j + 2] * odd;
                    v.z = (o[nt][2 * w + 1][j] - o[nt][2 * w + 1][j + 2]) * even;
                    v.w = o[nt][2 * w + 1][j + 2] * odd;
                    *reinterpret_cast<float4*>(merge + (warp * NC + c) * S::ROW + 32 * w + 4 * g) = v;
                }
            }

        // ---- the next segment's first records are on their way while this one is written
        const Segment done = state->sg;
        Segment next = done;
        long long at = state->at;
        const long long end = state->end, run = state->run;
        bool more = at < end;
        if (more) {
            if (++next.chunk >= next.s.chunks) {
                next.chunk = 0;
                do {
                    if (++next.b == p.B) { next.b = 0; ++next.h; }
                    next.s = sequence<NC>(p, next.b);
                } while (next.s.chunks == 0 && next.h < p.Hkv);
                more = next.h < p.Hkv;                 // (`at` < end, so it is, while the lengths stay as they are)
            }
            more = more && take(next, at, 0, end, run);   // (a run's last item may have no record in it)
        }
        if (more) begin(next, query + (~item & 1) * S::QUERY);
        const int col0 = done.chunk * NC, cols = min(done.s.nq * p.G - col0, NC);

        // ---- merge the warps
        const long long slot = SKV_INDEX(2 * (int)blockIdx.x + (done.r0 == 0 ? 1 : 0), 2 * MAX_GRID);
        __syncthreads();
        for (int i = threadIdx.x; i < cols * (D / 4); i += THREADS) {
            const int c = SKV_INDEX(i / (D / 4), NC), d = i % (D / 4) * 4;
            float2 ml[NW];
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                ml[w] = merge_ml[w * NC + c];
                M = fmaxf(M, ml[w].x);
            }
            float L = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float wt = fast_exp2(ml[w].x - M);
                const float4 v = *reinterpret_cast<const float4*>(merge + (w * NC + c) * S::ROW + d);
                L = fmaf(ml[w].y, wt, L);
                acc.x = fmaf(v.x, wt, acc.x); acc.y = fmaf(v.y, wt, acc.y);
                acc.z = fmaf(v.z, wt, acc.z); acc.w = fmaf(v.w, wt, acc.w);
            }
            if (done.whole) {
                store_out(p, done, D, col0 + c, d, acc, L);
            } else {
                *reinterpret_cast<float4*>(p.partial_o + (slot * NC + c) * D + d) = acc;
                if (d == 0) *reinterpret_cast<float2*>(p.partial_ml + (slot * NC + c) * 2) = make_float2(M, L);
            }
        }
        __syncthreads();

        // ---- an item that spans CTAs: the last one to arrive adds up
        if (!done.whole) {
            const int n = done.c_last - done.c_first + 1;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                int* ticket = p.tickets + SKV_INDEX(done.c_first, (int)gridDim.x);
                const int last = atomicAdd(ticket, 1) == n - 1;
                if (last) *ticket = 0;                 // ready for the next launch on this workspace
                state->last = last;
            }
            __syncthreads();
            if (state->last) {
                __threadfence();
                combine<D, NC, THREADS>(p, done, n, cols, col0, merge);
            }
            __syncthreads();
        }
        if (!more) break;
        if (threadIdx.x == 0) { state->sg = next; state->at = at; }   // (read behind the barrier that the operands need)
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
    const long long units = p.Hkv * (p.cu_q ? chunks : (long long)p.B * ((p.G + NC - 1) / NC)) * (S::SETUP + ((long long)p.N + 15) / 16);
    long long grid = sm_count(device) < MAX_GRID ? sm_count(device) : MAX_GRID;
    if (grid > (units + MIN_UNITS - 1) / MIN_UNITS) grid = (units + MIN_UNITS - 1) / MIN_UNITS;
    Params q = p;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (!q.status) q.status = reinterpret_cast<int*>(ws);
    q.tickets = reinterpret_cast<int*>(ws + TICKET_OFF);
    q.partial_ml = reinterpret_cast<float*>(ws + PARTIAL_OFF);
    q.partial_o = q.partial_ml + 2ll * MAX_GRID * NC * 2;
    SKV_CUDA_TRY(launch_pdl(gqa_decode_kv4_kernel<D, NT>, dim3((unsigned)grid), dim3(S::THREADS), S::SMEM, stream, q));
    SKV_CUDA_TRY(cudaGetLastError());
    return SKV_OK;
}

static size_t workspace_bytes(int D) { return PARTIAL_OFF + 2ull * MAX_GRID * 16 * (2 + D) * 4; }   // 16 columns: NT = 2

}  // namespace kv4
}  // namespace skv

using namespace skv;

extern "C" {

size_t skv_gqa_decode_kv4_workspace_bytes(int D) { return D == 64 || D == 128 ? kv4::workspace_bytes(D) : 0; }

int skv_gqa_decode_kv4(const void* q, int q_is_bf16, const void* pool, const int* page_table, const int* seq_lens,
                       const int* cu_q, void* out, int out_is_bf16, void* workspace, size_t workspace_bytes, int T, int B, int N,
                       int Hq, int Hkv, int D, int max_pages, int num_pages, long long pool_stride_page,
                       long long pool_stride_head, float scale, int* status, int device, void* stream) {
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
    if (pool_stride_page < 0 || pool_stride_page > 0xffffffffll)
        return fail(SKV_ERR_UNSUPPORTED, "a page stride of %lld bytes is not supported", pool_stride_page);
    if ((long long)T * (Hq / Hkv) > 0x7fffffffll - 16) return fail(SKV_ERR_UNSUPPORTED, "too many query rows");
    if (!workspace || workspace_bytes < kv4::workspace_bytes(D))
        return fail(SKV_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %zu required", workspace_bytes, kv4::workspace_bytes(D));
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(SKV_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(SKV_ERR_CUDA, "cannot switch to device %d", device);
    kv4::Params p = {};
    p.q = q; p.out = out; p.pool = static_cast<const uint8_t*>(pool);
    p.sp = (uint32_t)pool_stride_page; p.sh = pool_stride_head;
    p.page_table = page_table; p.seq_lens = seq_lens; p.cu_q = cu_q;
    p.B = B; p.T = T; p.N = N; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv;
    p.max_pages = max_pages; p.num_pages = num_pages; p.q_bf16 = q_is_bf16; p.out_bf16 = out_is_bf16;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.status = status;
    // Columns per pass over the cache, 8 or 16.  A pass of 16 takes 7/4 of one of 8, so it pays where it saves that many of the
    // mean sequence's (query token, head) pairs' passes.  Measured with 8 | 16, D = 128, us: 16 pairs of 8 sequences of 8192
    // tokens 42.5 | 39.9, 24 pairs 57.1 | 62.0, 32 pairs 71.6 | 63.5; 512 of one of 4096 76.2 | 65.7.  It loses where the work is
    // small (16 pairs of one sequence of 16384: 18.7 | 22.2), which the host does not see, for it does not know the lengths; and
    // it judges by the mean, so one chunk of a prompt among single tokens may get 8.
    const long long pairs = (long long)p.G * ((T + B - 1) / B);
    const bool wide = 7 * ((pairs + 15) / 16) < 4 * ((pairs + 7) / 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (D == 128) return wide ? kv4::launch<128, 2>(p, workspace, device, st) : kv4::launch<128, 1>(p, workspace, device, st);
    return wide ? kv4::launch<64, 2>(p, workspace, device, st) : kv4::launch<64, 1>(p, workspace, device, st);
}

}  // extern "C"

SKV_BOUNDS_GETTER(skv_debug_bounds_gqa_decode_kv4)
