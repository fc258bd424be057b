// Group normalisation over a ragged batch with what follows it in a residual block, in the norm's own passes:
//
//   y = drop(act((x - mean[s,g]) * rstd[s,g] * weight + bias (+ residual)))
//
// Rows are points, channels lie last.  mean and rstd are the statistics of the rows of sample s and the W = C / G consecutive
// channels of group g (G = 1: the ragged layer norm, G = C: the instance norm); act is the identity, ReLU, SiLU or the
// erf form of GELU; drop is the dropout of philox.cuh by element (y's row-major index).
//
// Backward, with z the activation's argument (made again from x, not stored), xh = (x - mean) * rstd and n = rows_s * W:
//   gz = drop'(g) * act'(z),   dresidual = gz,   dbias[c] = sum over rows of gz,   dweight[c] = sum over rows of gz * xh,
//   gh = gz * weight,   dx = rstd * (gh - sum_{s,g}(gh) / n - xh * sum_{s,g}(gh * xh) / n).
//
// Everything is held in fp32 between one read of an element and its one rounding, but for the statistics, which are fp64 from the element
// on: the sign of a ReLU's argument hangs on them, and where 32 bits summed them (1e-8 of a deviation off), about one of 70 million
// elements came out on the other side, each of which moves dbias by a whole gradient.
//
// Both directions take two passes over the rows, with sums between them, in one launch (behind a small one that lays the samples
// out).  A chunk is `rows` consecutive rows; a piece is what a chunk has of one sample, piece chunk + s (pieces are ordered, and
// the next one has a higher chunk or a higher sample by one).  Blocks take tickets, in ascending order, one at a time:
//   sums of a chunk  two sums per channel and piece, whatever the group's width, and from them two per group
//   apply of a chunk the second pass, once the sums of its samples are there
//   affine           dweight and dbias of some channels, once those of all samples are
// A sample's records of groups are merged by every block that applies rows of it, for itself: one turn through the L2 from the last
// piece to the first row, where one block that merges for all makes it two.  Where records are many (`window` pieces), the block that
// brings the last piece of a window merges these first.  Who merges does not matter to the result: records are merged in a fixed
// order, and no float is ever added by an atomic.  A ticket waits only for tickets before it, which blocks that run have taken, and
// sums wait for nothing: there is no deadlock, however few blocks are resident at once (a stream with a part of the chip).
// Tickets are ordered so that a sample is applied some chunks after its sums, in the hope that the wait for them is over by then.
//
// What is summed:
//   forward   mean and sum of squares about it.  A block sums x - k and its square, k the channel's value in the piece's first row:
//             as k is one of the n summed values, (k - mean)^2 is at most their sum of squares M2, and what cancels in
//             sum (x - k)^2 - n (mean - k)^2 is at most (n + 1) M2: n + 1 roundings of 2^-53 at worst.
//   backward  gz and gz * xh.
#pragma once
#include <algorithm>
#include <atomic>

#include "philox.cuh"
#include "rowwise.cuh"
#include "tcgen05.cuh"   // (the clock and the limit of bounded waits)

namespace pcx {

constexpr int NA_THREADS = 256;
constexpr int NA_BLOCKS = 3;          // of the kernel without the ring, on a multiprocessor
constexpr unsigned NA_STATUS = 32u;   // of a wait that ran out
constexpr int AFFINE_CHANNELS = 8;    // of a ticket
enum { TICKET = 0, WINDOWS_DONE = 1, WINDOWS = 2, CONTROL_WORDS = 4 };
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

// The chunks of a sample: b0 .. b1 have rows of it (b1 < b0: none), first .. next - 1 end in it, and these are applied from
// ticket `at` on.
struct Span { int b0, b1, first, next, at; };

struct NormAct {
    const void *x, *residual, *g;
    void *y, *dx, *dresidual;
    const float *weight, *bias;
    double *mean, *rstd;           // (S, G)
    float *dweight, *dbias;
    int64_t *offsets;              // (S + 1)
    Span *spans;                   // (S)
    float2 *rec;                   // backward (pieces, C): sums of gz and gz * xh
    double2 *scratch;              // forward, without the ring (blocks, C): mean and M2 of the piece that a block is at
    void *of_piece, *of_window;    // (pieces, G), (windows, G) of Record: the same of groups, the sums with the channels' weights
    int *control;                  // the words above, then windows that each sample has, pieces that each window has
    unsigned int *status;
    int64_t N, S;
    int C, G, W, rows, chunks, window, lag, act;
    int V, phase_bits;             // the ring's rows: 1 << phase_bits rows side by side, V channels
    int tile_rows, sums_tile_rows, stages, stage_bytes;   // of the ring
    uint32_t by_width;             // c / W = c * by_width >> 32 (c * W < 2^32); W = 1: c
    double eps;
    Dropping drop;
};

// One direction for rows of T (norm_act_*.cu); `vn` channels a lump.
template <typename T>
int norm_act_rows(const NormAct &p, int vn, bool backward, cudaStream_t stream);

#ifdef __CUDACC__
namespace {

__device__ __forceinline__ int *sample_count(const NormAct &p) { return p.control + CONTROL_WORDS; }
__device__ __forceinline__ int *window_count(const NormAct &p) { return sample_count(p) + p.S; }
// Windows are `window` pieces of a sample; they are numbered as pieces are: first_window + its windows before.
__host__ __device__ inline int64_t windows_in_all(int64_t chunks, int64_t S, int window) { return chunks / window + S + 1; }
__device__ __forceinline__ int64_t first_window(const NormAct &p, const Span &v, int64_t s) { return v.b0 / p.window + s; }
__device__ __forceinline__ int windows_of(const NormAct &p, const Span &v) { return (v.b1 - v.b0) / p.window + 1; }

// The channel of the first of a ring's row's, or of any.
__device__ __forceinline__ int channel_of(const NormAct &p, int v) { return p.phase_bits ? v % p.C : v; }
__device__ __forceinline__ int group_of(const NormAct &p, int c) { return p.W == 1 ? c : (int)__umulhi((uint32_t)c, p.by_width); }

// ------------------------------------------------------------ activations ----
__device__ __forceinline__ float ex2(float v) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v));
    return e;
}
__device__ __forceinline__ float rcp(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// 1 / (1 + exp(-z)): right to a part of its value for all z down to exp's range (zero from z = -87 on), as the reciprocal is of one number.
// (One for two, by their product, wants exp(-z) bounded by 2^62, and takes as long: forward with dropout 134 us for 135, backward 230 for 221,
// 1.1 million rows of 64 channels, bf16.)
__device__ __forceinline__ float2 sigmoid2(float2 z) {
    const float2 t = mul2(z, both(-1.4426950408889634f)), e = add2(both(1.f), make_float2(ex2(t.x), ex2(t.y)));
    return make_float2(rcp(e.x), rcp(e.y));
}

// The normal distribution's function and density.  With u = |z| and t = 1 / (1 + c u), Phi(-u) = exp(-u^2 / 2) t P(t), P a polynomial fitted
// to the quotient for all u by its least relative error (a weighted least-squares fit whose weights follow the error, on 4001
// points of t in 0 .. 1): so the tail, where GELU is z times Phi(-u), is right to the same part of it as the middle.  Relative error with its
// own roundings 3.3e-7 with ten coefficients, for rows of 32 bits, and 1e-6 with eight, a 200th of half a step of 16; the exponent's
// roundings add 2^-23 z^2, as z's own do.  One exponential serves both.
template <typename T>
__device__ __forceinline__ void normal2(float2 z, float2 &cdf, float2 &density) {
    constexpr bool WIDE = sizeof(T) == 4;
    constexpr int N = WIDE ? 10 : 8;
    constexpr float C = WIDE ? 0.315f : 0.325f;
    constexpr float p[10] = {WIDE ? 0.125666827f : 0.129656136f,   WIDE ? 0.125665396f : 0.129672810f,  WIDE ? 0.113254927f : 0.115494095f,  WIDE ? 0.0873554945f : 0.0935735404f,
                             WIDE ? 0.0617356598f : 0.0258780140f, WIDE ? -0.0127292043f : 0.0855680779f, WIDE ? 0.0785122886f : -0.113720231f, WIDE ? -0.153162092f : 0.0338778943f,
                             WIDE ? 0.0932994485f : 0.f,           WIDE ? -0.0195987169f : 0.f};
    const float2 v = fma2(make_float2(fabsf(z.x), fabsf(z.y)), both(C), both(1.f)), t = make_float2(rcp(v.x), rcp(v.y));
    const float2 h = mul2(mul2(z, z), both(-0.5f * 1.4426950408889634f));
    const float2 e = make_float2(ex2(h.x), ex2(h.y));   // exp(-z^2 / 2)
    float2 q = fma2(t, both(p[N - 1]), both(p[N - 2]));
#pragma unroll
    for (int i = N - 3; i >= 0; --i) q = fma2(t, q, both(p[i]));
    q = mul2(mul2(q, t), e);
    const float2 other = add2(both(1.f), neg2(q));
    cdf = make_float2(z.x < 0.f ? q.x : other.x, z.y < 0.f ? q.y : other.y);
    density = mul2(e, both(0.39894228f));
}

template <typename T>
__device__ __forceinline__ float2 act2(int act, float2 z) {
    if (act == ACT_RELU) return make_float2(relu(z.x), relu(z.y));
    if (act == ACT_SILU) return mul2(z, sigmoid2(z));
    if (act == ACT_GELU) {
        float2 cdf, density;
        normal2<T>(z, cdf, density);
        return mul2(z, cdf);
    }
    return z;
}
// g times the slope at z
template <typename T>
__device__ __forceinline__ float2 act2_backward(int act, float2 z, float2 g) {
    if (act == ACT_RELU) return make_float2(z.x > 0.f ? g.x : 0.f, z.y > 0.f ? g.y : 0.f);
    if (act == ACT_SILU) {   // s (1 + z (1 - s))
        const float2 v = sigmoid2(z);
        return mul2(g, fma2(mul2(z, v), add2(both(1.f), neg2(v)), v));
    }
    if (act == ACT_GELU) {
        float2 cdf, density;
        normal2<T>(z, cdf, density);
        return mul2(g, fma2(z, density, cdf));
    }
    return g;
}

// The last of `n` ascending values that `at(i)` gives which is not over `v`; -1 where all are.  A whole warp asks.
template <typename At>
__device__ __forceinline__ int64_t last_not_over(int64_t n, int64_t v, At at) {
    const int lane = threadIdx.x & 31;
    int64_t lo = 0, step = n;
    do {
        const int64_t end = min(n, lo + step);
        step = (end - lo + 31) / 32;
        const int64_t i = lo + lane * step;
        const unsigned found = __ballot_sync(0xffffffffu, i < end && at(i) <= v);
        if (!found) return lo - 1;   // (only before the first value)
        lo += (31 - __clz(found)) * step;
    } while (step > 1);
    return lo;
}

// The chunk that a ticket is for; true: its sums.
__device__ __forceinline__ bool take_ticket(const NormAct &p, int ticket, int *chunk) {
    // the last sample that is applied from this ticket on or from one before: its chunks, or sums of a later chunk
    const int64_t run = last_not_over(p.S, ticket, [&](int64_t s) { return (int64_t)p.spans[s].at; });
    *chunk = ticket;
    if (run < 0) return true;
    const Span v = p.spans[run];
    const bool sums = ticket - v.at >= v.next - v.first;
    *chunk = sums ? ticket - v.next : v.next - 1 - (ticket - v.at);   // (backwards: what was read last is still in the L2)
    return sums;
}

// ------------------------------------------------------------ columns ----
// Channels of a block: passes of `cols` lumps side by side, `lanes` rows.
struct Columns {
    int lumps, cols, lanes, passes, col, lane;
    __host__ __device__ __forceinline__ Columns(int C, int VN, int thread) {
        lumps = C / VN;
        passes = (lumps + NA_THREADS - 1) / NA_THREADS;
        cols = (lumps + passes - 1) / passes;
        lanes = NA_THREADS / cols;
        col = thread % cols, lane = thread / cols;
    }
};

// Barrier of the threads that work on rows (all but the ring's producer).
__device__ __forceinline__ void sync_workers() { asm volatile("bar.sync 1, %0;" ::"n"(NA_THREADS) : "memory"); }
__device__ __forceinline__ bool sync_workers_and(bool v) {
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(all) : "r"((uint32_t)v), "n"(NA_THREADS) : "memory");
    return all != 0;
}

struct Stats { double x, y; };   // mean and rstd, or the backward's two means

// Below zero, by roundings, is zero; a NaN stays one.
__device__ __forceinline__ double not_below_zero(double v) { return v < 0.0 ? 0.0 : v; }

// What a piece leaves of a group.  Forward: mean and M2.
template <bool BACKWARD>
struct Record;
template <>
struct __align__(16) Record<false> { double mean, m2; };
template <>
struct __align__(8) Record<true> { float x, y; };
__device__ __forceinline__ Record<true> load_record(const Record<true> *p) {
    const float2 v = __ldcg(reinterpret_cast<const float2 *>(p));
    return {v.x, v.y};
}
__device__ __forceinline__ Record<false> load_record(const Record<false> *p) {
    const double2 v = __ldcg(reinterpret_cast<const double2 *>(p));
    return {v.x, v.y};
}

// Records that follow one another: `count` of `unit` elements each, but for the first and the last.
template <bool BACKWARD>
struct Records {
    const Record<BACKWARD> *at;
    int count;
    double first, unit, last;
    double inverse;            // 1 / elements of all of them
};
// Rows lo .. hi by spans of `unit` rows, the first of which begins at `from`; `each` elements a row.
template <bool BACKWARD>
__device__ __forceinline__ Records<BACKWARD> records_of(const void *at, int64_t first, int count, int64_t lo, int64_t hi, int64_t from, int64_t unit, int each) {
    return {static_cast<const Record<BACKWARD> *>(at) + first, count, (double)((min(hi, from + unit) - lo) * each), (double)(unit * each),
            (double)((hi - (from + (count - 1) * unit)) * each), 1.0 / ((double)(hi - lo) * each)};
}

// Sums over records, of which a thread has some.  Forward about the first record's mean: a of differences from it, b of squares, each
// record's own among them.  Backward: of both sums.
template <bool BACKWARD>
struct RecordSums;
template <>
struct RecordSums<true> {
    static constexpr int AHEAD = 8;   // loads at once
    float a = 0.f, b = 0.f;
    __device__ __forceinline__ void add(const Records<true> &r, int stride, int g, int q, int deep) {
        const Record<true> *at = r.at + g;
        for (int i = q; i < r.count; i += AHEAD * deep) {
            Record<true> v[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) v[u] = i + u * deep < r.count ? load_record(at + (int64_t)(i + u * deep) * stride) : Record<true>{0.f, 0.f};
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) a += v[u].x, b += v[u].y;
        }
    }
    __device__ __forceinline__ Record<true> done(const Records<true> &) const { return {a, b}; }
};
template <>
struct RecordSums<false> {
    static constexpr int AHEAD = 8;
    double a = 0.0, b = 0.0, k = 0.0;
    __device__ __forceinline__ void add(const Records<false> &r, int stride, int g, int q, int deep) {
        const Record<false> *at = r.at + g;
        k = load_record(at).mean;
        for (int i = q; i < r.count; i += AHEAD * deep) {
            Record<false> v[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) v[u] = i + u * deep < r.count ? load_record(at + (int64_t)(i + u * deep) * stride) : Record<false>{k, 0.0};
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int j = i + u * deep;
                const double n = j == 0 ? r.first : j == r.count - 1 ? r.last : r.unit, d = v[u].mean - k, nd = n * d;
                a += nd, b += fma(nd, d, v[u].m2);
            }
        }
    }
    __device__ __forceinline__ Record<false> done(const Records<false> &r) const {
        const double off = a * r.inverse;
        return {k + off, not_below_zero(fma(-a, off, b))};
    }
};

// What a second pass needs of the groups that channels c0 .. c1 - 1 are in, from the sample's records, into `stats` (shared memory) by all
// workers: mean and rstd, or the backward's two means.  Every block does this for itself, with the sample's windows counted: a block
// that did it for all would keep them waiting for one more turn through the L2.  Threads stand side by side on the groups and, where
// there are fewer of them, in rows on the records.
template <bool BACKWARD>
__device__ __forceinline__ void merge_groups(const NormAct &p, const Records<BACKWARD> &r, int groups, Stats *stats, double2 *scratch) {
    const int wide = min(groups, NA_THREADS), at = threadIdx.x % wide, q = threadIdx.x / wide;
    const bool shuffles = wide < 32 && 32 % wide == 0;
    const int deep = NA_THREADS / wide;
    for (int base = 0; base < groups; base += wide) {
        const int g = base + at;
        RecordSums<BACKWARD> sums;
        if (g < groups && q < deep) sums.add(r, p.G, g, q, deep);
        if (shuffles) {   // a warp's rows first; then its first row has them
            for (int o = 16; o >= wide; o >>= 1) {
                sums.a += __shfl_xor_sync(0xffffffffu, sums.a, o), sums.b += __shfl_xor_sync(0xffffffffu, sums.b, o);
            }
        }
        const int rows = shuffles ? NA_THREADS / 32 : deep, step = shuffles ? 32 : wide;
        if (rows > 1) {
            scratch[threadIdx.x] = make_double2(sums.a, sums.b);
            sync_workers();
            if (q == 0)
#pragma unroll 4
                for (int i = 1; i < rows; ++i) {
                    const double2 v = scratch[i * step + at];
                    sums.a += v.x, sums.b += v.y;
                }
        }
        if (g < groups && q == 0) {
            if constexpr (BACKWARD) {
                stats[g] = {sums.a * r.inverse, sums.b * r.inverse};
            } else {
                const Record<false> v = sums.done(r);
                stats[g] = {v.mean, rsqrt(v.m2 * r.inverse + p.eps)};
            }
        }
        sync_workers();
    }
}

// Waits until a word is what a block before has to make it; at most a second, then it is reported, and the answer is false.
__device__ __forceinline__ bool wait_for(const int *word, int value, unsigned int *status) {
    __shared__ int there;
    sync_workers();
    if (threadIdx.x == 0) {
        int v = 0;
        const uint64_t t0 = tc::global_timer_ns();
        for (unsigned turn = 0;; ++turn) {
            asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(word) : "memory");
            if (v == value) break;
            if (turn % 64 == 63 && tc::global_timer_ns() - t0 > tc::WAIT_LIMIT_NS) {
                atomicOr(status, NA_STATUS);
                break;
            }
        }
        there = v == value;
    }
    sync_workers();
    return there;
}

// What the rows of a sample are mapped by, per channel of a pass, in shared memory: floats k of a lump's quad h lie side by side over the
// columns, so that a warp reads them without conflicts.  (In registers they were most of what a thread held: 24 to 40 floats.)
// z = (x - mu) a + b in both directions: mu is the mean rounded to 32 bits, and what that leaves of it is in b.  So z is off by roundings of its
// own terms, however many deviations the mean is from zero.  (With the mean in b whole, z = x a + b rounds by 2^-24 of |mean| / deviation.)
// Backward dx = gz a + m1 + (x - mu) m2, where m1 has the mean's rest too.
enum { K_A = 0, K_B = 1, K_MU = 2, K_M1 = 3, K_M2 = 4 };
struct Mapping {
    float a, b, mu, rest;
    __device__ __forceinline__ Mapping(double mean, double rstd, float w, float bias) {
        mu = (float)mean, a = (float)(rstd * w), rest = (float)(mean - mu);
        b = (float)fma(-(mean - mu), (double)a, (double)bias);
    }
};
template <int VN, bool BACKWARD>
struct Constants {
    static constexpr int QUAD = VN < 4 ? VN : 4, PAIRS = QUAD < 2 ? 1 : QUAD / 2, QUADS = VN / QUAD;
    float *at;
    Stats *stats;              // of the second pass: the groups'
    double2 *scratch;          // of merge_groups
    int64_t s = -1;            // whose they are
    int pass = -1;
    __device__ __forceinline__ void read(const Columns &l, int k, int h, float2 *out) const {
        // (volatile: read where they are used, in every round of a loop; taken out of it, as compilers would, they are registers again)
        const uint32_t q = tc::smem_u32(at + ((k * QUADS + h) * l.cols + l.col) * QUAD);
        float2 &a = out[0], &b = out[PAIRS - 1];
        if constexpr (QUAD == 4) asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(a.x), "=f"(a.y), "=f"(b.x), "=f"(b.y) : "r"(q) : "memory");
        else if constexpr (QUAD == 2) asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(a.x), "=f"(a.y) : "r"(q) : "memory");
        else asm volatile("ld.shared.f32 %0, [%1];" : "=f"(a.x) : "r"(q) : "memory");
        if (QUAD == 1) a.y = 0.f;
    }
    __device__ __forceinline__ void read_all(const Columns &l, int k, float2 *out) const {
#pragma unroll
        for (int h = 0; h < QUADS; ++h) {
            const float4 v = *reinterpret_cast<const float4 *>(at + ((k * QUADS + h) * l.cols + l.col) * 4);
            out[2 * h] = make_float2(v.x, v.y), out[2 * h + 1] = make_float2(v.z, v.w);
        }
    }
    // By all workers, once they have met.  `second`: of the second pass, for which the sample's records are waited for; false: in vain.
    template <bool PHASES = false>
    __device__ __forceinline__ bool load(const NormAct &p, const Columns &l, int64_t s_, int pass_, bool second) {
        const int c0 = pass_ * l.cols * VN, c1 = min(p.C, c0 + l.cols * VN), g0 = group_of(p, c0);
        float w = 1.f, bias = 0.f;   // of the thread's first channel: read before the wait
        double mean = 0.0, rstd = 0.0;
        const auto known = [&](int c) {
            if (p.weight) w = __ldg(p.weight + c), bias = __ldg(p.bias + c);
            if (BACKWARD) mean = __ldg(p.mean + s_ * p.G + group_of(p, c)), rstd = __ldg(p.rstd + s_ * p.G + group_of(p, c));
        };
        if (c0 + (int)threadIdx.x < c1) known(c0 + threadIdx.x);
        if (second) {
            const Span v = p.spans[s_];
            const int windows = windows_of(p, v);
            const Records<BACKWARD> r = records_of<BACKWARD>(p.of_window, first_window(p, v, s_) * p.G + g0, windows, p.offsets[s_], p.offsets[s_ + 1], (int64_t)v.b0 * p.rows, (int64_t)p.window * p.rows, p.W);
            if (!wait_for(sample_count(p) + s_, windows, p.status)) return false;
            merge_groups<BACKWARD>(p, r, group_of(p, c1 - 1) - g0 + 1, stats, scratch);
        }
        s = s_, pass = pass_;
        const int stride = QUADS * l.cols * QUAD;
        for (int t = threadIdx.x; t < c1 - c0; t += NA_THREADS) {
            if (t >= NA_THREADS) known(c0 + t);
            Stats m = {};
            if (second) m = stats[group_of(p, c0 + t) - g0];
            if (!BACKWARD) mean = m.x, rstd = m.y;
            const Mapping map(mean, rstd, w, bias);
            const float m2 = (float)(-m.y * rstd * rstd), m1 = (float)(-m.x * rstd) - map.rest * m2;
            for (int v = t; v < (PHASES ? p.V : t + 1); v += p.C) {
                float *to = at + ((v % VN / QUAD) * l.cols + v / VN) * QUAD + v % QUAD;
                to[K_A * stride] = map.a, to[K_B * stride] = map.b, to[K_MU * stride] = -map.mu;
                if (BACKWARD && second) to[K_M1 * stride] = m1, to[K_M2 * stride] = m2;
            }
        }
        sync_workers();
        return true;
    }
    // The statistics that were merged, for the caller: the block that has the sample's first chunk.
    __device__ __forceinline__ void put_stats(const NormAct &p, const Columns &l) const {
        const int c0 = pass * l.cols * VN, c1 = min(p.C, c0 + l.cols * VN), g0 = group_of(p, c0), groups = group_of(p, c1 - 1) - g0 + 1;
        for (int g = threadIdx.x; g < groups; g += NA_THREADS) p.mean[s * p.G + g0 + g] = stats[g].x, p.rstd[s * p.G + g0 + g] = stats[g].y;
    }
};

// ------------------------------------------------------------ sums of a piece ----
// Sums of entries q, q + step, .. of `lanes` that are `stride` apart, in eight chains: they do not wait for one another's additions, and
// one chain of 32 bits of all of them (85 lanes of four rows side by side, for 6 channels) rounds by 1e-6 of a gradient's size.
template <typename Two>
struct Chains {
    Two part[8];
    __device__ __forceinline__ Chains() {
#pragma unroll
        for (int u = 0; u < 8; ++u) part[u] = Two{};
    }
    __device__ __forceinline__ void add(const Two *from, int q, int step, int lanes, int stride) {
        for (; q < lanes; q += 8 * step) {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (q + u * step < lanes) {
                    const Two v = from[(q + u * step) * stride];
                    part[u].x += v.x, part[u].y += v.y;
                }
        }
    }
    __device__ __forceinline__ Two sum() const {
        Two v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u].x = part[u].x + part[u + 4].x, v[u].y = part[u].y + part[u + 4].y;
        Two all;
        all.x = (v[0].x + v[1].x) + (v[2].x + v[3].x), all.y = (v[0].y + v[1].y) + (v[2].y + v[3].y);
        return all;
    }
};

// Two sums per channel of a thread's rows (`part(i)`), folded over the block's row lanes; `out(c, a, b)` for every channel.
template <int VN, typename Two, typename Part, typename Out>
__device__ __forceinline__ void fold_lanes(const Columns &l, int pass, Two *fold, Part part, Out out) {
    sync_workers();   // (the piece before has been read)
#pragma unroll
    for (int i = 0; i < VN; ++i) fold[i * NA_THREADS + threadIdx.x] = part(i);
    sync_workers();
    for (int t = threadIdx.x; t < l.cols * VN; t += NA_THREADS) {
        const int i = t / l.cols, col = t % l.cols, lump = pass * l.cols + col;
        Chains<Two> chains;
        chains.add(fold + i * NA_THREADS + col, 0, 1, l.lanes, l.cols);
        const Two v = chains.sum();
        if (lump < l.lumps) out(lump * VN + i, v.x, v.y);
    }
}

// `U` rows of a thread's lumps, `lanes` apart; those behind the end are not read.  Rows are counted from the piece's first: a chunk's
// elements fit 32 bits.
template <typename T, int VN, int U>
struct Rows {
    Lump<T, VN> v[U];
    __device__ __forceinline__ void load(const T *__restrict__ col, int r, int n, int lanes, int C) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u * lanes < n) v[u].load(col + (r + u * lanes) * C);
    }
};

// Sums of a channel's x - k and of their squares, k its value in the piece's first row: 64 bits a rounding, from the element on.
template <int VN>
struct Moments {
    double a[VN], b[VN], k[VN];
    template <typename T>
    __device__ __forceinline__ explicit Moments(const Lump<T, VN> &first) {
#pragma unroll
        for (int i = 0; i < VN; ++i) a[i] = b[i] = 0.0, k[i] = first.get(i);
    }
    // Of a lump, the elements first <= i < end.
    template <typename T>
    __device__ __forceinline__ void add(const Lump<T, VN> &v, int first = 0, int end = VN) {
#pragma unroll
        for (int i = 0; i < VN; ++i) {
            const double d = i >= first && i < end ? (double)v.get(i) - k[i] : 0.0;
            a[i] += d, b[i] = fma(d, d, b[i]);
        }
    }
};
// The mean and M2 of n values, of which a and b are the sums about k.
__device__ __forceinline__ double2 moments_of(double k, double a, double b, double inverse) {
    const double off = a * inverse;
    return make_double2(k + off, not_below_zero(fma(-a, off, b)));
}

template <typename T, int VN>
__device__ __forceinline__ void stats_piece(const NormAct &p, const Columns &l, int64_t lo, int n, double2 *fold) {
    constexpr int U = VN == 8 ? 2 : 4;
    const T *x = static_cast<const T *>(p.x) + lo * p.C;
    const double inverse = 1.0 / (double)n;
    for (int pass = 0; pass < l.passes; ++pass) {
        const int lump = pass * l.cols + l.col;
        const bool mine = lump < l.lumps && l.lane < l.lanes;
        const T *col = x + (int64_t)(mine ? lump : 0) * VN;
        int r = mine ? l.lane : n;
        Rows<T, VN, U> in;
        in.load(col, r, n, l.lanes, p.C);
        Lump<T, VN> k;
        k.load(col);
        Moments<VN> sums(k);
        for (; r < n; r += U * l.lanes) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * l.lanes < n) sums.add(in.v[u]);
            in.load(col, r + U * l.lanes, n, l.lanes, p.C);
        }
        fold_lanes<VN>(l, pass, fold, [&](int i) { return make_double2(sums.a[i], sums.b[i]); }, [&](int c, double a, double b) {
            p.scratch[(int64_t)blockIdx.x * p.C + c] = moments_of(to_f32<T>(x[c]), a, b, inverse);
        });
    }
}

template <int VN>
__device__ __forceinline__ float2 drop2(const NormAct &p, const uint32_t *words, int j, float2 v) {
    v = mul2(v, both(p.drop.scale));
    return make_float2((words[j] << 16) > p.drop.over ? v.x : 0.f, words[j] > p.drop.over ? v.y : 0.f);
}

// ------------------------------------------------------------ signs ----
// In the backward pass a ReLU's argument z = (t = (x - mu) a + b) + residual has its sign from fp64 where 32 bits do not settle it: on the
// other side, an element would have a whole gradient too much or too little, and so would dbias and dweight.  (Forward it matters to no more
// than a rounding: y is some 1e-8 there, or zero.  Settling it would cost 6 us of 115 for 1.1 million rows of 64 channels.)  With u = 2^-24,
// z is off by u (2 |(x - mu) a| + |b| + |t| + |z|) at most, which for a z near zero, where |t| is next to |residual| and |(x - mu) a| at
// most |t| + |b|, is 3 u (|b| + |residual|): z is settled beyond 4 u of these.
constexpr float NEAR_BORDER = 0x1p-22f;
__device__ __forceinline__ float exact_argument(const NormAct &p, int64_t s, int c, float x, float residual) {
    const int64_t g = s * p.G + group_of(p, c);
    const double xh = ((double)x - __ldg(p.mean + g)) * __ldg(p.rstd + g);
    return (float)((p.weight ? xh * __ldg(p.weight + c) + __ldg(p.bias + c) : xh) + residual);
}
__device__ __noinline__ float exact_argument_call(const NormAct &p, int64_t s, int c, float x, float residual) { return exact_argument(p, s, c, x, residual); }
// Settles a pair of arguments where they are next to the border.  (By a call where all elements come by, in the kernel without the ring: what
// it would hold inline makes others spill, 1021 us for 979 of 34 thousand rows of 2048 channels, bf16, ReLU and residual, backward.)
template <int VN>
__device__ __forceinline__ void settle_by_call(const NormAct &p, int64_t s, int c, float2 x, float2 b, float2 residual, float2 &z) {
    if (fabsf(z.x) < NEAR_BORDER * (fabsf(b.x) + fabsf(residual.x))) z.x = exact_argument_call(p, s, channel_of(p, c), x.x, residual.x);
    if (VN > 1 && fabsf(z.y) < NEAR_BORDER * (fabsf(b.y) + fabsf(residual.y))) z.y = exact_argument_call(p, s, channel_of(p, c + 1), x.y, residual.y);
}
template <int VN>
__device__ __forceinline__ void settle(const NormAct &p, int64_t s, int c, float2 x, float2 b, float2 residual, float2 &z) {
    if (fabsf(z.x) < NEAR_BORDER * (fabsf(b.x) + fabsf(residual.x))) z.x = exact_argument(p, s, channel_of(p, c), x.x, residual.x);
    if (VN > 1 && fabsf(z.y) < NEAR_BORDER * (fabsf(b.y) + fabsf(residual.y))) z.y = exact_argument(p, s, channel_of(p, c + 1), x.y, residual.y);
}
// Whether two pairs of arguments have such a one, for the loops that all elements go through: the least beside the largest offset (`b_most`: of
// the thread's channels) and residual, and where that is near, one by one.  (Zeros of a channel without offset and residual are not near.
// A NaN in one channel: the others are looked at.)
__device__ __forceinline__ bool near_border(const float2 *z, const float2 *b, const float2 *residual, float b_most, float r_most) {
    const float least = fminf(fminf(fabsf(z[0].x), fabsf(z[0].y)), fminf(fabsf(z[1].x), fabsf(z[1].y)));
    if (least >= NEAR_BORDER * (b_most + r_most)) return false;
    bool any = false;
#pragma unroll
    for (int j = 0; j < 2; ++j) any |= fabsf(z[j].x) < NEAR_BORDER * (fabsf(b[j].x) + fabsf(residual[j].x)) || fabsf(z[j].y) < NEAR_BORDER * (fabsf(b[j].y) + fabsf(residual[j].y));
    return any;
}
__device__ __forceinline__ float largest(const float2 (&v)[4]) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, fmaxf(fabsf(v[j].x), fabsf(v[j].y)));
    return m;
}

// ------------------------------------------------------------ second pass, forward ----
template <typename T, int VN, int ACT, int DROP>
__device__ __forceinline__ bool apply_piece(const NormAct &p, const Columns &l, const Philox<DROP != 1> &rng, Constants<VN, false> &k, int64_t s, int64_t lo, int n, bool owner) {
    constexpr int U = (sizeof(T) == 4 && VN == 8 ? 2 : 4) / (DROP ? 2 : 1), P = (VN + 1) / 2, PAIRS = Constants<VN, false>::PAIRS;
    const int64_t from = lo * p.C;
    const T *x = static_cast<const T *>(p.x) + from, *res = p.residual ? static_cast<const T *>(p.residual) + from : nullptr;
    T *y = static_cast<T *>(p.y) + from;
    const int act = ACT < 0 ? p.act : ACT;
    const bool drop = DROP < 0 ? p.drop.on : DROP;
    for (int pass = 0; pass < l.passes; ++pass) {
        const int lump = pass * l.cols + l.col, c0 = lump * VN;
        const bool mine = lump < l.lumps && l.lane < l.lanes;
        int r = mine ? l.lane : n;
        Rows<T, VN, U> v, q;
        v.load(x + c0, r, n, l.lanes, p.C);   // (before the wait for the statistics)
        if (res) q.load(res + c0, r, n, l.lanes, p.C);
        if (k.s != s || k.pass != pass) {
            sync_workers();
            if (!k.load(p, l, s, pass, true)) return false;
        }
        if (owner) k.put_stats(p, l);
        for (; r < n; r += U * l.lanes) {
            uint32_t words[U][P];
            if (drop) {
#pragma unroll
                for (int u = 0; u < U; ++u) rng.words<VN>((uint64_t)(from + (r + u * l.lanes) * p.C + c0), words[u]);
            }
#pragma unroll
            for (int h = 0; h < Constants<VN, false>::QUADS; ++h) {
                float2 mu[PAIRS], a[PAIRS], b[PAIRS];
                k.read(l, K_MU, h, mu), k.read(l, K_A, h, a), k.read(l, K_B, h, b);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < PAIRS; ++i) {
                        const int j = h * PAIRS + i;
                        float2 z = fma2(add2(pair_of(v.v[u], j), mu[i]), a[i], b[i]);
                        if (res) z = add2(z, pair_of(q.v[u], j));
                        z = act2<T>(act, z);
                        if (drop) z = drop2<VN>(p, words[u], j, z);
                        set_pair(v.v[u], j, z);
                    }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * l.lanes < n) v.v[u].store(y + (r + u * l.lanes) * p.C + c0);
            v.load(x + c0, r + U * l.lanes, n, l.lanes, p.C);
            if (res) q.load(res + c0, r + U * l.lanes, n, l.lanes, p.C);
        }
    }
    return true;
}

// ------------------------------------------------------------ backward ----
// Sums of gz and gz * xh of a channel, from sums of gz and gz (x - mu).
__device__ __forceinline__ float2 sums_of(const NormAct &p, int64_t s, int c, float a, float b) {
    const double mean = __ldg(p.mean + s * p.G + group_of(p, c));
    return make_float2(a, fmaf(-(float)(mean - (float)mean), a, b) * (float)__ldg(p.rstd + s * p.G + group_of(p, c)));
}

// Rows of what both passes of the backward read, and gz of a pair of them.
template <typename T, int VN, int ACT, int DROP, int U>
struct BackwardRows {
    static constexpr int P = (VN + 1) / 2;
    Rows<T, VN, U> x, g, res;
    uint32_t words[U][P];
    // `from`: the element that the lumps' first one is
    __device__ __forceinline__ void load(const NormAct &p, const Columns &l, int64_t from, int r, int n) {
        x.load(static_cast<const T *>(p.x) + from, r, n, l.lanes, p.C);
        g.load(static_cast<const T *>(p.g) + from, r, n, l.lanes, p.C);
        if (p.residual) res.load(static_cast<const T *>(p.residual) + from, r, n, l.lanes, p.C);
    }
    __device__ __forceinline__ void draw(const NormAct &p, const Columns &l, const Philox<DROP != 1> &rng, int64_t from, int r) {
        if (DROP < 0 ? p.drop.on : DROP) {
#pragma unroll
            for (int u = 0; u < U; ++u) rng.words<VN>((uint64_t)(from + (r + u * l.lanes) * p.C), words[u]);
        }
    }
    // x - mu and gz of a lump's pairs 2 h and 2 h + 1, and whether they are next to a ReLU's border (then zeros, if such are to be left out).
    template <bool LEFT_OUT>
    __device__ __forceinline__ bool gz_told(const NormAct &p, int h, float b_most, const float2 *mu, const float2 *a, const float2 *b, float2 *xc, float2 *out) {
        constexpr int WORDS = Lump<T, VN>::WORDS / 2;
        float2 z[2], rs[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = 2 * h + i;
            rs[i] = p.residual ? pair_of(res.v[0], j) : both(0.f);
            xc[i] = add2(pair_of(x.v[0], j), mu[j]);
            z[i] = fma2(xc[i], a[j], b[j]);
            if (p.residual) z[i] = add2(z[i], rs[i]);
        }
        const bool near = near_border(z, b + 2 * h, rs, b_most, p.residual ? res.v[0].largest_of_half(h) : 0.f);
        if (LEFT_OUT) {
#pragma unroll
            for (int w = 0; w < WORDS; ++w) g.v[0].w[WORDS * h + w] = near ? 0u : g.v[0].w[WORDS * h + w];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 v = act2_backward<T>(ACT_RELU, z[i], pair_of(g.v[0], 2 * h + i));
            out[i] = DROP ? drop2<VN>(p, words[0], 2 * h + i, v) : v;
        }
        return near;
    }
    // x - mu and gz of COUNT pairs from the j0-th on, of sample s, the lump's first channel c0.
    template <int COUNT, bool SETTLED>
    __device__ __forceinline__ void gz(const NormAct &p, int64_t s, int c0, int u, int j0, const float2 *mu, const float2 *a, const float2 *b, float2 *xc, float2 *out) const {
        const int act = ACT < 0 ? p.act : ACT;
#pragma unroll
        for (int j = 0; j < COUNT; ++j) {
            const float2 xs = pair_of(x.v[u], j0 + j), rs = p.residual ? pair_of(res.v[u], j0 + j) : both(0.f);
            xc[j] = add2(xs, mu[j]);
            float2 z = fma2(xc[j], a[j], b[j]);
            if (p.residual) z = add2(z, rs);
            if (SETTLED && act == ACT_RELU)
                settle_by_call<VN>(p, s, c0 + 2 * (j0 + j), xs, b[j], rs, z);
            const float2 v = act2_backward<T>(act, z, pair_of(g.v[u], j0 + j));
            out[j] = (DROP < 0 ? p.drop.on : DROP) ? drop2<VN>(p, words[u], j0 + j, v) : v;
        }
    }
};
template <typename T, int VN>
constexpr int BACKWARD_ROWS = sizeof(T) == 4 && VN == 8 ? 1 : 2;

template <typename T, int VN, int ACT, int DROP>
__device__ __forceinline__ void bwd_sums_piece(const NormAct &p, const Columns &l, const Philox<DROP != 1> &rng, Constants<VN, true> &k, int64_t piece, int64_t s, int64_t lo, int n,
                                               float2 *fold) {
    constexpr int U = BACKWARD_ROWS<T, VN>, P = (VN + 1) / 2, PAIRS = Constants<VN, true>::PAIRS;
    for (int pass = 0; pass < l.passes; ++pass) {
        const int lump = pass * l.cols + l.col;
        const int64_t from = lo * p.C + lump * VN;
        float2 a[P], b[P];
#pragma unroll
        for (int j = 0; j < P; ++j) a[j] = b[j] = both(0.f);
        int r = lump < l.lumps && l.lane < l.lanes ? l.lane : n;
        BackwardRows<T, VN, ACT, DROP, U> in;
        in.load(p, l, from, r, n);
        if (k.s != s || k.pass != pass) {
            sync_workers();
            k.load(p, l, s, pass, false);
        }
        for (; r < n; r += U * l.lanes) {
            in.draw(p, l, rng, from, r);
#pragma unroll
            for (int h = 0; h < Constants<VN, true>::QUADS; ++h) {
                float2 mu[PAIRS], fa[PAIRS], fb[PAIRS];
                k.read(l, K_MU, h, mu), k.read(l, K_A, h, fa), k.read(l, K_B, h, fb);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r + u * l.lanes < n)
                    {
                        float2 xc[PAIRS], gz[PAIRS];
                        in.template gz<PAIRS, true>(p, s, lump * VN, u, h * PAIRS, mu, fa, fb, xc, gz);
#pragma unroll
                        for (int i = 0; i < PAIRS; ++i) a[h * PAIRS + i] = add2(a[h * PAIRS + i], gz[i]), b[h * PAIRS + i] = fma2(gz[i], xc[i], b[h * PAIRS + i]);
                    }
            }
            in.load(p, l, from, r + U * l.lanes, n);
        }
        fold_lanes<VN>(l, pass, fold, [&](int i) { return i % 2 ? make_float2(a[i / 2].y, b[i / 2].y) : make_float2(a[i / 2].x, b[i / 2].x); }, [&](int c, float sa, float sb) {
            p.rec[piece * p.C + c] = sums_of(p, s, c, sa, sb);
        });
    }
}

template <typename T, int VN, int ACT, int DROP>
__device__ __forceinline__ bool bwd_apply_piece(const NormAct &p, const Columns &l, const Philox<DROP != 1> &rng, Constants<VN, true> &k, int64_t s, int64_t lo, int n) {
    constexpr int U = BACKWARD_ROWS<T, VN>, PAIRS = Constants<VN, true>::PAIRS;
    T *dx = static_cast<T *>(p.dx), *dres = static_cast<T *>(p.dresidual);
    for (int pass = 0; pass < l.passes; ++pass) {
        const int lump = pass * l.cols + l.col;
        const int64_t from = lo * p.C + lump * VN;
        int r = lump < l.lumps && l.lane < l.lanes ? l.lane : n;
        BackwardRows<T, VN, ACT, DROP, U> in;
        in.load(p, l, from, r, n);   // (before the wait for the sums)
        if (k.s != s || k.pass != pass) {
            sync_workers();
            if (!k.load(p, l, s, pass, true)) return false;
        }
        for (; r < n; r += U * l.lanes) {
            in.draw(p, l, rng, from, r);
#pragma unroll
            for (int h = 0; h < Constants<VN, true>::QUADS; ++h) {
                float2 mu[PAIRS], fa[PAIRS], fb[PAIRS], m1[PAIRS], m2[PAIRS];
                k.read(l, K_MU, h, mu), k.read(l, K_A, h, fa), k.read(l, K_B, h, fb), k.read(l, K_M1, h, m1), k.read(l, K_M2, h, m2);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float2 xc[PAIRS], gz[PAIRS];
                    if (r + u * l.lanes < n) in.template gz<PAIRS, true>(p, s, lump * VN, u, h * PAIRS, mu, fa, fb, xc, gz);
                    else continue;
#pragma unroll
                    for (int i = 0; i < PAIRS; ++i) {
                        const int j = h * PAIRS + i;
                        set_pair(in.g.v[u], j, gz[i]);
                        set_pair(in.x.v[u], j, fma2(gz[i], fa[i], fma2(xc[i], m2[i], m1[i])));
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * l.lanes < n) {
                    const int64_t at = from + (r + u * l.lanes) * p.C;
                    if (dres) in.g.v[u].store(dres + at);
                    in.x.v[u].store(dx + at);
                }
            in.load(p, l, from, r + U * l.lanes, n);
        }
    }
    return true;
}

// ------------------------------------------------------------ merging ----
// Who merges: the block's workers, or one warp.
struct BlockTeam {
    static constexpr int SIZE = NA_THREADS;
    __device__ __forceinline__ static int rank() { return threadIdx.x; }
    __device__ __forceinline__ static void sync() { sync_workers(); }
};
struct WarpTeam {
    static constexpr int SIZE = 32;
    __device__ __forceinline__ static int rank() { return threadIdx.x & 31; }
    __device__ __forceinline__ static void sync() { __syncwarp(); }
};

// Merges the pieces of a window: a part of what merge_groups does, where records are many.
template <bool BACKWARD, typename Team>
__device__ __forceinline__ void merge_window(const NormAct &p, const Records<BACKWARD> &r, Record<BACKWARD> *to) {
    for (int g = Team::rank(); g < p.G; g += Team::SIZE) {
        RecordSums<BACKWARD> sums;
        sums.add(r, p.G, g, 0, 1);
        to[g] = sums.done(r);
    }
}

// Lanes of a warp that share a group's channels.
template <typename Team>
__device__ __forceinline__ int lanes_of_group(const NormAct &p) {
    int share = 32;
    while (share > 1 && (Team::SIZE / share < p.G || share / 2 >= p.W)) share /= 2;
    return share;
}

// The records of a piece's groups, of `n` rows, from its channels' (`channel(c)`, visible to the team).
template <bool BACKWARD, typename Team, typename Channel>
__device__ __forceinline__ void group_records(const NormAct &p, int share, int64_t piece, int n, Channel channel) {
    const int l = Team::rank() % share;
    const auto sum = [&](auto v) {
        for (int o = share / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    Record<BACKWARD> *to = static_cast<Record<BACKWARD> *>(p.of_piece) + piece * p.G;
    const double inverse = 1.0 / p.W;
    for (int g0 = 0; g0 < p.G; g0 += Team::SIZE / share) {   // (the same rounds for all lanes of a warp)
        const int g = g0 + Team::rank() / share, c0 = min(g, p.G - 1) * p.W, end = g < p.G ? p.W : 0;
        if constexpr (BACKWARD) {
            float a = 0.f, b = 0.f;
#pragma unroll 4
            for (int i = l; i < end; i += share) {
                const float2 v = channel(c0 + i);
                const float w = p.weight ? __ldg(p.weight + c0 + i) : 1.f;
                a += w * v.x, b += w * v.y;
            }
            a = sum(a), b = sum(b);
            if (g < p.G && l == 0) to[g] = {a, b};
        } else {   // the mean about the first channel's, then squares about it
            const double k = channel(c0).x;
            double a = 0.0, b = 0.0;
#pragma unroll 4
            for (int i = l; i < end; i += share) a += channel(c0 + i).x - k;
            const double mean = k + sum(a) * inverse;
#pragma unroll 4
            for (int i = l; i < end; i += share) {
                const double2 v = channel(c0 + i);
                const double d = v.x - mean;
                b += fma((double)n * d, d, v.y);
            }
            b = sum(b);
            if (g < p.G && l == 0) to[g] = {mean, b};
        }
    }
}

// Counts what the team has written; true in all of its threads where that was the last of `of`, and then the others' is there to be read.
template <typename Team>
__device__ __forceinline__ bool brings_the_last(int *count, int of, int *told) {
    Team::sync();
    if (Team::rank() == 0) {
        __threadfence();
        *told = atomicAdd(count, 1);
    }
    Team::sync();
    const bool last = *told == of - 1;
    Team::sync();   // (before it is told again)
    if (last) __threadfence();
    return last;
}

// After the team has written the records of piece (chunk, s).
template <bool BACKWARD, typename Team>
__device__ __forceinline__ void count_piece(const NormAct &p, const Span &v, int chunk, int64_t s, int *told) {
    if (p.window > 1) {
        const int w = (chunk - v.b0) / p.window, b = v.b0 + w * p.window, pieces = min(p.window, v.b1 - b + 1);
        const int64_t number = first_window(p, v, s) + w, from = (int64_t)b * p.rows;
        if (!brings_the_last<Team>(window_count(p) + number, pieces, told)) return;
        const int64_t lo = max(p.offsets[s], from), hi = min(p.offsets[s + 1], from + (int64_t)pieces * p.rows);
        merge_window<BACKWARD, Team>(p, records_of<BACKWARD>(p.of_piece, (b + s) * p.G, pieces, lo, hi, from, p.rows, p.W),
                                     static_cast<Record<BACKWARD> *>(p.of_window) + number * p.G);
    }
    Team::sync();
    if (Team::rank() == 0) {
        __threadfence();
        atomicAdd(sample_count(p) + s, 1);
        if (BACKWARD && p.dweight) atomicAdd(p.control + WINDOWS_DONE, 1);
    }
}

// dweight and dbias of some channels: the pieces' sums in a fixed order, in fp64.  (There may be tens of thousands of them.)
__device__ __noinline__ void affine_gradients(const NormAct &p, int tile, double2 *scratch) {
    constexpr int DEEP = NA_THREADS / AFFINE_CHANNELS;
    const int lane = threadIdx.x % AFFINE_CHANNELS, q = threadIdx.x / AFFINE_CHANNELS, c = tile * AFFINE_CHANNELS + lane;
    const int64_t pieces = p.N / p.rows + p.S;   // (numbers that no piece has hold zeros)
    double a = 0.0, b = 0.0;
    if (c < p.C)
#pragma unroll 8
        for (int64_t i = q; i < pieces; i += DEEP) {
            const float2 v = __ldcg(p.rec + i * p.C + c);
            a += v.x, b += v.y;
        }
    sync_workers();
    scratch[threadIdx.x] = make_double2(a, b);
    sync_workers();
    if (q == 0 && c < p.C) {
        double da = 0.0, db = 0.0;
        for (int i = 0; i < DEEP; ++i) da += scratch[i * AFFINE_CHANNELS + lane].x, db += scratch[i * AFFINE_CHANNELS + lane].y;
        p.dbias[c] = (float)da, p.dweight[c] = (float)db;
    }
}

// ------------------------------------------------------------ the kernel ----
// Pairs of 32 bits that folding takes (at least what affine_gradients does).
template <int VN, bool BACKWARD>
__host__ __device__ constexpr int fold_entries() { return (BACKWARD ? (VN < 2 ? 2 : VN) : 2 * VN) * NA_THREADS; }
template <int VN, bool BACKWARD>
size_t shared_bytes(int C) {
    const Columns l(C, VN, 0);
    return (size_t)fold_entries<VN, BACKWARD>() * sizeof(float2) + (size_t)(BACKWARD ? 8 : 3) * l.cols * VN * sizeof(float) +
           NA_THREADS * sizeof(double2) + (size_t)(l.cols * VN + 1) * sizeof(Stats);
}

// ACT, DROP = -1: as the arguments say; DROP = 0: none, 1: the seed is in the arguments, 2: on the device.
template <typename T, int VN, int ACT, int DROP, bool BACKWARD>
__global__ void __launch_bounds__(NA_THREADS, NA_BLOCKS) na_kernel(const __grid_constant__ NormAct p) {
    start_after_previous();
    extern __shared__ __align__(128) char shared[];
    __shared__ int next, told;
    float2 *fold = reinterpret_cast<float2 *>(shared);   // sums of threads, or records that are merged
    const Columns l(p.C, VN, threadIdx.x);
    Constants<VN, BACKWARD> k_sums, k_apply;
    k_apply.at = reinterpret_cast<float *>(fold + fold_entries<VN, BACKWARD>());
    k_sums.at = k_apply.at + 5 * l.cols * VN;
    k_apply.scratch = reinterpret_cast<double2 *>(k_apply.at + ((BACKWARD ? 8 : 3) * l.cols * VN + 3) / 4 * 4);
    k_apply.stats = reinterpret_cast<Stats *>(k_apply.scratch + NA_THREADS);
    const Philox<DROP != 1> rng(p.drop);
    const int tiles = BACKWARD && p.dweight ? (p.C + AFFINE_CHANNELS - 1) / AFFINE_CHANNELS : 0;
    for (;;) {
        __syncthreads();
        if (threadIdx.x == 0) next = atomicAdd(p.control + TICKET, 1);
        __syncthreads();
        const int ticket = next;
        if (ticket >= 2 * p.chunks + tiles) return;
        if (BACKWARD && ticket >= 2 * p.chunks) {
            if (!wait_for(p.control + WINDOWS_DONE, p.control[WINDOWS], p.status)) return;
            affine_gradients(p, ticket - 2 * p.chunks, reinterpret_cast<double2 *>(fold));
            continue;
        }
        int chunk;
        const bool sums = take_ticket(p, ticket, &chunk);
        const int64_t row0 = (int64_t)chunk * p.rows, row1 = min(p.N, row0 + p.rows);
        for (int64_t s = last_not_over(p.S, row0, [&](int64_t q) { return p.offsets[q]; }); s < p.S && p.offsets[s] < row1; ++s) {
            const int64_t lo = max(row0, p.offsets[s]), hi = min(row1, p.offsets[s + 1]);
            if (hi <= lo) continue;   // a sample without rows
            if (sums) {
                if constexpr (BACKWARD) bwd_sums_piece<T, VN, ACT, DROP>(p, l, rng, k_sums, chunk + s, s, lo, (int)(hi - lo), fold);
                else stats_piece<T, VN>(p, l, lo, (int)(hi - lo), reinterpret_cast<double2 *>(fold));
                sync_workers();
                group_records<BACKWARD, BlockTeam>(p, lanes_of_group<BlockTeam>(p), chunk + s, (int)(hi - lo), [&](int c) {   // (what this block has written)
                    if constexpr (BACKWARD) return __ldcg(p.rec + (chunk + s) * p.C + c);
                    else return __ldcg(p.scratch + (int64_t)blockIdx.x * p.C + c);
                });
                count_piece<BACKWARD, BlockTeam>(p, p.spans[s], chunk, s, &told);
            } else {
                bool there;
                if constexpr (BACKWARD) there = bwd_apply_piece<T, VN, ACT, DROP>(p, l, rng, k_apply, s, lo, (int)(hi - lo));
                else there = apply_piece<T, VN, ACT, DROP>(p, l, rng, k_apply, s, lo, (int)(hi - lo), chunk == p.spans[s].b0);
                if (!there) return;
            }
        }
    }
}

// ------------------------------------------------------------ the ring ----
// The same tickets at 16-byte addresses, up to 1024 channels.  Where a row is no whole number of lumps of eight channels, 2, 4 or 8 rows
// side by side are (50 channels: four rows, 200), and such rows are what "row" means here: they are counted from the tensor's first,
// so a sample may begin and end inside one.  What is outside of it (or behind the tensor) is left out of sums, and not written.
// A warp, the producer, takes the tickets and brings their rows, which lie side by side, by bulk copies into a ring of tiles in shared
// memory; eight warps work on them; the sums of a piece go to another warp, the clerk, which folds them, writes the record, counts it and
// merges.  So whatever a ticket waits for (its number, the samples' offsets, the first bytes) passes while tiles before it are worked
// on, and rows are not kept waiting by records: with both done by the workers, between tickets, a ticket of 64 KB took 4.7 us and 2 more
// to be counted.
//
// Bound by bytes where the tail is short, every input read once a pass: 1.1 million points of 64 channels, bf16, eight samples, ReLU and
// residual: forward 563 MB in 113 us, 5.0 TB/s; backward 1126 MB in 224 us, 5.0 TB/s, where 6.5 TB/s are a copy's.  By instructions with
// SiLU and dropout of 0.1: 422 MB in 134 us, 704 MB in 221 us (without dropout 105 and 166).  Forward, sums of 64 bits take the conversion
// of each element, of which the chip does 16 a clock and SM: hidden behind 141 MB a tensor but for 5 us, and 2 of 40 us
// where 38 MB are.  Where all rows are some megabytes the launch is latency: one sample of 942 points and 256 channels 12 to 15 us, of which
// a first read, the records' turn through the L2 and the code's own way into the instruction cache are most.  (Lags of few chunks, so
// that the second pass finds its rows in the L2, do not pay: what is in flight until a sample's records are there is as much as the L2
// keeps beside what is written.)
enum { TILE_SUMS = 0, TILE_APPLY = 1, TILE_AFFINE = 2, TILE_END = 3, TILE_NONE = 4 };
constexpr int RING_CHANNELS = 1024;                // of a row, at most (their constants take room from the ring)
constexpr int RING_STAGES = 8;                     // at most
constexpr int FOLD_SLOTS = 2;                      // pieces on their way to the clerk, at most
constexpr int RING_THREADS = NA_THREADS + 64;
constexpr int RING_BLOCKS = 2;                     // on a multiprocessor
struct __align__(16) Tile {
    int kind, s, chunk, n;       // n rows
    int64_t from;                // the first element
    int last;                    // sums: the rows (of C channels) of the piece that this is the last tile of, or 0; apply: whether it is the first of a sample
    int end;                     // with phases: behind the sample's last element
    int first, whole;            // and a lump is the sample's, whole, if its place less `first` is below `whole`
};
struct Piece { int kind, s, chunk, rows; };
// A warp of workers that has lumps with a ReLU's argument next to its border in a tile asks the clerk to settle them, and waits: (the tile's
// place and its round's parity) * 4 + one of these.
enum { ASK_NOTHING = 0, ASK_SUMS = 1, ASK_APPLY = 2, ASK_ANSWERED = 3 };
// What passes between them, in the room of merge_groups (no block merges while one of its warps is at a tile).
struct Asked {
    uint32_t rounds[NA_THREADS];   // bit 2 i + h: half h of the lump of the thread's i-th row in the tile (there are 12 at most)
    float2 sums[8][32];            // the answer: what those lumps add to a channel's sums
};
static_assert(sizeof(Asked) <= NA_THREADS * sizeof(double2), "room");

struct Ring {
    uint64_t full[RING_STAGES], empty[RING_STAGES], folded[FOLD_SLOTS], taken[FOLD_SLOTS];
    Tile tiles[RING_STAGES];
    Piece pieces[FOLD_SLOTS];
    int told, abort;
    volatile int asked[NA_THREADS / 32];   // of the clerk, by the workers' warps (enum above)
};
// Whether whole rows of columns make a warp (64 channels: 8 columns, 4 rows): its lanes are then folded before the clerk has them.
__host__ __device__ __forceinline__ bool warps_fold(const Columns &l) { return l.cols < 32 && 32 % l.cols == 0; }
// Where sums of pieces wait for the clerk: 33 KB.  Backward pairs of 32 bits in two slots, forward of 64 in two where warps fold their own
// (128 of them or fewer for each channel of the lumps), and in one otherwise.
template <bool BACKWARD>
struct Folds {
    using Two = std::conditional_t<BACKWARD, float2, double2>;
    static constexpr int BYTES = 2 * 8 * (NA_THREADS + 2) * (int)sizeof(float2);
    int rows, stride, slots;   // rows of columns; from a channel of the lumps to the next, so that the clerk finds no bank conflicts
    __host__ __device__ __forceinline__ explicit Folds(const Columns &l) {
        rows = warps_fold(l) ? NA_THREADS / 32 : l.lanes;
        stride = BACKWARD ? NA_THREADS + 2 : rows * l.cols | 1;
        slots = BACKWARD || stride <= NA_THREADS / 2 + 1 ? FOLD_SLOTS : 1;
    }
};
// (behind the ring's tiles) slots of sums, what is taken off the channels' values for each, constants
struct RingMemory {
    char *stages;
    char *fold;
    float *firsts, *constants;
    Stats *stats;
    double2 *scratch;
    __device__ __forceinline__ RingMemory(const NormAct &p, char *shared) {
        stages = shared;
        fold = shared + (size_t)p.stages * p.stage_bytes;
        scratch = reinterpret_cast<double2 *>(fold + Folds<true>::BYTES);
        stats = reinterpret_cast<Stats *>(scratch + NA_THREADS);
        constants = reinterpret_cast<float *>(stats + p.G);
        firsts = constants + 3 * p.V;   // (forward alone)
    }
};
inline size_t ring_bytes(int V, int G, bool backward) {   // without the tiles
    return (size_t)Folds<true>::BYTES + NA_THREADS * sizeof(double2) + (size_t)G * sizeof(Stats) +
           (size_t)(backward ? 8 : 3 + Folds<false>(Columns(V, 8, 0)).slots + 1) * V * sizeof(float);
}

__device__ __forceinline__ void bulk_copy(uint32_t to, const void *from, uint32_t bytes, uint32_t bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(to), "l"(from), "r"(bytes), "r"(bar), "l"(policy)
                 : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A place in a ring of `size`, and the parity of its round.
struct Place {
    int at = -1, parity = 0;
    __device__ __forceinline__ void next(int size) {
        if (++at == size) at = 0, parity ^= 1;
    }
};

template <typename T, bool BACKWARD, bool PHASES>
__device__ __forceinline__ void ring_producer(const NormAct &p, Ring &ring, const RingMemory &m) {
    const int lane = threadIdx.x & 31, tiles = BACKWARD && p.dweight ? (p.C + AFFINE_CHANNELS - 1) / AFFINE_CHANNELS : 0;
    const uint32_t step = (uint32_t)p.tile_rows * p.V * sizeof(T), stages = tc::smem_u32(m.stages);
    uint64_t keep, drop;
    asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(keep));
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(drop));
    Place place;
    int brought = 0;
    const auto push = [&](const Tile &t) -> bool {
        place.next(p.stages);
        if (brought >= p.stages &&
            !__all_sync(0xffffffffu, tc::mbar_wait_abortable(tc::smem_u32(&ring.empty[place.at]), place.parity ^ 1, NA_STATUS, p.status, &ring.abort))) {
            return false;
        }
        const bool stats = !BACKWARD && t.kind == TILE_SUMS;   // (of x alone)
        const uint32_t to = stages + (uint32_t)place.at * p.stage_bytes;
        uint32_t each = (uint32_t)t.n * p.V * sizeof(T);
        if (PHASES && t.kind <= TILE_APPLY) {
            const int64_t there = (p.N * p.C - t.from) * (int64_t)sizeof(T);
            if (there < each) {   // the tensor's last row: what is no multiple of 16 bytes, one by one
                each = (uint32_t)there & ~15u;
                const int64_t at = t.from + each / sizeof(T) + lane;
                if (lane < ((int)there & 15) / (int)sizeof(T)) {
                    T *into = reinterpret_cast<T *>(m.stages + (size_t)place.at * p.stage_bytes + each) + lane;
                    *into = static_cast<const T *>(p.x)[at], into += step / sizeof(T);
                    if (BACKWARD) *into = static_cast<const T *>(p.g)[at], into += step / sizeof(T);
                    if (p.residual && !stats) *into = static_cast<const T *>(p.residual)[at];
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // (bulk copies will write there)
                __syncwarp();
            }
        }
        if (lane == 0) {
            ring.tiles[place.at] = t;
            const uint32_t bar = tc::smem_u32(&ring.full[place.at]);
            if (t.kind <= TILE_APPLY && each) {
                const uint64_t policy = t.kind == TILE_SUMS ? keep : drop;
                uint32_t into = to;
                expect_bytes(bar, each * ((BACKWARD ? 2 : 1) + (p.residual && !stats)));
                bulk_copy(into, static_cast<const T *>(p.x) + t.from, each, bar, policy), into += step;
                if (BACKWARD) bulk_copy(into, static_cast<const T *>(p.g) + t.from, each, bar, policy), into += step;
                if (p.residual && !stats) bulk_copy(into, static_cast<const T *>(p.residual) + t.from, each, bar, policy);
            } else {
                tc::mbar_arrive(bar);
            }
        }
        ++brought;
        return true;
    };
    const auto all = [&]() -> bool {
        int ticket = 0, upcoming = 0;
        if (lane == 0) ticket = atomicAdd(p.control + TICKET, 1);
        ticket = __shfl_sync(0xffffffffu, ticket, 0);
        for (;; ticket = __shfl_sync(0xffffffffu, upcoming, 0)) {
            if (ticket >= 2 * p.chunks + tiles) return push(Tile{TILE_END});
            if (lane == 0) upcoming = atomicAdd(p.control + TICKET, 1);
            if (ticket >= 2 * p.chunks) {
                if (!push(Tile{TILE_AFFINE, 0, ticket - 2 * p.chunks})) return false;
                continue;
            }
            int chunk;
            const bool sums = take_ticket(p, ticket, &chunk);
            const int tile_rows = sums ? p.sums_tile_rows : p.tile_rows;
            const int64_t row0 = (int64_t)chunk * p.rows, row1 = min(p.N, row0 + p.rows);
            for (int64_t s = last_not_over(p.S, row0, [&](int64_t q) { return p.offsets[q]; }); s < p.S; ++s) {
                const int64_t at = p.offsets[s], lo = max(row0, at), hi = min(row1, p.offsets[s + 1]);
                if (at >= row1) break;
                const bool owner = !BACKWARD && !sums && chunk == p.spans[s].b0;   // (of the statistics)
                if (hi <= lo) continue;
                const int64_t v0 = PHASES ? lo >> p.phase_bits : lo, v1 = PHASES ? (hi + (1 << p.phase_bits) - 1) >> p.phase_bits : hi;
                for (int64_t r = v0; r < v1; r += tile_rows) {
                    const int n = (int)min((int64_t)tile_rows, v1 - r);
                    Tile t{sums ? TILE_SUMS : TILE_APPLY, (int)s, chunk, n, r * p.V, sums ? (r + n == v1 ? (int)(hi - lo) : 0) : owner && r == v0};
                    if (PHASES) {
                        t.first = (int)max(lo * p.C - t.from, (int64_t)0), t.end = (int)min((int64_t)n * p.V, hi * p.C - t.from);
                        t.whole = max(t.end - t.first - 7, 0);
                    }
                    if (!push(t)) return false;
                }
            }
        }
    };
    if (!all()) {   // shared memory is not given back under copies in flight
        const int behind = min(brought, p.stages);
        Place q;
        for (int j = 0; j < brought; ++j) {
            q.next(p.stages);
            if (j >= brought - behind) tc::mbar_wait(tc::smem_u32(&ring.full[q.at]), q.parity, NA_STATUS, p.status);
        }
    }
}

// Of a pair at `at`, what is within first <= at < end.
__device__ __forceinline__ float2 within(float2 v, int at, int first, int end) {
    return make_float2(at >= first && at < end ? v.x : 0.f, at + 1 >= first && at + 1 < end ? v.y : 0.f);
}

// The clerk's answer to warp `w`: lane for lane what its threads would do, with the arguments' signs settled.  Halves of lumps were left out
// of the sums; of the results lumps are written once more.  Few elements come here (with a residual some ten of 70 million), but many may:
// values of 16 bits come again, and a channel's border may lie at one of them (one channel of 64, 600 thousand rows a sample: 196 us for 170; all
// channels, a seventh of their rows: 2.8 ms).  (The workers do not do it themselves: whatever they would hold for it costs all other
// elements registers.  1.1 million points of 64 channels, bf16, residual, backward: 222 us, 256 where they do, 280 by a call.)
template <typename T, int DROP, bool PHASES>
__device__ __forceinline__ void settle_tile(const NormAct &p, Ring &ring, const RingMemory &m, int w) {
    constexpr int VN = 8;
    const int lane = threadIdx.x & 31, request = ring.asked[w], kind = request & 3, parity = request >> 2 & 1, place = request >> 3;
    Asked &asked = *reinterpret_cast<Asked *>(m.scratch);
    __threadfence_block();
    tc::mbar_wait(tc::smem_u32(&ring.full[place]), parity, NA_STATUS, p.status);   // (is there: the tile's bytes are this warp's to read, too)
    __syncwarp();
    const Tile &t = ring.tiles[place];
    const Columns l(p.V, VN, 32 * w + lane);
    const Philox<DROP != 1> rng(p.drop);
    const int c0 = l.col * VN, tensor = p.tile_rows * p.V, s = t.s;
    const T *x = reinterpret_cast<const T *>(m.stages + (size_t)place * p.stage_bytes) + c0;
    Constants<VN, true> k;
    k.at = m.constants + (kind == ASK_SUMS ? 5 * p.V : 0);
    float2 a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = b[j] = both(0.f);
    uint32_t rounds = asked.rounds[32 * w + lane];
    for (int at = l.lane * p.V; rounds; rounds >>= 2, at += l.lanes * p.V) {
        if (!(rounds & 3)) continue;
        const int64_t to = t.from + at + c0;
        const int first = PHASES ? t.first - at - c0 : 0, end = PHASES ? t.end - at - c0 : VN;
        BackwardRows<T, VN, ACT_RELU, DROP, 1> in;
        in.x.v[0].load(x + at);
        in.g.v[0].load(x + tensor + at);
        if (p.residual) in.res.v[0].load(x + 2 * tensor + at);
        if (DROP) rng.template words<VN>((uint64_t)to, in.words[0]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (kind == ASK_SUMS && !(rounds >> h & 1)) continue;
            float2 mu[2], fa[2], fb[2], m1[2], m2[2];
            k.read(l, K_MU, h, mu), k.read(l, K_A, h, fa), k.read(l, K_B, h, fb);
            if (kind == ASK_APPLY) k.read(l, K_M1, h, m1), k.read(l, K_M2, h, m2);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = 2 * h + i;
                const float2 xs = pair_of(in.x.v[0], j), rs = p.residual ? pair_of(in.res.v[0], j) : both(0.f), xc = add2(xs, mu[i]);
                float2 z = fma2(xc, fa[i], fb[i]);
                if (p.residual) z = add2(z, rs);
                settle<VN>(p, s, c0 + 2 * j, xs, fb[i], rs, z);
                z = act2_backward<T>(ACT_RELU, z, pair_of(in.g.v[0], j));
                if (DROP) z = drop2<VN>(p, in.words[0], j, z);
                if (kind == ASK_APPLY) {
                    set_pair(in.g.v[0], j, z), set_pair(in.x.v[0], j, fma2(z, fa[i], fma2(xc, m2[i], m1[i])));
                } else {
                    z = within(z, 2 * j, first, end);
                    a[j] = add2(a[j], z), b[j] = fma2(z, within(xc, 2 * j, first, end), b[j]);
                }
            }
        }
        if (kind == ASK_APPLY) {
            if (p.dresidual) in.g.v[0].store_part(static_cast<T *>(p.dresidual) + to, first, end);
            in.x.v[0].store_part(static_cast<T *>(p.dx) + to, first, end);
        }
    }
    if (kind == ASK_SUMS) {
#pragma unroll
        for (int j = 0; j < 4; ++j) asked.sums[2 * j][lane] = a[j], asked.sums[2 * j + 1][lane] = b[j];
    }
    __threadfence_block();
    __syncwarp();
    if (lane == 0) ring.asked[w] = kind == ASK_SUMS ? ASK_ANSWERED : ASK_NOTHING;
    if (kind == ASK_SUMS) {   // the next answer takes the place of this one: until it has been read
        const uint64_t t0 = tc::global_timer_ns();
        while (ring.asked[w] == ASK_ANSWERED && !*const_cast<volatile int *>(&ring.abort) && tc::global_timer_ns() - t0 <= tc::WAIT_LIMIT_NS) __nanosleep(20);
    }
    __syncwarp();
}

// Until a piece's sums are there; meanwhile warps that ask are answered.  False: a wait has run out.
template <typename T, int DROP, bool PHASES>
__device__ __forceinline__ bool answer_until_folded(const NormAct &p, Ring &ring, const RingMemory &m, const Place &slot) {
    const int lane = threadIdx.x & 31;
    uint64_t t0 = tc::global_timer_ns();
    for (int turn = 0;; ++turn) {
        if (__all_sync(0xffffffffu, tc::mbar_try_wait_parked(tc::smem_u32(&ring.folded[slot.at]), slot.parity, 500u))) return true;
        const int asked = lane < NA_THREADS / 32 ? ring.asked[lane] & 3 : ASK_NOTHING;
        unsigned warps = __ballot_sync(0xffffffffu, asked == ASK_SUMS || asked == ASK_APPLY);
        if (warps) {
            for (; warps; warps &= warps - 1) settle_tile<T, DROP, PHASES>(p, ring, m, __ffs(warps) - 1);
            t0 = tc::global_timer_ns();
        }
        if (turn % 64 != 63) continue;   // (each look at the clock is slow: at every turn, 179 us for 153 of 273 thousand rows of 256 channels, bf16)
        const bool late = tc::global_timer_ns() - t0 > tc::WAIT_LIMIT_NS, over = *const_cast<volatile int *>(&ring.abort);
        if (__any_sync(0xffffffffu, late || over)) {
            if (lane == 0 && !over) ring.abort = 1, atomicOr(p.status, NA_STATUS);
            return false;
        }
    }
}

// Folds the sums of pieces over the row lanes and takes them from there.
template <typename T, int ACT, int DROP, bool BACKWARD, bool PHASES>
__device__ __forceinline__ void ring_clerk(const NormAct &p, Ring &ring, const RingMemory &m) {
    const int lane = threadIdx.x & 31;
    const Columns l(p.V, 8, 0);
    const Folds<BACKWARD> folds(l);
    using Two = typename Folds<BACKWARD>::Two;
    const bool few = !PHASES && folds.rows <= 8;   // one chain (with eight, a call of 942 points and 256 channels takes a microsecond more)
    int parts = 1;                                 // lanes of a channel
    while (!few && 2 * parts * p.C <= 32) parts *= 2;
    const int share = lanes_of_group<WarpTeam>(p);
    Place slot;
    for (int pieces = 0;; ++pieces) {
        slot.next(folds.slots);
        if constexpr (BACKWARD && ACT == ACT_RELU) {
            if (!answer_until_folded<T, DROP, PHASES>(p, ring, m, slot)) return;
        } else {
            if (!__all_sync(0xffffffffu, tc::mbar_wait_abortable(tc::smem_u32(&ring.folded[slot.at]), slot.parity, NA_STATUS, p.status, &ring.abort))) return;
        }
        const Piece piece = ring.pieces[slot.at];
        if (piece.kind == TILE_END) return;
        Two *fold = reinterpret_cast<Two *>(m.fold) + slot.at * 8 * folds.stride;
        const float *firsts = m.firsts + pieces % (folds.slots + 1) * p.V;
        const int64_t number = piece.chunk + (int64_t)piece.s;
        const double inverse = 1.0 / piece.rows;
        for (int base = 0; base < p.C; base += 32 / parts) {   // (the same rounds for all lanes)
            const int c = base + lane / parts;
            Two sums{};
            if (few) {
                if (c >= p.C) continue;
                const Two *from = fold + c % 8 * folds.stride + c / 8;
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (q < folds.rows) sums.x += from[q * l.cols].x, sums.y += from[q * l.cols].y;
            } else {
                Chains<Two> chains;
                if (c < p.C)
                    for (int at = c; at < (PHASES ? p.V : c + 1); at += p.C) chains.add(fold + at % 8 * folds.stride + at / 8, lane % parts, parts, folds.rows, l.cols);
                sums = chains.sum();
            }
            for (int o = parts / 2; o > 0; o >>= 1) sums.x += __shfl_xor_sync(0xffffffffu, sums.x, o), sums.y += __shfl_xor_sync(0xffffffffu, sums.y, o);
            if (c >= p.C || lane % parts) continue;
            if constexpr (BACKWARD) {
                sums = sums_of(p, piece.s, c, sums.x, sums.y);
                if (p.dweight) p.rec[number * p.C + c] = sums;
            } else {
                sums = moments_of(firsts[c], sums.x, sums.y, inverse);
            }
            fold[c % 8 * folds.stride + c / 8] = sums;
        }
        __syncwarp();
        group_records<BACKWARD, WarpTeam>(p, share, number, piece.rows, [&](int c) { return fold[c % 8 * folds.stride + c / 8]; });
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(tc::smem_u32(&ring.taken[slot.at]));
        count_piece<BACKWARD, WarpTeam>(p, p.spans[piece.s], piece.chunk, piece.s, &ring.told);
    }
}

// The workers' warps wait for tiles each by itself, and meet where the sample changes.  One whose wait has run out comes to the next
// meeting with that, whichever it is, and then all of them leave: a meeting is the first barrier that a warp comes to after any tile.
template <typename T, int ACT, int DROP, bool BACKWARD, bool PHASES>
__device__ __forceinline__ void ring_worker(const NormAct &p, Ring &ring, const RingMemory &m) {
    constexpr int VN = 8, P = 4;
    const Columns l(p.V, VN, threadIdx.x);
    const Folds<BACKWARD> folds(l);
    using Two = typename Folds<BACKWARD>::Two;
    const Philox<DROP != 1> rng(p.drop);
    const bool mine = l.lane < l.lanes;
    const int c0 = l.col * VN, step = l.lanes * p.V;   // elements from one of a thread's rows to its next
    const int tensor = p.tile_rows * p.V;              // elements from one tensor's tile to the next one's
    Constants<8, BACKWARD> k_sums, k_apply;
    k_apply.at = m.constants, k_sums.at = m.constants + 5 * p.V;
    k_apply.stats = m.stats, k_apply.scratch = m.scratch;
    Place place, slot;
    int pieces = 0;
    Tile t;
    const auto next_tile = [&] {
        place.next(p.stages);
        if (__all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&ring.full[place.at]), place.parity, NA_STATUS, p.status))) t = ring.tiles[place.at];
        else t.kind = TILE_NONE;
    };
    // Whether a lump is no sample's whole.  (Read where it is asked for: in registers the bounds made others spill.)
    const auto cut = [&](int at) -> bool {
        int first, whole;
        asm volatile("ld.shared.v2.s32 {%0, %1}, [%2];" : "=r"(first), "=r"(whole) : "r"(tc::smem_u32(&ring.tiles[place.at].first)) : "memory");
        return (uint32_t)(at - first) >= (uint32_t)whole;
    };
    const auto ends = [&] {
        const Tile &q = ring.tiles[place.at];
        return make_int2(q.first, q.end);
    };
    const auto release = [&] {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) tc::mbar_arrive(tc::smem_u32(&ring.empty[place.at]));
    };
    const auto rows_at = [&] { return reinterpret_cast<const T *>(m.stages + (size_t)place.at * p.stage_bytes) + c0; };
    // A slot for sums, when they are ready; false: the clerk has not come for the ones before.
    const auto next_slot = [&]() -> bool {
        slot.next(folds.slots);
        return ++pieces <= folds.slots || __all_sync(0xffffffffu, tc::mbar_wait(tc::smem_u32(&ring.taken[slot.at]), slot.parity ^ 1, NA_STATUS, p.status));
    };
    const auto send = [&](const Piece &piece) {
        if (threadIdx.x == 0) ring.pieces[slot.at] = piece;
        __syncwarp();
        if ((threadIdx.x & 31) == 0) tc::mbar_arrive(tc::smem_u32(&ring.folded[slot.at]));
    };
    // Has the clerk settle the tile's lumps of these rounds; false: it did not come.
    const auto ask = [&](int kind, uint32_t rounds) -> bool {
        const int w = threadIdx.x >> 5;
        reinterpret_cast<Asked *>(m.scratch)->rounds[threadIdx.x] = rounds;
        __threadfence_block();   // (what has been written of the results is overwritten)
        __syncwarp();
        if ((threadIdx.x & 31) == 0) ring.asked[w] = (place.at * 2 + place.parity) * 4 + kind;
        __syncwarp();
        const int answered = kind == ASK_SUMS ? ASK_ANSWERED : ASK_NOTHING;
        const uint64_t t0 = tc::global_timer_ns();
        bool there = false;
        while (!(there = ring.asked[w] == answered) && tc::global_timer_ns() - t0 <= tc::WAIT_LIMIT_NS) __nanosleep(50);
        there = __all_sync(0xffffffffu, there);
        if (!there && (threadIdx.x & 31) == 0) atomicOr(p.status, NA_STATUS);
        __threadfence_block();
        return there;
    };
    // A piece's sums, `part(i)` those of the lump's channels, into its slot: over the warp's row lanes first, where that is whole.
    const auto fold_and_send = [&](const Piece &piece, auto part) {
        Two sums[VN];
#pragma unroll
        for (int i = 0; i < VN; ++i) {
            sums[i] = part(i);
            if (warps_fold(l))
                for (int o = 16; o >= l.cols; o >>= 1) sums[i].x += __shfl_xor_sync(0xffffffffu, sums[i].x, o), sums[i].y += __shfl_xor_sync(0xffffffffu, sums[i].y, o);
        }
        if (warps_fold(l) ? (threadIdx.x & 31) < l.cols : mine) {
            Two *fold = reinterpret_cast<Two *>(m.fold) + slot.at * 8 * folds.stride + (warps_fold(l) ? (threadIdx.x >> 5) * l.cols + (threadIdx.x & 31) : threadIdx.x);
#pragma unroll
            for (int i = 0; i < VN; ++i) fold[i * folds.stride] = sums[i];
        }
        send(piece);
    };
    next_tile();
    for (;;) {
        if (t.kind == TILE_SUMS && !BACKWARD) {
            const int s = t.s, chunk = t.chunk;
            Lump<T, VN> k;
            if constexpr (PHASES) {
                const T *first = rows_at() - c0 + ends().x;
                int c = channel_of(p, c0);
#pragma unroll
                for (int i = 0; i < VN; ++i) {
                    k.set(i, to_f32<T>(first[c]));
                    if (++c == p.C) c = 0;
                }
            } else {
                k.load(rows_at());
            }
            if (l.lane == 0) {   // (C of V are read.  One more in turn than there are slots: the clerk may still be at all of those)
#pragma unroll
                for (int i = 0; i < VN; ++i) m.firsts[pieces % (folds.slots + 1) * p.V + c0 + i] = k.get(i);
            }
            Moments<VN> sums(k);
            int rows = 0;
            for (bool more = true; more;) {
                const T *x = rows_at();
                if (mine)
#pragma unroll 2
                    for (int r = l.lane, at = l.lane * p.V; r < t.n; r += l.lanes, at += step) {
                        Lump<T, VN> v;
                        v.load(x + at);
                        if (PHASES && cut(at + c0)) {
                            const int2 e = ends();
                            sums.add(v, e.x - at - c0, e.y - at - c0);
                        } else {
                            sums.add(v);
                        }
                    }
                rows = t.last;
                more = !rows;
                release();
                next_tile();
                if (t.kind == TILE_NONE) more = false;
            }
            if (!next_slot()) t.kind = TILE_NONE;
            if constexpr (!BACKWARD)
                if (t.kind != TILE_NONE) fold_and_send(Piece{TILE_SUMS, s, chunk, rows}, [&](int i) { return make_double2(sums.a[i], sums.b[i]); });
        } else if (t.kind == TILE_SUMS) {
            float2 a[P], b[P], mu[P], fa[P], fb[P];
            const int s = t.s, chunk = t.chunk;
            if (k_sums.s != s) {
                if (!sync_workers_and(true)) break;
                k_sums.template load<PHASES>(p, l, s, 0, false);
            }
#pragma unroll
            for (int j = 0; j < P; ++j) a[j] = b[j] = both(0.f);
            k_sums.read_all(l, K_MU, mu), k_sums.read_all(l, K_A, fa), k_sums.read_all(l, K_B, fb);
            const float b_most = ACT == ACT_RELU ? largest(fb) : 0.f;
            int rows = 0;
            for (bool more = true; more;) {
                const T *x = rows_at();
                uint32_t unsettled = 0, round = 1;
                if (mine)
#pragma unroll 1   // (two at a time spill registers)
                    for (int r = l.lane, at = l.lane * p.V; r < t.n; r += l.lanes, at += step, round <<= 2) {
                        BackwardRows<T, VN, ACT, DROP, 1> in;
                        in.x.v[0].load(x + at);
                        in.g.v[0].load(x + tensor + at);
                        if (p.residual) in.res.v[0].load(x + 2 * tensor + at);
                        if (DROP) rng.template words<VN>((uint64_t)(t.from + at + c0), in.words[0]);
                        const bool part = PHASES && cut(at + c0);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float2 xc[2], gz[2];
                            if constexpr (ACT == ACT_RELU) unsettled |= in.template gz_told<true>(p, h, b_most, mu, fa, fb, xc, gz) ? round << h : 0;
                            else in.template gz<2, false>(p, s, c0, 0, 2 * h, mu + 2 * h, fa + 2 * h, fb + 2 * h, xc, gz);
                            if (part) {
                                const int2 e = ends();
#pragma unroll
                                for (int i = 0; i < 2; ++i) xc[i] = within(xc[i], at + c0 + 4 * h + 2 * i, e.x, e.y), gz[i] = within(gz[i], at + c0 + 4 * h + 2 * i, e.x, e.y);
                            }
#pragma unroll
                            for (int i = 0; i < 2; ++i) a[2 * h + i] = add2(a[2 * h + i], gz[i]), b[2 * h + i] = fma2(gz[i], xc[i], b[2 * h + i]);
                        }
                    }
                bool lost = false;
                if constexpr (ACT == ACT_RELU && BACKWARD)
                    if (__any_sync(0xffffffffu, unsettled != 0)) {
                        lost = !ask(ASK_SUMS, unsettled);
                        const Asked &asked = *reinterpret_cast<const Asked *>(m.scratch);
#pragma unroll
                        for (int j = 0; j < P; ++j) a[j] = add2(a[j], asked.sums[2 * j][threadIdx.x & 31]), b[j] = add2(b[j], asked.sums[2 * j + 1][threadIdx.x & 31]);
                        __syncwarp();
                        if ((threadIdx.x & 31) == 0) ring.asked[threadIdx.x >> 5] = ASK_NOTHING;
                    }
                rows = t.last;
                more = !rows;
                release();
                next_tile();
                if (lost) t.kind = TILE_NONE;
                if (t.kind == TILE_NONE) more = false;
            }
            if (!next_slot()) t.kind = TILE_NONE;
            if constexpr (BACKWARD)
                if (t.kind != TILE_NONE)
                    fold_and_send(Piece{TILE_SUMS, s, chunk, rows}, [&](int i) { return i % 2 ? make_float2(a[i / 2].y, b[i / 2].y) : make_float2(a[i / 2].x, b[i / 2].x); });
        } else if (t.kind == TILE_APPLY) {
            const int s = t.s;
            if (k_apply.s != s) {
                if (!sync_workers_and(true)) break;
                if (!k_apply.template load<PHASES>(p, l, s, 0, true)) break;
            }
            float2 mu[P], fa[P], fb[P], m1[P], m2[P];
            k_apply.read_all(l, K_MU, mu), k_apply.read_all(l, K_A, fa), k_apply.read_all(l, K_B, fb);
            if constexpr (BACKWARD) k_apply.read_all(l, K_M1, m1), k_apply.read_all(l, K_M2, m2);
            const float b_most = ACT == ACT_RELU ? largest(fb) : 0.f;
            do {
                const T *x = rows_at();
                if (!BACKWARD && t.last) k_apply.put_stats(p, l);
                uint32_t unsettled = 0, round = 1;
                if (mine)
#pragma unroll 1   // (two at a time spill registers)
                    for (int r = l.lane, at = l.lane * p.V; r < t.n; r += l.lanes, at += step, round <<= 2) {
                        const int64_t to = t.from + at + c0;
                        BackwardRows<T, VN, ACT, DROP, 1> in;
                        in.x.v[0].load(x + at);
                        if constexpr (BACKWARD) in.g.v[0].load(x + tensor + at);
                        if (p.residual) in.res.v[0].load(x + (BACKWARD ? 2 : 1) * tensor + at);
                        if (DROP) rng.template words<VN>((uint64_t)to, in.words[0]);
                        if constexpr (BACKWARD) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float2 xc[2], gz[2];
                                if constexpr (ACT == ACT_RELU) unsettled |= in.template gz_told<false>(p, h, b_most, mu, fa, fb, xc, gz) ? round << h : 0;
                                else in.template gz<2, false>(p, s, c0, 0, 2 * h, mu + 2 * h, fa + 2 * h, fb + 2 * h, xc, gz);
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    const int j = 2 * h + i;
                                    set_pair(in.g.v[0], j, gz[i]);
                                    set_pair(in.x.v[0], j, fma2(gz[i], fa[j], fma2(xc[i], m2[j], m1[j])));
                                }
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < P; ++j) {
                                float2 z = fma2(add2(pair_of(in.x.v[0], j), mu[j]), fa[j], fb[j]);
                                if (p.residual) z = add2(z, pair_of(in.res.v[0], j));
                                z = act2<T>(ACT, z);
                                if (DROP) z = drop2<VN>(p, in.words[0], j, z);
                                set_pair(in.x.v[0], j, z);
                            }
                        }
                        if (PHASES && cut(at + c0)) {
                            const int2 e = ends();
                            if (BACKWARD && p.dresidual) in.g.v[0].store_part(static_cast<T *>(p.dresidual) + to, e.x - at - c0, e.y - at - c0);
                            in.x.v[0].store_part(static_cast<T *>(BACKWARD ? p.dx : p.y) + to, e.x - at - c0, e.y - at - c0);
                        } else {
                            if (BACKWARD && p.dresidual) in.g.v[0].store_streaming(static_cast<T *>(p.dresidual) + to);
                            in.x.v[0].store_streaming(static_cast<T *>(BACKWARD ? p.dx : p.y) + to);
                        }
                    }
                bool lost = false;
                if constexpr (ACT == ACT_RELU && BACKWARD)
                    if (__any_sync(0xffffffffu, unsettled != 0)) lost = !ask(ASK_APPLY, unsettled);
                release();
                next_tile();
                if (lost) t.kind = TILE_NONE;
            } while (t.kind == TILE_APPLY && t.s == s);
        } else {
            if (!sync_workers_and(t.kind != TILE_NONE)) break;
            if (t.kind == TILE_END) {
                if (!next_slot()) break;
                send(Piece{TILE_END, 0, 0, 0});
                return;
            }
            if (!wait_for(p.control + WINDOWS_DONE, p.control[WINDOWS], p.status)) break;
            affine_gradients(p, t.chunk, reinterpret_cast<double2 *>(m.scratch));
            release();
            next_tile();
        }
    }
    ring.abort = 1;
}

// PHASES: several rows side by side.  (Always so, the samples' ends cost registers where none is inside of a row: at 1.1 million points of
// 64 channels, bf16, 236 us backward for 221 and 118 forward for 107.)
template <typename T, int ACT, int DROP, bool BACKWARD, bool PHASES>
__global__ void __launch_bounds__(RING_THREADS, RING_BLOCKS) na_ring_kernel(const __grid_constant__ NormAct p) {
    extern __shared__ __align__(128) char shared[];
    __shared__ Ring ring;
    if (threadIdx.x == 0) {
        for (int q = 0; q < p.stages; ++q) tc::mbar_init(tc::smem_u32(&ring.full[q]), 1), tc::mbar_init(tc::smem_u32(&ring.empty[q]), NA_THREADS / 32);
        for (int q = 0; q < FOLD_SLOTS; ++q) tc::mbar_init(tc::smem_u32(&ring.folded[q]), NA_THREADS / 32), tc::mbar_init(tc::smem_u32(&ring.taken[q]), 1);
        ring.abort = 0;
        for (int w = 0; w < NA_THREADS / 32; ++w) ring.asked[w] = ASK_NOTHING;
        tc::fence_mbar_init();
    }
    start_after_previous();
    __syncthreads();
    const RingMemory m(p, shared);
    if (threadIdx.x < NA_THREADS) ring_worker<T, ACT, DROP, BACKWARD, PHASES>(p, ring, m);
    else if (threadIdx.x < NA_THREADS + 32) ring_producer<T, BACKWARD, PHASES>(p, ring, m);
    else ring_clerk<T, ACT, DROP, BACKWARD, PHASES>(p, ring, m);
}

template <typename T, int ACT, int DROP, bool BACKWARD, bool PHASES>
int run_phases(const NormAct &p, cudaStream_t stream) {
    const auto kernel = na_ring_kernel<T, ACT, DROP, BACKWARD, PHASES>;
    static std::atomic<uint64_t> allowed;
    if (int rc = allow_shared_memory((const void *)kernel, &allowed, true)) return rc;
    const int64_t tickets = 2 * (int64_t)p.chunks;
    launch_after(kernel, (unsigned)std::min<int64_t>(tickets, RING_BLOCKS * num_sms()), RING_THREADS, (size_t)p.stages * p.stage_bytes + ring_bytes(p.V, p.G, BACKWARD), stream, p);
    PCX_LAUNCH_CHECK();
    return PCX_OK;
}

template <typename T, int ACT, int DROP, bool BACKWARD>
int run_ring(const NormAct &p, cudaStream_t stream) {
    return p.phase_bits ? run_phases<T, ACT, DROP, BACKWARD, true>(p, stream) : run_phases<T, ACT, DROP, BACKWARD, false>(p, stream);
}

template <typename T, int VN, int ACT, int DROP, bool BACKWARD>
int run_kernel(const NormAct &p, cudaStream_t stream) {
    const auto kernel = na_kernel<T, VN, ACT, DROP, BACKWARD>;
    static std::atomic<uint64_t> allowed;
    const size_t smem = shared_bytes<VN, BACKWARD>(p.C);
    if (smem > 40 << 10)
        if (int rc = allow_shared_memory((const void *)kernel, &allowed)) return rc;
    const int64_t tickets = 2 * (int64_t)p.chunks + (BACKWARD && p.dweight ? (p.C + AFFINE_CHANNELS - 1) / AFFINE_CHANNELS : 0);
    launch_after(kernel, (unsigned)std::min<int64_t>(tickets, NA_BLOCKS * num_sms()), NA_THREADS, smem, stream, p);
    PCX_LAUNCH_CHECK();
    return PCX_OK;
}
template <typename T, bool BACKWARD, int DROP>
int run_act(const NormAct &p, cudaStream_t stream) {
    if (p.act == ACT_RELU) return run_ring<T, ACT_RELU, DROP, BACKWARD>(p, stream);
    if (p.act == ACT_SILU) return run_ring<T, ACT_SILU, DROP, BACKWARD>(p, stream);
    if (p.act == ACT_GELU) return run_ring<T, ACT_GELU, DROP, BACKWARD>(p, stream);
    return run_ring<T, ACT_NONE, DROP, BACKWARD>(p, stream);
}
template <typename T, bool BACKWARD>
int run_lump(const NormAct &p, int vn, cudaStream_t stream) {
    if (p.stages) return !p.drop.on ? run_act<T, BACKWARD, 0>(p, stream) : p.drop.state ? run_act<T, BACKWARD, 2>(p, stream) : run_act<T, BACKWARD, 1>(p, stream);
    if (vn == 8) return run_kernel<T, 8, -1, -1, BACKWARD>(p, stream);
    if (vn == 4) return run_kernel<T, 4, -1, -1, BACKWARD>(p, stream);
    if (vn == 2) return run_kernel<T, 2, -1, -1, BACKWARD>(p, stream);
    return run_kernel<T, 1, -1, -1, BACKWARD>(p, stream);
}

}  // namespace

template <typename T>
int norm_act_rows(const NormAct &p, int vn, bool backward, cudaStream_t stream) {
    return backward ? run_lump<T, true>(p, vn, stream) : run_lump<T, false>(p, vn, stream);
}
#endif

}  // namespace pcx
