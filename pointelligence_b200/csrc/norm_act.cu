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
// Everything is held in fp32 between one read of an element and its one rounding; sums of chunks are merged in fp64.
//
// Both directions take two passes over the rows, with sums between them.  A chunk is `rows` consecutive rows; a piece is what a
// chunk has of one sample, piece chunk + s (pieces are ordered, and the next one has a higher chunk or a higher sample by one).
// A block leaves two floats per channel and piece, whatever the group's width; they are merged in a fixed order, so that
// results do not depend on scheduling, and no float is ever added by an atomic:
//   forward   mean and sum of squares about it.  A block sums x - k and its square, k the channel's value in the piece's first row:
//             as k is one of the n summed values, (k - mean)^2 is at most their sum of squares M2, and what cancels in
//             sum (x - k)^2 - n (mean - k)^2 is at most (n + 1) M2: n + 1 roundings at worst, one where rows are alike.
//   backward  sums of gz and gz * xh.
#include <algorithm>

#include "philox.cuh"
#include "rowwise.cuh"

namespace pcx {
namespace {

constexpr int NA_THREADS = 256;
constexpr int NA_CHUNK_BYTES = 32 << 10;
constexpr int NA_MAX_C = 1 << 16;

struct NormAct {
    const void *x, *residual, *g;
    void *y, *dx, *dresidual;
    const float *weight, *bias;
    float *mean, *rstd;            // (S, G)
    float *dweight, *dbias;
    int64_t *offsets;              // (S + 1)
    float2 *rec;                   // (pieces, C)
    float2 *of_sample;             // (S, C): mean and M2; or sums of gz and gz * xh
    float2 *of_group;              // (S, G): the backward's two means
    int64_t N, S;
    int C, G, W, rows;
    uint32_t by_width;             // c / W = c * by_width >> 32 (c * W < 2^32); W = 1: c
    float eps;
    Dropping drop;
};

__device__ __forceinline__ int group_of(const NormAct &p, int c) { return p.W == 1 ? c : (int)__umulhi((uint32_t)c, p.by_width); }

// ------------------------------------------------------------ columns ----
// Channels of a block: passes of `cols` lumps side by side, `lanes` rows.
struct Columns {
    int lumps, cols, lanes, passes, col, lane;
    template <int VN>
    __device__ __forceinline__ static Columns make(int C) {
        Columns l;
        l.lumps = C / VN;
        l.passes = (l.lumps + NA_THREADS - 1) / NA_THREADS;
        l.cols = (l.lumps + l.passes - 1) / l.passes;
        l.lanes = NA_THREADS / l.cols;
        l.col = threadIdx.x % l.cols, l.lane = threadIdx.x / l.cols;
        return l;
    }
};

// ------------------------------------------------------------ activations ----
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

template <int ACT>
__device__ __forceinline__ float act(float z) {
    if constexpr (ACT == ACT_RELU) return relu(z);
    if constexpr (ACT == ACT_SILU) return z * __fdividef(1.f, 1.f + __expf(-z));
    if constexpr (ACT == ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678f));
    return z;
}
template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if constexpr (ACT == ACT_SILU) {
        const float s = __fdividef(1.f, 1.f + __expf(-z));
        return s * (1.f + z * (1.f - s));
    }
    if constexpr (ACT == ACT_GELU) return 0.5f * (1.f + erff(z * 0.70710678f)) + z * 0.39894228f * __expf(-0.5f * z * z);
    return 1.f;
}

// ------------------------------------------------------------ offsets ----
// Row offsets of the samples.  Whatever the lengths say, they ascend within 0 .. N, and rows behind the last sample are its own.
constexpr int OFFSETS_THREADS = 1024;
__global__ void __launch_bounds__(OFFSETS_THREADS) na_offsets_kernel(const int64_t *__restrict__ lengths, int64_t *offsets, int64_t S, int64_t N) {
    start_after_previous();
    __shared__ int64_t sums[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t carry = 0;
    for (int64_t base = 0; base < S; base += blockDim.x) {
        const int64_t s = base + threadIdx.x;
        const int64_t v = s < S ? min(max(lengths[s], (int64_t)0), N) : 0;
        int64_t up_to = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t before = __shfl_up_sync(0xffffffffu, up_to, o);
            if (lane >= o) up_to = min(up_to + before, N);
        }
        const int64_t in_warp = __shfl_up_sync(0xffffffffu, up_to, 1);   // (of sums that stop at N no length can be taken off again)
        if (lane == 31) sums[warp] = up_to;
        __syncthreads();
        int64_t before = carry, all = carry;
        for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
            if (w < warp) before = min(before + sums[w], N);
            all = min(all + sums[w], N);
        }
        if (s < S) offsets[s] = min(before + (lane ? in_warp : 0), N);
        carry = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) offsets[S] = N;
}

// ------------------------------------------------------------ sums of a piece ----
// Two sums per channel of a thread's rows, folded over the block's row lanes; `out(c, a, b)` for every channel.
template <int VN, typename Out>
__device__ __forceinline__ void fold_lanes(const Columns &l, int pass, int C, const float *a, const float *b, float2 *fold, Out out) {
    __syncthreads();   // (the piece before has been read)
#pragma unroll
    for (int i = 0; i < VN; ++i) fold[i * NA_THREADS + threadIdx.x] = make_float2(a[i], b[i]);
    __syncthreads();
    for (int t = threadIdx.x; t < l.cols * VN; t += NA_THREADS) {
        const int i = t / l.cols, col = t % l.cols, lump = pass * l.cols + col;
        float sa = 0.f, sb = 0.f;
#pragma unroll 8
        for (int q = 0; q < l.lanes; ++q) {
            const float2 v = fold[i * NA_THREADS + q * l.cols + col];
            sa += v.x, sb += v.y;
        }
        if (lump < l.lumps) out(lump * VN + i, sa, sb);
    }
}

constexpr int NA_UNROLL = 4;   // rows a thread has in flight

template <typename T, int VN>
__device__ __forceinline__ void stats_piece(const NormAct &p, const Columns &l, int64_t piece, int64_t lo, int64_t hi, float2 *fold) {
    const T *x = static_cast<const T *>(p.x);
    for (int pass = 0; pass < l.passes; ++pass) {
        const int lump = pass * l.cols + l.col;
        const bool mine = lump < l.lumps && l.lane < l.lanes;
        float a[VN], b[VN];
#pragma unroll
        for (int i = 0; i < VN; ++i) a[i] = b[i] = 0.f;
        if (mine) {
            const T *col = x + (int64_t)lump * VN;
            Lump<T, VN> first;
            first.load(col + lo * p.C);
            for (int64_t r = lo + l.lane; r < hi; r += (int64_t)NA_UNROLL * l.lanes) {
                Lump<T, VN> v[NA_UNROLL];
#pragma unroll
                for (int u = 0; u < NA_UNROLL; ++u)
                    if (r + (int64_t)u * l.lanes < hi) v[u].load(col + (r + (int64_t)u * l.lanes) * p.C);
                    else v[u] = first;   // adds nothing
#pragma unroll
                for (int u = 0; u < NA_UNROLL; ++u)
#pragma unroll
                    for (int i = 0; i < VN; ++i) {
                        const float d = v[u].get(i) - first.get(i);
                        a[i] += d, b[i] += d * d;
                    }
            }
        }
        fold_lanes<VN>(l, pass, p.C, a, b, fold, [&](int c, float sa, float sb) {
            const float n = (float)(hi - lo), off = sa / n;
            p.rec[piece * p.C + c] = make_float2(to_f32<T>(x[lo * p.C + c]) + off, fmaxf(sb - sa * off, 0.f));
        });
    }
}

// What a thread keeps of the affine map of its channels in one sample.
template <int VN>
struct Affine {
    float mu[VN], a[VN], b[VN];   // z = (x - mu) * a + b
    __device__ __forceinline__ void load(const NormAct &p, int64_t s, int c0) {
#pragma unroll
        for (int i = 0; i < VN; ++i) {
            const int64_t at = s * p.G + group_of(p, c0 + i);
            mu[i] = p.mean[at];
            a[i] = p.rstd[at] * (p.weight ? p.weight[c0 + i] : 1.f);
            b[i] = p.weight ? p.bias[c0 + i] : 0.f;
        }
    }
};

template <typename T, int VN, int ACT>
__device__ __forceinline__ void apply_piece(const NormAct &p, const Columns &l, const Philox &rng, int64_t s, int64_t lo, int64_t hi) {
    const T *x = static_cast<const T *>(p.x), *res = static_cast<const T *>(p.residual);
    for (int pass = 0; pass < l.passes; ++pass) {
        const int lump = pass * l.cols + l.col, c0 = lump * VN;
        if (lump >= l.lumps || l.lane >= l.lanes) continue;
        Affine<VN> f;
        f.load(p, s, c0);
        for (int64_t r = lo + l.lane; r < hi; r += (int64_t)NA_UNROLL * l.lanes) {
            Lump<T, VN> v[NA_UNROLL], q[NA_UNROLL];
#pragma unroll
            for (int u = 0; u < NA_UNROLL; ++u)
                if (r + (int64_t)u * l.lanes < hi) v[u].load(x + (r + (int64_t)u * l.lanes) * p.C + c0);
            if (res) {
#pragma unroll
                for (int u = 0; u < NA_UNROLL; ++u)
                    if (r + (int64_t)u * l.lanes < hi) q[u].load(res + (r + (int64_t)u * l.lanes) * p.C + c0);
            }
#pragma unroll
            for (int u = 0; u < NA_UNROLL; ++u) {
                const int64_t at = (r + (int64_t)u * l.lanes) * p.C + c0;
                if (r + (int64_t)u * l.lanes >= hi) break;
                const uint32_t kept = p.drop.on ? rng.kept<VN>((uint64_t)at, p.drop.over) : 0;
                Lump<T, VN> out;
#pragma unroll
                for (int i = 0; i < VN; ++i) {
                    float z = (v[u].get(i) - f.mu[i]) * f.a[i] + f.b[i];
                    if (res) z += q[u].get(i);
                    z = act<ACT>(z);
                    if (p.drop.on) z = kept >> i & 1 ? z * p.drop.scale : 0.f;
                    out.set(i, z);
                }
                out.store(static_cast<T *>(p.y) + at);
            }
        }
    }
}

// gz of one lump
template <typename T, int VN, int ACT>
__device__ __forceinline__ void grad_z(const NormAct &p, const Affine<VN> &f, const Lump<T, VN> &g, const float *xc, const Lump<T, VN> &res, uint32_t kept, float *gz) {
#pragma unroll
    for (int i = 0; i < VN; ++i) {
        float z = xc[i] * f.a[i] + f.b[i];
        if (p.residual) z += res.get(i);
        gz[i] = g.get(i) * slope<ACT>(z);
        if (ACT == ACT_RELU) gz[i] = z > 0.f ? g.get(i) : 0.f;
        if (p.drop.on) gz[i] = kept >> i & 1 ? gz[i] * p.drop.scale : 0.f;
    }
}

template <typename T, int VN, int ACT>
__device__ __forceinline__ void bwd_sums_piece(const NormAct &p, const Columns &l, const Philox &rng, int64_t piece, int64_t s, int64_t lo, int64_t hi, float2 *fold) {
    const T *x = static_cast<const T *>(p.x), *res = static_cast<const T *>(p.residual), *g = static_cast<const T *>(p.g);
    constexpr int U = NA_UNROLL / 2;
    for (int pass = 0; pass < l.passes; ++pass) {
        const int lump = pass * l.cols + l.col, c0 = lump * VN;
        float a[VN], b[VN];
#pragma unroll
        for (int i = 0; i < VN; ++i) a[i] = b[i] = 0.f;
        if (lump < l.lumps && l.lane < l.lanes) {
            Affine<VN> f;
            f.load(p, s, c0);
            for (int64_t r = lo + l.lane; r < hi; r += (int64_t)U * l.lanes) {
                Lump<T, VN> xv[U], gv[U], q[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r + (int64_t)u * l.lanes < hi) {
                        const int64_t at = (r + (int64_t)u * l.lanes) * p.C + c0;
                        xv[u].load(x + at), gv[u].load(g + at);
                        if (res) q[u].load(res + at);
                    }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t at = (r + (int64_t)u * l.lanes) * p.C + c0;
                    if (r + (int64_t)u * l.lanes >= hi) break;
                    const uint32_t kept = p.drop.on ? rng.kept<VN>((uint64_t)at, p.drop.over) : 0;
                    float xc[VN], gz[VN];
#pragma unroll
                    for (int i = 0; i < VN; ++i) xc[i] = xv[u].get(i) - f.mu[i];
                    grad_z<T, VN, ACT>(p, f, gv[u], xc, q[u], kept, gz);
#pragma unroll
                    for (int i = 0; i < VN; ++i) a[i] += gz[i], b[i] += gz[i] * xc[i];
                }
            }
        }
        fold_lanes<VN>(l, pass, p.C, a, b, fold, [&](int c, float sa, float sb) {
            p.rec[piece * p.C + c] = make_float2(sa, sb * p.rstd[s * p.G + group_of(p, c)]);
        });
    }
}

template <typename T, int VN, int ACT>
__device__ __forceinline__ void bwd_apply_piece(const NormAct &p, const Columns &l, const Philox &rng, int64_t s, int64_t lo, int64_t hi) {
    const T *x = static_cast<const T *>(p.x), *res = static_cast<const T *>(p.residual), *g = static_cast<const T *>(p.g);
    constexpr int U = NA_UNROLL / 2;
    for (int pass = 0; pass < l.passes; ++pass) {
        const int lump = pass * l.cols + l.col, c0 = lump * VN;
        if (lump >= l.lumps || l.lane >= l.lanes) continue;
        Affine<VN> f;
        f.load(p, s, c0);
        float m1[VN], m2[VN];   // dx = gz * a - m1 - xc * m2
#pragma unroll
        for (int i = 0; i < VN; ++i) {
            const int64_t at = s * p.G + group_of(p, c0 + i);
            const float2 m = p.of_group[at];
            const float rs = p.rstd[at];
            m1[i] = m.x * rs, m2[i] = m.y * rs * rs;
        }
        for (int64_t r = lo + l.lane; r < hi; r += (int64_t)U * l.lanes) {
            Lump<T, VN> xv[U], gv[U], q[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + (int64_t)u * l.lanes < hi) {
                    const int64_t at = (r + (int64_t)u * l.lanes) * p.C + c0;
                    xv[u].load(x + at), gv[u].load(g + at);
                    if (res) q[u].load(res + at);
                }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = (r + (int64_t)u * l.lanes) * p.C + c0;
                if (r + (int64_t)u * l.lanes >= hi) break;
                const uint32_t kept = p.drop.on ? rng.kept<VN>((uint64_t)at, p.drop.over) : 0;
                float xc[VN], gz[VN];
#pragma unroll
                for (int i = 0; i < VN; ++i) xc[i] = xv[u].get(i) - f.mu[i];
                grad_z<T, VN, ACT>(p, f, gv[u], xc, q[u], kept, gz);
                Lump<T, VN> out;
                if (p.dresidual) {
#pragma unroll
                    for (int i = 0; i < VN; ++i) out.set(i, gz[i]);
                    out.store(static_cast<T *>(p.dresidual) + at);
                }
#pragma unroll
                for (int i = 0; i < VN; ++i) out.set(i, gz[i] * f.a[i] - m1[i] - xc[i] * m2[i]);
                out.store(static_cast<T *>(p.dx) + at);
            }
        }
    }
}

// ------------------------------------------------------------ kernels ----
enum { STATS = 0, APPLY = 1, BWD_SUMS = 2, BWD_APPLY = 3 };

template <typename T, int VN, int ACT, int PASS>
__global__ void __launch_bounds__(NA_THREADS, PASS == STATS || PASS == APPLY ? 4 : 3) na_rows_kernel(const __grid_constant__ NormAct p) {
    start_after_previous();
    __shared__ float2 fold[PASS == STATS || PASS == BWD_SUMS ? VN * NA_THREADS : 1];
    const Columns l = Columns::make<VN>(p.C);
    const Philox rng(p.drop);
    const int64_t row0 = (int64_t)blockIdx.x * p.rows, row1 = min(p.N, row0 + p.rows);
    const int64_t s_first = segment_of_row(p.offsets, p.S, row0);
    for (int64_t s = s_first; s < p.S && p.offsets[s] < row1; ++s) {
        const int64_t lo = max(row0, p.offsets[s]), hi = min(row1, p.offsets[s + 1]);
        if (hi <= lo) continue;   // a sample without rows
        if constexpr (PASS == STATS) stats_piece<T, VN>(p, l, blockIdx.x + s, lo, hi, fold);
        if constexpr (PASS == APPLY) apply_piece<T, VN, ACT>(p, l, rng, s, lo, hi);
        if constexpr (PASS == BWD_SUMS) bwd_sums_piece<T, VN, ACT>(p, l, rng, blockIdx.x + s, s, lo, hi, fold);
        if constexpr (PASS == BWD_APPLY) bwd_apply_piece<T, VN, ACT>(p, l, rng, s, lo, hi);
    }
}

// A block per sample merges the records of its pieces: a warp a channel, then a thread a group.
template <bool BACKWARD>
__global__ void __launch_bounds__(NA_THREADS) na_merge_kernel(const __grid_constant__ NormAct p) {
    start_after_previous();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t s = blockIdx.x, lo = p.offsets[s], hi = p.offsets[s + 1], n = hi - lo;
    const int64_t b0 = lo / p.rows, b1 = n > 0 ? (hi - 1) / p.rows : b0 - 1;
    for (int c = warp; c < p.C; c += NA_THREADS / 32) {
        double sum = 0.0, second = 0.0;
        for (int64_t b = b0 + lane; b <= b1; b += 32) {
            const float2 v = p.rec[(b + s) * p.C + c];
            if constexpr (BACKWARD) {
                sum += v.x, second += v.y;
            } else {
                sum += (double)(min(hi, (b + 1) * p.rows) - max(lo, b * p.rows)) * v.x;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            second += __shfl_xor_sync(0xffffffffu, second, o);
        }
        if constexpr (!BACKWARD) {
            sum /= (double)max(n, (int64_t)1);
            for (int64_t b = b0 + lane; b <= b1; b += 32) {
                const float2 v = p.rec[(b + s) * p.C + c];
                const double d = (double)v.x - sum;
                second += (double)v.y + (double)(min(hi, (b + 1) * p.rows) - max(lo, b * p.rows)) * d * d;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) second += __shfl_xor_sync(0xffffffffu, second, o);
        }
        if (lane == 0) p.of_sample[s * p.C + c] = make_float2((float)sum, (float)second);
    }
    __syncthreads();
    for (int g = warp; g < p.G; g += NA_THREADS / 32) {
        double a = 0.0, b = 0.0;
        const float2 *v = p.of_sample + s * p.C + (int64_t)g * p.W;
        for (int c = lane; c < p.W; c += 32) {
            const double w = BACKWARD && p.weight ? (double)p.weight[g * p.W + c] : 1.0;
            a += w * v[c].x;
            if constexpr (BACKWARD) b += w * v[c].y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        const double count = (double)max(n, (int64_t)1) * p.W;
        if constexpr (BACKWARD) {
            if (lane == 0) p.of_group[s * p.G + g] = make_float2((float)(a / count), (float)(b / count));
        } else {
            const double mu = a / p.W;
            for (int c = lane; c < p.W; c += 32) {
                const double d = (double)v[c].x - mu;
                b += (double)v[c].y + (double)n * d * d;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) b += __shfl_xor_sync(0xffffffffu, b, o);
            if (lane == 0) p.mean[s * p.G + g] = (float)mu, p.rstd[s * p.G + g] = (float)(1.0 / sqrt(b / count + (double)p.eps));
        }
    }
}

// dweight, dbias: a warp a channel over the samples' sums, in a fixed order.
__global__ void __launch_bounds__(NA_THREADS) na_affine_kernel(const __grid_constant__ NormAct p) {
    start_after_previous();
    const int lane = threadIdx.x & 31, c = blockIdx.x * (NA_THREADS / 32) + (threadIdx.x >> 5);
    if (c >= p.C) return;
    double a = 0.0, b = 0.0;
    for (int64_t s = lane; s < p.S; s += 32) {
        const float2 v = p.of_sample[s * p.C + c];
        a += v.x, b += v.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    if (lane == 0) p.dbias[c] = (float)a, p.dweight[c] = (float)b;
}

// ------------------------------------------------------------ host ----
// Rows of a chunk: 32 KB of them, fewer where that would leave multiprocessors without one.
int chunk_rows(int64_t N, int C, int dtype) {
    const int64_t by_bytes = NA_CHUNK_BYTES / ((int64_t)C * (int64_t)elem_size(dtype)), by_chip = (N + 4 * num_sms() - 1) / (4 * num_sms());
    return (int)std::max<int64_t>(1, std::min(by_bytes, by_chip));
}

size_t carve(void *ws, int64_t N, int64_t S, int C, int G, int dtype, NormAct *out) {
    Carver c(ws);
    NormAct p = out ? *out : NormAct{};
    p.rows = chunk_rows(N, C, dtype);
    p.offsets = c.take<int64_t>((size_t)S + 1);
    p.rec = c.take<float2>((size_t)((N + p.rows - 1) / p.rows + S) * C);
    p.of_sample = c.take<float2>((size_t)S * C);
    p.of_group = c.take<float2>((size_t)S * G);
    if (out) *out = p;
    return c.off;
}

bool sizes_ok(int64_t N, int64_t S, int C, int G, int dtype, int activation) {
    return N >= 0 && S > 0 && S <= INT32_MAX && C > 0 && C <= NA_MAX_C && G > 0 && C % G == 0 && S * (int64_t)C <= INT32_MAX &&
           (dtype == PCX_F32 || dtype == PCX_F16 || dtype == PCX_BF16) && activation >= ACT_NONE && activation <= ACT_GELU &&
           (N == 0 || N <= INT64_MAX / 8 / C) && N / chunk_rows(std::max<int64_t>(N, 1), C, dtype) < INT32_MAX;
}

template <typename T, int VN, int ACT>
int run_rows(const NormAct &p, int pass, cudaStream_t stream) {
    const unsigned grid = (unsigned)((p.N + p.rows - 1) / p.rows);
    if (pass == STATS) launch_after(na_rows_kernel<T, VN, ACT_NONE, STATS>, grid, NA_THREADS, 0, stream, p);
    if (pass == APPLY) launch_after(na_rows_kernel<T, VN, ACT, APPLY>, grid, NA_THREADS, 0, stream, p);
    if (pass == BWD_SUMS) launch_after(na_rows_kernel<T, VN, ACT, BWD_SUMS>, grid, NA_THREADS, 0, stream, p);
    if (pass == BWD_APPLY) launch_after(na_rows_kernel<T, VN, ACT, BWD_APPLY>, grid, NA_THREADS, 0, stream, p);
    PCX_LAUNCH_CHECK();
    return PCX_OK;
}
template <typename T, int VN>
int run_act(const NormAct &p, int activation, int pass, cudaStream_t stream) {
    if (activation == ACT_RELU) return run_rows<T, VN, ACT_RELU>(p, pass, stream);
    if (activation == ACT_SILU) return run_rows<T, VN, ACT_SILU>(p, pass, stream);
    if (activation == ACT_GELU) return run_rows<T, VN, ACT_GELU>(p, pass, stream);
    return run_rows<T, VN, ACT_NONE>(p, pass, stream);
}
template <typename T>
int run_lump(const NormAct &p, int vn, int activation, int pass, cudaStream_t stream) {
    if (vn == 8) return run_act<T, 8>(p, activation, pass, stream);
    if (vn == 4) return run_act<T, 4>(p, activation, pass, stream);
    if (vn == 2) return run_act<T, 2>(p, activation, pass, stream);
    return run_act<T, 1>(p, activation, pass, stream);
}
int run(const NormAct &p, int dtype, int vn, int activation, int pass, cudaStream_t stream) {
    if (dtype == PCX_F32) return run_lump<float>(p, vn, activation, pass, stream);
    if (dtype == PCX_F16) return run_lump<__half>(p, vn, activation, pass, stream);
    return run_lump<__nv_bfloat16>(p, vn, activation, pass, stream);
}

}  // namespace

int sample_offsets(const int64_t *d_lengths, int64_t *offsets, int64_t S, int64_t N, cudaStream_t stream) {
    launch_after(na_offsets_kernel, 1, S <= 256 ? 256 : OFFSETS_THREADS, 0, stream, d_lengths, offsets, S, N);
    PCX_LAUNCH_CHECK();
    return PCX_OK;
}

}  // namespace pcx

using namespace pcx;

extern "C" {

size_t pcx_ragged_group_norm_act_workspace_bytes(int64_t N, int64_t S, int C, int G, int dtype) {
    return sizes_ok(N, S, C, G, dtype, ACT_NONE) ? carve(nullptr, N, S, C, G, dtype, nullptr) : 0;
}

int pcx_ragged_group_norm_act(const void *d_x, const int64_t *d_lengths, const float *d_weight, const float *d_bias, const void *d_residual, void *d_y,
                              float *d_mean, float *d_rstd, int64_t N, int64_t S, int C, int G, double eps, int activation, double dropout, uint64_t seed,
                              uint64_t offset, const int64_t *d_rng, int dtype, void *d_ws, size_t ws_bytes, void *stream_) {
    cudaStream_t stream = (cudaStream_t)stream_;
    if (!sizes_ok(N, S, C, G, dtype, activation))
        PCX_FAIL(PCX_E_ARG, "pcx_ragged_group_norm_act: bad sizes, activation or dtype (C <= %d must be a multiple of G)", NA_MAX_C);
    if (!d_lengths || !d_mean || !d_rstd || !d_ws || (N > 0 && (!d_x || !d_y)) || ((d_weight == nullptr) != (d_bias == nullptr)))
        PCX_FAIL(PCX_E_ARG, "pcx_ragged_group_norm_act: null pointer (weight and bias come together)");
    if ((uintptr_t)d_ws % 256) PCX_FAIL(PCX_E_ALIGN, "pcx_ragged_group_norm_act: workspace must be 256-byte aligned");
    NormAct p = {};
    if (!make_dropping(dropout, seed, offset, d_rng, &p.drop)) PCX_FAIL(PCX_E_ARG, "pcx_ragged_group_norm_act: dropout %g is no probability", dropout);
    const size_t need = carve(d_ws, N, S, C, G, dtype, &p);
    if (ws_bytes < need) PCX_FAIL(PCX_E_CAPACITY, "pcx_ragged_group_norm_act: workspace %zu < %zu bytes", ws_bytes, need);
    p.x = d_x, p.residual = d_residual, p.y = d_y, p.weight = d_weight, p.bias = d_bias, p.mean = d_mean, p.rstd = d_rstd;
    p.N = N, p.S = S, p.C = C, p.G = G, p.W = C / G, p.by_width = (uint32_t)((0xFFFFFFFFull + p.W) / p.W), p.eps = (float)eps;
    const int vn = lump_of(C, dtype, {d_x, d_residual, d_y});
    prof_begin("group_norm_act(fwd)", stream);
    if (int rc = sample_offsets(d_lengths, p.offsets, S, N, stream)) return rc;
    if (N > 0)
        if (int rc = run(p, dtype, vn, activation, STATS, stream)) return rc;
    launch_after(na_merge_kernel<false>, (unsigned)S, NA_THREADS, 0, stream, p);
    PCX_LAUNCH_CHECK();
    if (N > 0)
        if (int rc = run(p, dtype, vn, activation, APPLY, stream)) return rc;
    prof_end(stream);
    return PCX_OK;
}

int pcx_ragged_group_norm_act_backward(const void *d_grad_y, const void *d_x, const void *d_residual, const int64_t *d_lengths, const float *d_weight,
                                       const float *d_bias, const float *d_mean, const float *d_rstd, void *d_grad_x, float *d_grad_weight,
                                       float *d_grad_bias, void *d_grad_residual, int64_t N, int64_t S, int C, int G, int activation, double dropout,
                                       uint64_t seed, uint64_t offset, const int64_t *d_rng, int dtype, void *d_ws, size_t ws_bytes, void *stream_) {
    cudaStream_t stream = (cudaStream_t)stream_;
    if (!sizes_ok(N, S, C, G, dtype, activation))
        PCX_FAIL(PCX_E_ARG, "pcx_ragged_group_norm_act_backward: bad sizes, activation or dtype (C <= %d must be a multiple of G)", NA_MAX_C);
    if (!d_lengths || !d_mean || !d_rstd || !d_ws || (N > 0 && (!d_grad_y || !d_x || !d_grad_x)) || ((d_weight == nullptr) != (d_bias == nullptr)) ||
        ((d_grad_weight == nullptr) != (d_grad_bias == nullptr)))
        PCX_FAIL(PCX_E_ARG, "pcx_ragged_group_norm_act_backward: null pointer (weight and bias come together, and so do their gradients)");
    if ((uintptr_t)d_ws % 256) PCX_FAIL(PCX_E_ALIGN, "pcx_ragged_group_norm_act_backward: workspace must be 256-byte aligned");
    NormAct p = {};
    if (!make_dropping(dropout, seed, offset, d_rng, &p.drop))
        PCX_FAIL(PCX_E_ARG, "pcx_ragged_group_norm_act_backward: dropout %g is no probability", dropout);
    const size_t need = carve(d_ws, N, S, C, G, dtype, &p);
    if (ws_bytes < need) PCX_FAIL(PCX_E_CAPACITY, "pcx_ragged_group_norm_act_backward: workspace %zu < %zu bytes", ws_bytes, need);
    p.x = d_x, p.residual = d_residual, p.g = d_grad_y, p.dx = d_grad_x, p.dresidual = d_grad_residual, p.weight = d_weight, p.bias = d_bias;
    p.mean = const_cast<float *>(d_mean), p.rstd = const_cast<float *>(d_rstd), p.dweight = d_grad_weight, p.dbias = d_grad_bias;
    p.N = N, p.S = S, p.C = C, p.G = G, p.W = C / G, p.by_width = (uint32_t)((0xFFFFFFFFull + p.W) / p.W);
    const int vn = lump_of(C, dtype, {d_x, d_residual, d_grad_y, d_grad_x, d_grad_residual});
    prof_begin("group_norm_act(bwd)", stream);
    if (int rc = sample_offsets(d_lengths, p.offsets, S, N, stream)) return rc;
    if (N > 0)
        if (int rc = run(p, dtype, vn, activation, BWD_SUMS, stream)) return rc;
    launch_after(na_merge_kernel<true>, (unsigned)S, NA_THREADS, 0, stream, p);
    PCX_LAUNCH_CHECK();
    if (d_grad_weight) {
        launch_after(na_affine_kernel, (unsigned)((C + NA_THREADS / 32 - 1) / (NA_THREADS / 32)), NA_THREADS, 0, stream, p);
        PCX_LAUNCH_CHECK();
    }
    if (N > 0)
        if (int rc = run(p, dtype, vn, activation, BWD_APPLY, stream)) return rc;
    prof_end(stream);
    return PCX_OK;
}

}  // extern "C"
