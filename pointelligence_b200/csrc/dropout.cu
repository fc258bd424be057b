// Dropout over a ragged batch with the tail of a residual block, its mask made by counting (philox.cuh) and never stored:
//
//   y = relu?((residual +) keep[u] * x / (1 - p))
//
// A unit u is an element (row-major index), a channel of a sample (s * C + c: feature dropout) or a sample (s: drop path, which
// drops a residual branch whole).  Backward, with g masked where y > 0 does not hold (relu): dresidual = g, dx = keep[u] * g / (1 - p).
// What is dropped is zero whatever it was, and rows of a dropped sample are not read.  Bound by bytes: by element, 730 thousand rows of 96
// channels, bf16, 280 MB in 46 us, 6.1 TB/s (a copy's 6.5), beside which a generator call for every eight elements has room; by
// sample with residual and ReLU, 500 thousand rows of 64 channels, p = 0.3, 173 MB in 32 us forward and 256 MB in 42 us backward.
#include <algorithm>

#include "philox.cuh"
#include "rowwise.cuh"

namespace pcx {
namespace {

constexpr int DO_THREADS = 256;
// Lumps a thread has in flight (by channel or sample).  Four where that fits the registers: 70 million elements of 64 channels, bf16, by
// sample 46 us for 52 with two; backward 86 and 85, rows side by side 65 and 63 (33 channels), so two there, and in 32 bits, which spill.
template <typename T, bool BACKWARD, bool PHASES>
constexpr int DO_UNROLL = sizeof(T) == 2 && !BACKWARD && !PHASES ? 4 : 2;
constexpr int DO_CALLS = 2;                   // of the generator, a thread (by element)
constexpr int DO_CHANNELS = 2048;             // whose words a block keeps, at most
constexpr int DO_CHUNK_BYTES = 32 << 10;      // of rows, a block of the units' kernel (16 KB: 56 us; 64 KB: 44, but 91 for 86 backward)

struct DropArgs {
    const void *x, *residual, *y_in;          // (backward: the gradient, none, the result for the ReLU)
    void *y, *masked;                         // (backward: the input's gradient, the residual's)
    const int64_t *offsets;
    int64_t N, S;
    int C, rows, relu, phase_bits;            // 1 << phase_bits rows side by side (the units' kernel)
    Dropping drop;
};

// `words`: of the lump's units; all ones: kept.
__device__ __forceinline__ bool is_kept(const DropArgs &p, const uint32_t *words, int i) { return (i % 2 ? words[i / 2] : words[i / 2] << 16) > p.drop.over; }

template <typename T, int VN, bool BACKWARD>
__device__ __forceinline__ void drop_lump(const DropArgs &p, int64_t at, const Lump<T, VN> &x, const Lump<T, VN> &other, const uint32_t *words) {
    Lump<T, VN> out;
    if constexpr (BACKWARD) {
        Lump<T, VN> g = x;
        if (p.relu) {
#pragma unroll
            for (int i = 0; i < VN; ++i) g.set(i, other.get(i) > 0.f ? x.get(i) : 0.f);
        }
#pragma unroll
        for (int i = 0; i < VN; ++i) out.set(i, is_kept(p, words, i) ? g.get(i) * p.drop.scale : 0.f);
        if (p.masked) g.store(static_cast<T *>(p.masked) + at);
    } else {
#pragma unroll
        for (int i = 0; i < VN; ++i) {
            float v = is_kept(p, words, i) ? x.get(i) * p.drop.scale : 0.f;
            if (p.residual) v += other.get(i);
            out.set(i, p.relu ? relu(v) : v);
        }
    }
    out.store(static_cast<T *>(p.y) + at);
}

// By element: a thread takes groups of eight consecutive ones, with the words of one call.  PLAIN: nothing but the dropout; WIDE: accesses
// of 16 bytes (addresses are multiples of that).
template <typename T, bool WIDE, bool STATE, bool PLAIN, bool BACKWARD>
__global__ void __launch_bounds__(DO_THREADS, 6) drop_elements_kernel(const __grid_constant__ DropArgs p, int64_t n) {
    start_after_previous();
    const Philox<STATE> rng(p.drop);
    const T *x = static_cast<const T *>(p.x), *other = static_cast<const T *>(BACKWARD ? p.y_in : p.residual);
    const bool reads = !PLAIN && (BACKWARD ? p.relu != 0 : p.residual != nullptr);
    const int64_t call0 = (int64_t)blockIdx.x * (DO_THREADS * DO_CALLS) + threadIdx.x;
    uint32_t words[DO_CALLS][4];
    if (WIDE && ((int64_t)blockIdx.x + 1) * (DO_THREADS * DO_CALLS * 8) <= n) {
        Lump<T, 8> v[DO_CALLS], q[DO_CALLS];
        x += call0 * 8;
        if (reads) other += call0 * 8;
#pragma unroll
        for (int u = 0; u < DO_CALLS; ++u) {
            v[u].load(x + u * DO_THREADS * 8);
            if (reads) q[u].load(other + u * DO_THREADS * 8);
        }
#pragma unroll
        for (int u = 0; u < DO_CALLS; ++u) {   // (while the loads are on their way)
#pragma unroll
            for (int j = 0; j < 4; ++j) words[u][j] = ~0u;
            if (PLAIN || p.drop.on) rng.template words<8>((uint64_t)(call0 + u * DO_THREADS) * 8, words[u]);
        }
#pragma unroll
        for (int u = 0; u < DO_CALLS; ++u) {
            if constexpr (PLAIN) {
                T *y = static_cast<T *>(p.y) + call0 * 8;
                Lump<T, 8> out;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = mul2(pair_of(v[u], j), both(p.drop.scale));
                    set_pair(out, j, make_float2((words[u][j] << 16) > p.drop.over ? f.x : 0.f, words[u][j] > p.drop.over ? f.y : 0.f));
                }
                out.store(y + u * DO_THREADS * 8);
            } else {
                drop_lump<T, 8, BACKWARD>(p, (call0 + u * DO_THREADS) * 8, v[u], q[u], words[u]);
            }
        }
        return;
    }
    for (int u = 0; u < DO_CALLS; ++u) {   // one by one
        const int64_t from = (call0 + u * DO_THREADS) * 8;
        if (from >= n) break;
        words[0][0] = words[0][1] = words[0][2] = words[0][3] = ~0u;
        if (p.drop.on) rng.template words<8>((uint64_t)from, words[0]);
        const int count = (int)min(n - from, (int64_t)8);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= count) break;
            Lump<T, 1> v, q;
            v.load(x + from + i);
            if (reads) q.load(other + from + i);
            const uint32_t word = words[0][i / 2] >> 16 * (i & 1);
            drop_lump<T, 1, BACKWARD>(p, from + i, v, q, &word);
        }
    }
}

// The words of a sample's channels, by the block, 16 bits each.
__device__ __forceinline__ void channel_words(const DropArgs &p, const Philox<true> &rng, int64_t s, uint16_t *to) {
    const int64_t first = s * p.C, call0 = first >> 3;
    for (int k = threadIdx.x; k <= (int)((first + p.C - 1 >> 3) - call0); k += DO_THREADS) {
        uint32_t w[4];
        rng.words<8>((uint64_t)(call0 + k) * 8, w);
        const int c = (int)((call0 + k) * 8 - first);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i >= 0 && c + i < p.C) to[c + i] = (uint16_t)(w[i / 2] >> 16 * (i & 1));
    }
}

// By channels of a sample, or by samples: a block has `rows` consecutive rows, and goes through them sample by sample.  PHASES: rows that
// are no whole number of eight channels are taken 2, 4 or 8 side by side, V channels, counted from the tensor's first, so that accesses
// are of 16 bytes; lumps that a sample's end cuts go one by one.  70 million elements of 33 channels, bf16: by channel 72 us, by sample 63,
// one channel at a time 167 and 169.  (80 thousand rows of 20 channels, where the words' way through shared memory shows: 6.2 us for 4.6.)
template <typename T, int VN, bool BACKWARD, bool SAMPLES, bool PHASES>
__global__ void __launch_bounds__(DO_THREADS, 4) drop_units_kernel(const __grid_constant__ DropArgs p) {
    constexpr int UNROLL = DO_UNROLL<T, BACKWARD, PHASES>;
    start_after_previous();
    const Philox<true> rng(p.drop);
    const T *x = static_cast<const T *>(p.x), *other = static_cast<const T *>(BACKWARD ? p.y_in : p.residual);
    const bool reads = BACKWARD ? p.relu != 0 : p.residual != nullptr;
    const int V = PHASES ? p.C << p.phase_bits : p.C, lumps = V / VN, cols = min(lumps, DO_THREADS), lanes = DO_THREADS / cols, col = threadIdx.x % cols, lane = threadIdx.x / cols;
    const int64_t row0 = (int64_t)blockIdx.x * p.rows, row1 = min(p.N, row0 + p.rows);
    __shared__ uint16_t of_channel[PHASES && !SAMPLES ? DO_CHANNELS : 1];
    if (!(PHASES && !SAMPLES) && lane >= lanes) return;
    for (int64_t s = segment_of_row(p.offsets, p.S, row0); s < p.S && p.offsets[s] < row1; ++s) {
        const int64_t lo = max(row0, p.offsets[s]), hi = min(row1, p.offsets[s + 1]);
        if (hi <= lo) continue;
        const int64_t begin = lo * p.C, end = hi * p.C;
        const int64_t v0 = PHASES ? lo >> p.phase_bits : lo, v1 = PHASES ? (hi + (1 << p.phase_bits) - 1) >> p.phase_bits : hi;
        uint32_t words[(VN + 1) / 2];
#pragma unroll
        for (int j = 0; j < (VN + 1) / 2; ++j) words[j] = ~0u;
        if (SAMPLES && p.drop.on) {
            rng.words<1>((uint64_t)s, words);
            words[0] = (words[0] & 0xffff) * 0x10001;   // the sample's, for all
#pragma unroll
            for (int j = 1; j < (VN + 1) / 2; ++j) words[j] = words[0];
        }
        if (PHASES && !SAMPLES && p.drop.on) {
            __syncthreads();   // (the sample before has been read)
            channel_words(p, rng, s, of_channel);
            __syncthreads();
        }
        for (int lump = lane < lanes ? col : lumps; lump < lumps; lump += cols) {
            const int c0 = lump * VN;
            if (!SAMPLES && p.drop.on) {
                if constexpr (PHASES) {
                    int c = c0 % p.C;
#pragma unroll
                    for (int i = 0; i < VN; ++i) {
                        words[i / 2] = i % 2 ? words[i / 2] | (uint32_t)of_channel[c] << 16 : of_channel[c];
                        if (++c == p.C) c = 0;
                    }
                } else {
                    rng.words<VN>((uint64_t)s * p.C + c0, words);
                }
            }
            bool want = BACKWARD && p.masked;
#pragma unroll
            for (int i = 0; i < VN; ++i) want |= is_kept(p, words, i);
            for (int64_t r = v0 + lane; r < v1; r += (int64_t)UNROLL * lanes) {
                Lump<T, VN> v[UNROLL], q[UNROLL];
                const auto whole = [&](int64_t row) { return PHASES ? row * V + c0 >= begin && row * V + c0 + VN <= end : row < v1; };
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    const int64_t row = r + (int64_t)u * lanes, at = row * V + c0;
#pragma unroll
                    for (int w = 0; w < Lump<T, VN>::WORDS; ++w) v[u].w[w] = 0;
                    if (whole(row)) {
                        if (want) v[u].load(x + at);
                        if (reads) q[u].load(other + at);
                    }
                }
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    const int64_t row = r + (int64_t)u * lanes, at = row * V + c0;
                    if (whole(row)) {
                        drop_lump<T, VN, BACKWARD>(p, at, v[u], q[u], words);
                    } else if (PHASES) {
#pragma unroll
                        for (int i = 0; i < VN; ++i) {
                            if (at + i < begin || at + i >= end) continue;
                            const uint32_t word = words[i / 2] >> 16 * (i & 1);
                            Lump<T, 1> one, two;
                            one.w[0] = 0;
                            if ((word << 16) > p.drop.over || (BACKWARD && p.masked)) one.load(x + at + i);
                            if (reads) two.load(other + at + i);
                            drop_lump<T, 1, BACKWARD>(p, at + i, one, two, &word);
                        }
                    }
                }
            }
        }
    }
}

enum { UNIT_ELEMENT = 0, UNIT_CHANNEL = 1, UNIT_SAMPLE = 2 };

template <typename T, bool WIDE, bool STATE, bool BACKWARD>
int run_elements(const DropArgs &p, int64_t n, cudaStream_t stream) {
    const unsigned grid = (unsigned)((n + 8 * DO_THREADS * DO_CALLS - 1) / (8 * DO_THREADS * DO_CALLS));
    if (!BACKWARD && WIDE && p.drop.on && !p.residual && !p.relu) launch_after(drop_elements_kernel<T, WIDE, STATE, true, BACKWARD>, grid, DO_THREADS, 0, stream, p, n);
    else launch_after(drop_elements_kernel<T, WIDE, STATE, false, BACKWARD>, grid, DO_THREADS, 0, stream, p, n);
    PCX_LAUNCH_CHECK();
    return PCX_OK;
}

template <typename T, int VN, bool BACKWARD, bool PHASES = false>
int run_units(const DropArgs &p, int unit, cudaStream_t stream) {
    const unsigned grid = (unsigned)((p.N + p.rows - 1) / p.rows);
    if (unit == UNIT_SAMPLE) launch_after(drop_units_kernel<T, VN, BACKWARD, true, PHASES>, grid, DO_THREADS, 0, stream, p);
    else launch_after(drop_units_kernel<T, VN, BACKWARD, false, PHASES>, grid, DO_THREADS, 0, stream, p);
    PCX_LAUNCH_CHECK();
    return PCX_OK;
}

template <typename T, bool BACKWARD>
int run(const DropArgs &p, int unit, int vn, cudaStream_t stream) {
    if (unit == UNIT_ELEMENT) {
        const int64_t n = p.N * p.C;
        if (vn < 8) return run_elements<T, false, true, BACKWARD>(p, n, stream);
        return p.drop.state ? run_elements<T, true, true, BACKWARD>(p, n, stream) : run_elements<T, true, false, BACKWARD>(p, n, stream);
    }
    if (p.phase_bits) return run_units<T, 8, BACKWARD, true>(p, unit, stream);
    if (vn == 8) return run_units<T, 8, BACKWARD>(p, unit, stream);
    if (vn == 4) return run_units<T, 4, BACKWARD>(p, unit, stream);
    if (vn == 2) return run_units<T, 2, BACKWARD>(p, unit, stream);
    return run_units<T, 1, BACKWARD>(p, unit, stream);
}

size_t carve(void *ws, int64_t S, int unit, int64_t **offsets) {
    Carver c(ws);
    int64_t *at = c.take<int64_t>(unit == UNIT_ELEMENT ? 0 : (size_t)S + 1);
    if (offsets) *offsets = at;
    return c.off;
}

bool sizes_ok(int64_t N, int64_t S, int C, int unit, int dtype) {
    return N >= 0 && C > 0 && unit >= UNIT_ELEMENT && unit <= UNIT_SAMPLE && (unit == UNIT_ELEMENT || (S > 0 && S <= INT32_MAX)) &&
           (dtype == PCX_F32 || dtype == PCX_F16 || dtype == PCX_BF16) && N <= INT64_MAX / 8 / C && N * C / (8 * DO_THREADS * DO_CALLS) < INT32_MAX;
}

template <bool BACKWARD>
int drop(const char *name, DropArgs p, const int64_t *d_lengths, int unit, double dropout, uint64_t seed, uint64_t offset, const int64_t *d_rng,
         int dtype, void *d_ws, size_t ws_bytes, cudaStream_t stream) {
    if (!sizes_ok(p.N, p.S, p.C, unit, dtype)) PCX_FAIL(PCX_E_ARG, "%s: bad sizes, unit or dtype", name);
    if ((p.N > 0 && (!p.x || !p.y)) || (unit != UNIT_ELEMENT && (!d_lengths || !d_ws)) || (BACKWARD && p.relu && p.N > 0 && !p.y_in))
        PCX_FAIL(PCX_E_ARG, "%s: null pointer", name);
    if (!make_dropping(dropout, seed, offset, d_rng, &p.drop)) PCX_FAIL(PCX_E_ARG, "%s: %g is no probability", name, dropout);
    if (p.N == 0) return PCX_OK;
    const int by_address = lump_of(8, dtype, {p.x, p.residual, p.y_in, p.y, p.masked}), vn = unit == UNIT_ELEMENT ? by_address : lump_of(p.C, dtype, {p.x, p.residual, p.y_in, p.y, p.masked});
    prof_begin(BACKWARD ? "dropout(bwd)" : "dropout(fwd)", stream);
    if (unit != UNIT_ELEMENT) {
        if ((uintptr_t)d_ws % 256) PCX_FAIL(PCX_E_ALIGN, "%s: workspace must be 256-byte aligned", name);
        int64_t *offsets = nullptr;
        const size_t need = carve(d_ws, p.S, unit, &offsets);
        if (ws_bytes < need) PCX_FAIL(PCX_E_CAPACITY, "%s: workspace %zu < %zu bytes", name, ws_bytes, need);
        p.offsets = offsets;
        const int64_t by_bytes = DO_CHUNK_BYTES / ((int64_t)p.C * (int64_t)elem_size(dtype)), by_chip = (p.N + 4 * num_sms() - 1) / (4 * num_sms());
        p.rows = (int)std::max<int64_t>(1, std::min(by_bytes, by_chip));
        if (by_address == 8 && p.C <= DO_CHANNELS) {
            while (((int64_t)p.C << p.phase_bits) % 8) ++p.phase_bits;
            p.rows = ((p.rows - 1) >> p.phase_bits) + 1 << p.phase_bits;
        }
        if (p.N / p.rows >= INT32_MAX) PCX_FAIL(PCX_E_ARG, "%s: bad sizes, unit or dtype", name);
        if (int rc = sample_offsets(d_lengths, offsets, p.S, p.N, stream)) return rc;
    }
    int rc = PCX_OK;
    if (dtype == PCX_F32) rc = run<float, BACKWARD>(p, unit, vn, stream);
    else if (dtype == PCX_F16) rc = run<__half, BACKWARD>(p, unit, vn, stream);
    else rc = run<__nv_bfloat16, BACKWARD>(p, unit, vn, stream);
    prof_end(stream);
    return rc;
}

__global__ void rng_state_kernel(const int64_t *seed, const int64_t *offset, int64_t more, int64_t *out) {
    start_after_previous();
    if (threadIdx.x == 0) out[0] = *seed, out[1] = *offset + more;
}

}  // namespace
}  // namespace pcx

using namespace pcx;

extern "C" {

size_t pcx_dropout_workspace_bytes(int64_t S, int unit) {
    return unit == UNIT_ELEMENT || S <= 0 || S > INT32_MAX ? 0 : carve(nullptr, S, unit, nullptr);
}

int pcx_dropout(const void *d_x, const int64_t *d_lengths, const void *d_residual, void *d_y, int64_t N, int64_t S, int C, int unit, int relu,
                double dropout, uint64_t seed, uint64_t offset, const int64_t *d_rng, int dtype, void *d_ws, size_t ws_bytes, void *stream) {
    DropArgs p = {};
    p.x = d_x, p.residual = d_residual, p.y = d_y, p.N = N, p.S = S, p.C = C, p.relu = relu;
    return drop<false>("pcx_dropout", p, d_lengths, unit, dropout, seed, offset, d_rng, dtype, d_ws, ws_bytes, (cudaStream_t)stream);
}

int pcx_dropout_backward(const void *d_grad_y, const void *d_y, const int64_t *d_lengths, void *d_grad_x, void *d_grad_residual, int64_t N, int64_t S,
                         int C, int unit, int relu, double dropout, uint64_t seed, uint64_t offset, const int64_t *d_rng, int dtype, void *d_ws,
                         size_t ws_bytes, void *stream) {
    DropArgs p = {};
    p.x = d_grad_y, p.y_in = relu ? d_y : nullptr, p.y = d_grad_x, p.masked = d_grad_residual, p.N = N, p.S = S, p.C = C, p.relu = relu;
    return drop<true>("pcx_dropout_backward", p, d_lengths, unit, dropout, seed, offset, d_rng, dtype, d_ws, ws_bytes, (cudaStream_t)stream);
}

int pcx_rng_state(const int64_t *d_seed, const int64_t *d_offset, int64_t more, int64_t *d_rng, void *stream) {
    if (!d_seed || !d_offset || !d_rng) PCX_FAIL(PCX_E_ARG, "pcx_rng_state: null pointer");
    launch_after(rng_state_kernel, 1, 32, 0, (cudaStream_t)stream, d_seed, d_offset, more, d_rng);
    PCX_LAUNCH_CHECK();
    return PCX_OK;
}

}  // extern "C"
