// Entry points of the group norm with activation and dropout (norm_act.cuh): arguments, workspace, and the launch that lays the
// samples out.
#include <cmath>

#include "norm_act.cuh"

namespace pcx {
int device_status_address(unsigned int **d_status);

extern template int norm_act_rows<float>(const NormAct &, int, bool, cudaStream_t);
extern template int norm_act_rows<__half>(const NormAct &, int, bool, cudaStream_t);
extern template int norm_act_rows<__nv_bfloat16>(const NormAct &, int, bool, cudaStream_t);

namespace {

constexpr int NA_CHUNK_BYTES = 96 << 10;        // of x
constexpr int NA_STAGE_BYTES = 24 << 10;        // of a tile, all tensors
constexpr int NA_RING_BYTES = 110 << 10;        // of shared memory, a block: two on a multiprocessor
constexpr int NA_MAX_C = 1 << 16;
constexpr int NA_RECORDS = 8 << 10;             // of groups that a block reads for itself without windows: 128 KB where all rows are one sample's
constexpr int64_t NA_LAG_BYTES = 64 << 20;      // of x, and of the gradient

// ------------------------------------------------------------ the samples' rows ----
// Row offsets of the samples.  Whatever the lengths say, they ascend within 0 .. N, and rows behind the last sample are its own.
constexpr int OFFSETS_THREADS = 1024;
__device__ __forceinline__ void scan_lengths(const int64_t *__restrict__ lengths, int64_t *offsets, int64_t S, int64_t N) {
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
    __syncthreads();
}

__global__ void __launch_bounds__(OFFSETS_THREADS) na_offsets_kernel(const int64_t *__restrict__ lengths, int64_t *offsets, int64_t S, int64_t N) {
    start_after_previous();
    scan_lengths(lengths, offsets, S, N);
}

// Offsets, spans, cleared counters, and what there is to say of samples without rows.
template <bool BACKWARD>
__global__ void __launch_bounds__(OFFSETS_THREADS) na_layout_kernel(const int64_t *__restrict__ lengths, const __grid_constant__ NormAct p) {
    start_after_previous();
    const int64_t words = CONTROL_WORDS + p.S + (p.window > 1 ? windows_in_all(p.chunks, p.S, p.window) : 0);
    for (int64_t t = threadIdx.x; t < words; t += blockDim.x) p.control[t] = 0;
    scan_lengths(lengths, p.offsets, p.S, p.N);
    int windows = 0;
    for (int64_t s = threadIdx.x; s < p.S; s += blockDim.x) {
        const int64_t lo = p.offsets[s], hi = p.offsets[s + 1];
        Span v;
        v.b0 = (int)(lo / p.rows);
        v.b1 = hi > lo ? (int)((hi - 1) / p.rows) : v.b0 - 1;
        v.first = lo == p.N ? p.chunks : v.b0;
        v.next = hi == p.N ? p.chunks : (int)(hi / p.rows);
        const int last = hi > 0 ? (int)((hi - 1) / p.rows) : -1;
        v.at = v.first + min(p.chunks - 1, last + p.lag) + 1;
        p.spans[s] = v;
        if (hi > lo) windows += windows_of(p, v);
        if (!BACKWARD && hi == lo)
            for (int g = 0; g < p.G; ++g) p.mean[s * p.G + g] = 0.0, p.rstd[s * p.G + g] = 1.0 / sqrt(p.eps);
        if (BACKWARD && p.dweight && (hi == lo || hi % p.rows == 0))   // behind a sample that ends with a chunk, and for one without rows, a number is left out
            for (int c = 0; c < p.C; ++c) p.rec[(hi / p.rows + s) * p.C + c] = make_float2(0.f, 0.f);
    }
    if (windows) atomicAdd(p.control + WINDOWS, windows);   // (cleared before the barriers of scan_lengths)
}

// ------------------------------------------------------------ host ----
// Rows that are side by side in one of the ring's, as a power of two: as many as make whole lumps of eight channels, if that is no
// row too long for it.
int phase_bits_of(int C) {
    int bits = 0;
    while (((int64_t)C << bits) % 8) ++bits;
    return ((int64_t)C << bits) <= RING_CHANNELS ? bits : 0;
}

// Rows of a chunk: 96 KB of them at most, and as many as give every block of the chip the same number of chunks, in whole rows of lanes.
// (With two for a block wherever they were small, some blocks had two and some one: 20 thousand rows of 50 channels, fp32, 34 us
// forward and 36 backward for 24 and 26, 5000 of 256, fp16, with dropout 28 and 36 for 23 and 31; with one, whatever 96 KB allow, 200
// thousand of 96, bf16, 45 for 40.)
int chunk_rows(int64_t N, int C, int dtype) {
    const int bits = phase_bits_of(C);
    int vn = 8;
    while ((C << bits) % vn) vn /= 2;
    const int lanes = Columns(C << bits, vn, 0).lanes << bits;
    const int64_t most = std::max<int64_t>(1, NA_CHUNK_BYTES / ((int64_t)C * (int64_t)elem_size(dtype))), blocks = RING_BLOCKS * num_sms();
    const int64_t rounds = std::max<int64_t>(1, (N + most * blocks - 1) / (most * blocks)), rows = (N + rounds * blocks - 1) / (rounds * blocks);
    return (int)((std::max<int64_t>(rows, 1) + lanes - 1) / lanes) * lanes;
}

// Pieces of a window: as many as leave a block NA_RECORDS records to read for itself, but not so many that the warp that merges a
// window takes longer than all blocks with theirs: that time grows with the window, the blocks' with the number of windows, and at 1458
// pieces they are alike at eight (one sample of 273 thousand rows, 256 instance norms, bf16, forward: windows of 4, 8, 16 and 46 (as
// NA_RECORDS alone has it) pieces 178, 161, 178 and 247 us).
int window_of(int chunks, int G) {
    const int64_t by_records = (chunks * (int64_t)G + NA_RECORDS - 1) / NA_RECORDS;
    const int64_t by_turns = std::max<int64_t>(8, (int64_t)std::sqrt(chunks / 24.0));
    return (int)std::max<int64_t>(1, std::min(by_records, by_turns));
}

size_t carve(void *ws, int64_t N, int64_t S, int C, int G, int dtype, NormAct *out) {
    Carver c(ws);
    NormAct p = out ? *out : NormAct{};
    p.rows = chunk_rows(N, C, dtype);
    p.chunks = (int)((N + p.rows - 1) / p.rows);
    p.offsets = c.take<int64_t>((size_t)S + 1);
    p.spans = c.take<Span>((size_t)S);
    p.rec = c.take<float2>(std::max((size_t)(p.chunks + S) * C, (size_t)std::min<int64_t>(2 * (int64_t)p.chunks, NA_BLOCKS * num_sms()) * C * 2));
    p.scratch = reinterpret_cast<double2 *>(p.rec);   // (forward; the other is backward)
    p.window = window_of(p.chunks, G);
    const size_t windows = p.window > 1 ? (size_t)windows_in_all(p.chunks, S, p.window) : 0;
    p.of_piece = c.take<double2>((size_t)(p.chunks + S) * G);   // (backward: of float2)
    p.of_window = windows ? c.take<double2>(windows * G) : p.of_piece;
    p.control = c.take<int>(CONTROL_WORDS + (size_t)S + windows);
    if (out) *out = p;
    return c.off;
}

bool too_many_samples(int64_t S, int C) { return S > 0 && C > 0 && S > INT32_MAX / C; }   // (counts of samples and windows are 32 bits, and no larger batch is tested)

bool sizes_ok(int64_t N, int64_t S, int C, int G, int dtype, int activation) {
    return N >= 0 && S > 0 && C > 0 && C <= NA_MAX_C && G > 0 && C % G == 0 && !too_many_samples(S, C) &&
           (dtype == PCX_F32 || dtype == PCX_F16 || dtype == PCX_BF16) && activation >= ACT_NONE && activation <= ACT_GELU &&
           (N == 0 || N <= INT64_MAX / 8 / C) && N / chunk_rows(std::max<int64_t>(N, 1), C, dtype) < INT32_MAX / 4;
}

// Both launches of a direction.
template <bool BACKWARD>
int run(const int64_t *d_lengths, NormAct &p, int dtype, int activation, std::initializer_list<const void *> tensors_at, cudaStream_t stream) {
    const int vn = lump_of(p.C, dtype, tensors_at);
    p.act = activation;
    if (int rc = device_status_address(&p.status)) return rc;
    const int64_t lag = NA_LAG_BYTES / ((int64_t)p.rows * p.C * (int64_t)elem_size(dtype) * (BACKWARD ? 2 : 1));
    p.lag = (int)std::max<int64_t>(1, std::min<int64_t>(lag, p.chunks));
    p.stages = 0, p.phase_bits = phase_bits_of(p.C), p.V = p.C << p.phase_bits;
    if (lump_of(p.V, dtype, tensors_at) == 8 && p.V <= RING_CHANNELS) {   // the ring
        const int lanes = Columns(p.V, 8, 0).lanes, tensors = (BACKWARD ? 2 : 1) + (p.residual ? 1 : 0), row_bytes = p.V * (int)elem_size(dtype);
        const int room = NA_RING_BYTES - (int)ring_bytes(p.V, p.G, BACKWARD);
        // (Where two tiles of 24 KB do not fit, smaller ones: 1024 channels, bf16, backward 295 us of 70 million elements, 485 by the general
        // kernel; where they do, three of two thirds are no better: 512 channels with a residual 248 and 250.)
        const int stage = room >= 2 * NA_STAGE_BYTES ? NA_STAGE_BYTES : room / 3;
        p.tile_rows = lanes * std::max(1, stage / (lanes * row_bytes * tensors));   // (at most 12 of a thread: lanes are more than half of the threads)
        p.sums_tile_rows = BACKWARD ? p.tile_rows : p.tile_rows * tensors;
        p.stage_bytes = (p.tile_rows * row_bytes * tensors + 127) / 128 * 128;
        p.stages = std::min(RING_STAGES, room / p.stage_bytes);
        if (p.stages < 2) p.stages = 0;
    }
    if (!p.stages) p.phase_bits = 0;
    launch_after(na_layout_kernel<BACKWARD>, 1, p.S <= 256 ? 256 : OFFSETS_THREADS, 0, stream, d_lengths, p);
    PCX_LAUNCH_CHECK();
    if (p.N == 0) {
        if (BACKWARD && p.dweight) {
            PCX_CUDA(cudaMemsetAsync(p.dweight, 0, (size_t)p.C * sizeof(float), stream));
            PCX_CUDA(cudaMemsetAsync(p.dbias, 0, (size_t)p.C * sizeof(float), stream));
        }
        return PCX_OK;
    }
    if (dtype == PCX_F32) return norm_act_rows<float>(p, vn, BACKWARD, stream);
    if (dtype == PCX_F16) return norm_act_rows<__half>(p, vn, BACKWARD, stream);
    return norm_act_rows<__nv_bfloat16>(p, vn, BACKWARD, stream);
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
                              double *d_mean, double *d_rstd, int64_t N, int64_t S, int C, int G, double eps, int activation, double dropout, uint64_t seed,
                              uint64_t offset, const int64_t *d_rng, int dtype, void *d_ws, size_t ws_bytes, void *stream_) {
    cudaStream_t stream = (cudaStream_t)stream_;
    if (too_many_samples(S, C)) PCX_FAIL(PCX_E_ARG, "pcx_ragged_group_norm_act: %lld samples of %d channels: S * C has to be below 2^31", (long long)S, C);
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
    p.N = N, p.S = S, p.C = C, p.G = G, p.W = C / G, p.by_width = (uint32_t)((0xFFFFFFFFull + p.W) / p.W), p.eps = eps;
    prof_begin("group_norm_act(fwd)", stream);
    const int rc = run<false>(d_lengths, p, dtype, activation, {d_x, d_residual, d_y}, stream);
    prof_end(stream);
    return rc;
}

int pcx_ragged_group_norm_act_backward(const void *d_grad_y, const void *d_x, const void *d_residual, const int64_t *d_lengths, const float *d_weight,
                                       const float *d_bias, const double *d_mean, const double *d_rstd, void *d_grad_x, float *d_grad_weight,
                                       float *d_grad_bias, void *d_grad_residual, int64_t N, int64_t S, int C, int G, int activation, double dropout,
                                       uint64_t seed, uint64_t offset, const int64_t *d_rng, int dtype, void *d_ws, size_t ws_bytes, void *stream_) {
    cudaStream_t stream = (cudaStream_t)stream_;
    if (too_many_samples(S, C)) PCX_FAIL(PCX_E_ARG, "pcx_ragged_group_norm_act_backward: %lld samples of %d channels: S * C has to be below 2^31", (long long)S, C);
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
    p.mean = const_cast<double *>(d_mean), p.rstd = const_cast<double *>(d_rstd), p.dweight = d_grad_weight, p.dbias = d_grad_bias;
    p.N = N, p.S = S, p.C = C, p.G = G, p.W = C / G, p.by_width = (uint32_t)((0xFFFFFFFFull + p.W) / p.W);
    prof_begin("group_norm_act(bwd)", stream);
    const int rc = run<true>(d_lengths, p, dtype, activation, {d_x, d_residual, d_grad_y, d_grad_x, d_grad_residual}, stream);
    prof_end(stream);
    return rc;
}

}  // extern "C"
