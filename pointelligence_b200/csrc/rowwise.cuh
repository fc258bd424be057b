// Row-wise access helpers of the byte-bound kernels (norms, segment reductions):
// 16-byte vector loads / stores of VN consecutive channels converted to fp32, and
// the thread layout (vector column, row lane) they share.
#pragma once
#include <initializer_list>
#include <type_traits>

#include "common.cuh"

namespace pcx {

template <typename T>
struct VecWidth { static constexpr int value = 16 / sizeof(T); };

// VN == 1: scalar access (any channel count, any alignment); VN == 16 / sizeof(T): one 16-byte access
template <typename T, int VN>
__device__ __forceinline__ void load_vec(const T *__restrict__ p, float *out) {
    if constexpr (VN == 1) {
        out[0] = to_f32<T>(p[0]);
    } else {
        const uint4 raw = *reinterpret_cast<const uint4 *>(p);
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < VN; ++i) out[i] = to_f32<T>(e[i]);
    }
}

template <typename T, int VN>
__device__ __forceinline__ void store_vec(T *__restrict__ p, const float *in) {
    if constexpr (VN == 1) {
        p[0] = from_f32<T>(in[0]);
    } else {
        uint4 raw;
        T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int i = 0; i < VN; ++i) e[i] = from_f32<T>(in[i]);
        *reinterpret_cast<uint4 *>(p) = raw;
    }
}

// Thread layout over a block of rows: `vcb` vector columns side by side, blockDim / vcb
// row lanes; a thread keeps its vector column for the whole pass.
struct RowLayout {
    int vc_total;   // vector columns of a row (C / VN)
    int vcb;        // vector columns handled per pass (<= blockDim)
    int lanes;      // row lanes
    int vc, lane;   // this thread's column inside a pass and its row lane (lane >= lanes: idle)
    __device__ __forceinline__ RowLayout(int C, int VN) {
        vc_total = C / VN;
        vcb = vc_total < (int)blockDim.x ? vc_total : (int)blockDim.x;
        lanes = blockDim.x / vcb;
        vc = threadIdx.x % vcb;
        lane = threadIdx.x / vcb;
    }
};

// first segment s with offsets[s + 1] > row (offsets has S + 1 entries)
__device__ __forceinline__ int64_t segment_of_row(const int64_t *__restrict__ offsets, int64_t S, int64_t row) {
    int64_t lo = 0, hi = S;
    while (lo < hi) {
        int64_t mid = (lo + hi) >> 1;
        if (offsets[mid + 1] <= row) lo = mid + 1; else hi = mid;
    }
    return lo;
}

static inline bool vec_ok(int C, int dtype, std::initializer_list<const void *> ptrs) {
    const int vn = 16 / (int)elem_size(dtype);
    if (C % vn) return false;
    for (const void *p : ptrs)
        if (p && ((uintptr_t)p & 15)) return false;
    return true;
}

// VN consecutive channels as they lie in memory: accesses of at most 16 bytes.
template <typename T, int VN>
struct Lump {
    static constexpr int BYTES = VN * (int)sizeof(T);
    static constexpr int WORDS = (BYTES + 3) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void load(const T *__restrict__ p) {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int q = 0; q < BYTES / 16; ++q) {
                const uint4 v = reinterpret_cast<const uint4 *>(p)[q];
                w[4 * q] = v.x, w[4 * q + 1] = v.y, w[4 * q + 2] = v.z, w[4 * q + 3] = v.w;
            }
        } else if constexpr (BYTES == 8) {
            const uint2 v = *reinterpret_cast<const uint2 *>(p);
            w[0] = v.x, w[1] = v.y;
        } else if constexpr (BYTES == 4) {
            w[0] = *reinterpret_cast<const uint32_t *>(p);
        } else {
            w[0] = *reinterpret_cast<const uint16_t *>(p);
        }
    }
    __device__ __forceinline__ void store(T *__restrict__ p) const {
        if constexpr (BYTES >= 16) {
#pragma unroll
            for (int q = 0; q < BYTES / 16; ++q) reinterpret_cast<uint4 *>(p)[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
        } else if constexpr (BYTES == 8) {
            *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
        } else if constexpr (BYTES == 4) {
            *reinterpret_cast<uint32_t *>(p) = w[0];
        } else {
            *reinterpret_cast<uint16_t *>(p) = (uint16_t)w[0];
        }
    }
    // What is not read again soon goes from the L2 first.
    __device__ __forceinline__ void store_streaming(T *__restrict__ p) const {
        static_assert(BYTES >= 16, "whole accesses");
#pragma unroll
        for (int q = 0; q < BYTES / 16; ++q) __stcs(reinterpret_cast<uint4 *>(p) + q, make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]));
    }
    // The elements first <= i < end.
    __device__ __forceinline__ void store_part(T *__restrict__ p, int first, int end) const {
#pragma unroll
        for (int i = 0; i < VN; ++i)
            if (i >= first && i < end) p[i] = reinterpret_cast<const T *>(w)[i];
    }
    // The largest magnitude of the elements 4 h .. 4 h + 3 of eight.
    __device__ __forceinline__ float largest_of_half(int h) const {
        static_assert(VN == 8, "a whole lump");
        if constexpr (sizeof(T) == 4) {   // (NaN aside)
            const float a = fmaxf(fabsf(__uint_as_float(w[4 * h])), fabsf(__uint_as_float(w[4 * h + 1]))), b = fmaxf(fabsf(__uint_as_float(w[4 * h + 2])), fabsf(__uint_as_float(w[4 * h + 3])));
            return fmaxf(a, b);
        } else {   // by pairs (of values without a sign the order is that of whole numbers; a NaN is above them all)
            const uint32_t m = __vmaxu2(w[2 * h] & 0x7fff7fffu, w[2 * h + 1] & 0x7fff7fffu);
            const uint16_t v = (uint16_t)max(m & 0xffffu, m >> 16);
            return to_f32<T>(reinterpret_cast<const T &>(v));
        }
    }
    __device__ __forceinline__ float get(int i) const { return to_f32<T>(reinterpret_cast<const T *>(w)[i]); }
    __device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T *>(w)[i] = from_f32<T>(v); }
};

// Channels are worked on in pairs: sm_100 has fp32 instructions for two at once.  (A lump of one channel is a pair with nothing behind.)
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)), "l"(*reinterpret_cast<uint64_t *>(&c)));
    return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t *>(&a)), "l"(*reinterpret_cast<uint64_t *>(&b)));
    return *reinterpret_cast<float2 *>(&d);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 neg2(float2 v) { return make_float2(-v.x, -v.y); }

template <typename T>
__device__ __forceinline__ float2 unpack(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
template <>
__device__ __forceinline__ float2 unpack<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<__half2 *>(&w)); }

template <typename T, int VN>
__device__ __forceinline__ float2 pair_of(const Lump<T, VN> &v, int j) {
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(v.w[2 * j]), VN > 1 ? __uint_as_float(v.w[2 * j + (VN > 1)]) : 0.f);
    else return unpack<T>(v.w[j]);
}
template <typename T, int VN>
__device__ __forceinline__ void set_pair(Lump<T, VN> &v, int j, float2 f) {
    if constexpr (sizeof(T) == 4) {
        v.w[2 * j] = __float_as_uint(f.x);
        if (VN > 1) v.w[2 * j + (VN > 1)] = __float_as_uint(f.y);
    } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(f.x, f.y);
        v.w[j] = *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
        v.w[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
}

// max(v, 0) that hands a NaN on
__device__ __forceinline__ float relu(float v) {
    float out;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(out) : "f"(v));
    return out;
}

// Channels of a lump: the most that divide a row and that the pointers are aligned for.
static inline int lump_of(int C, int dtype, std::initializer_list<const void *> pointers) {
    int vn = 8;
    for (; vn > 1; vn /= 2) {
        const uintptr_t align = vn * elem_size(dtype) < 16 ? vn * elem_size(dtype) : 16;
        bool ok = C % vn == 0;
        for (const void *q : pointers) ok = ok && (uintptr_t)q % align == 0;
        if (ok) break;
    }
    return vn;
}

// Row offsets (S + 1) of a batch from its lengths: they ascend within 0 .. N whatever the lengths say, and rows behind the last
// sample are its own.  (norm_act.cu)
int sample_offsets(const int64_t *d_lengths, int64_t *offsets, int64_t S, int64_t N, cudaStream_t stream);

}  // namespace pcx
