// Random words of the dropout kernels: Philox4x32-10, the counter-based generator of Salmon, Moraes, Dror and Shaw
// ("Parallel random numbers: as easy as 1, 2, 3", 2011), written from the paper's definition.
//
// What is dropped is decided by units (elements, channels of a sample, samples).  Unit u has word u % 8, of 16 bits, of the call with
// the counter (u / 8, offset) and the key seed; it is kept where the word is at least round(65536 p), and scaled by the inverse
// of the share that is kept.  A mask is a function of (seed, offset): it is never stored, and the backward pass makes it again.
// 16 bits a word, not 32: a call is about 60 integer operations, and with eight words of it a unit costs 8 of them, with
// four 15, which is more than the memory takes to bring an element of 16 bits (integer products run at half rate).  The
// probability is then a multiple of 2^-16, and the scale goes by the one that is used, so that the mean is kept exactly.
#pragma once
#include "common.cuh"

namespace pcx {

struct Dropping {
    uint32_t over = 0;              // kept: a word in the upper half of 32 bits that is over this
    float scale = 1.f;              // of what is kept
    bool on = false;
    uint64_t seed = 0, offset = 0;
    const int64_t *state = nullptr; // or on the device: (seed, offset), read when the kernel runs
};

// `p` in [0, 1]; false for anything else.
inline bool make_dropping(double p, uint64_t seed, uint64_t offset, const int64_t *state, Dropping *out) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    const uint32_t t = (uint32_t)(65536.0 * p + 0.5);
    out->on = t > 0;
    out->over = t * 65536u - 1u;    // (t = 65536: nothing is over 2^32 - 1)
    out->scale = t < 65536u ? (float)(65536.0 / (double)(65536u - t)) : 0.f;
    out->seed = seed, out->offset = offset, out->state = state;
    return true;
}

struct Philox {
    uint32_t k0, k1, c2, c3;
    __device__ __forceinline__ explicit Philox(const Dropping &d) {
        uint64_t seed = d.seed, offset = d.offset;
        if (d.on && d.state) seed = (uint64_t)d.state[0], offset = (uint64_t)d.state[1];
        k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    }
    __device__ __forceinline__ uint4 call(uint64_t block) const {
        uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32), c = c2, d = c3;
#pragma unroll
        for (int r = 0; r < 10; ++r) {
            const uint64_t p = (uint64_t)a * 0xD2511F53u, q = (uint64_t)c * 0xCD9E8D57u;
            const uint32_t x0 = k0 + r * 0x9E3779B9u, x1 = k1 + r * 0xBB67AE85u;
            a = (uint32_t)(q >> 32) ^ b ^ x0, b = (uint32_t)q;
            c = (uint32_t)(p >> 32) ^ d ^ x1, d = (uint32_t)p;
        }
        return make_uint4(a, b, c, d);
    }
    // The kept ones of units u .. u + VN - 1 as bits; u is a multiple of VN, which divides 8.
    template <int VN>
    __device__ __forceinline__ uint32_t kept(uint64_t u, uint32_t over) const {
        const uint4 w = call(u >> 3);
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
        uint32_t bits = 0;
        if constexpr (VN == 8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) bits |= (uint32_t)((words[i] << 16) > over) << (2 * i) | (uint32_t)(words[i] > over) << (2 * i + 1);
        } else if constexpr (VN == 4) {
            const bool upper = u & 4;
            const uint32_t lo = upper ? w.z : w.x, hi = upper ? w.w : w.y;
            bits = (uint32_t)((lo << 16) > over) | (uint32_t)(lo > over) << 1 | (uint32_t)((hi << 16) > over) << 2 | (uint32_t)(hi > over) << 3;
        } else {
            const uint32_t pair = u & 4 ? (u & 2 ? w.w : w.z) : (u & 2 ? w.y : w.x);
            if constexpr (VN == 2) bits = (uint32_t)((pair << 16) > over) | (uint32_t)(pair > over) << 1;
            else bits = (u & 1 ? pair : pair << 16) > over;
        }
        return bits;
    }
};

}  // namespace pcx
