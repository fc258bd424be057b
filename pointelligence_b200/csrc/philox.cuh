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
    bool on = false;                // (not on: words of all ones are kept)
    uint32_t keys[20] = {};         // of the ten rounds
    uint64_t offset = 0;
    const int64_t *state = nullptr; // or on the device: (seed, offset), read when the kernel runs
};

constexpr uint32_t PHILOX_M0 = 0xD2511F53u, PHILOX_M1 = 0xCD9E8D57u, PHILOX_W0 = 0x9E3779B9u, PHILOX_W1 = 0xBB67AE85u;

// `p` in [0, 1]; false for anything else.
inline bool make_dropping(double p, uint64_t seed, uint64_t offset, const int64_t *state, Dropping *out) {
    if (!(p >= 0.0 && p <= 1.0)) return false;
    const uint32_t t = (uint32_t)(65536.0 * p + 0.5);
    out->on = t > 0;
    out->over = t ? t * 65536u - 1u : 0;    // (t = 65536: nothing is over 2^32 - 1)
    out->scale = t < 65536u ? (float)(65536.0 / (double)(65536u - t)) : 0.f;
    for (uint32_t r = 0; r < 10; ++r) out->keys[2 * r] = (uint32_t)seed + r * PHILOX_W0, out->keys[2 * r + 1] = (uint32_t)(seed >> 32) + r * PHILOX_W1;
    out->offset = offset, out->state = state;
    return true;
}

// STATE: the seed may be on the device.  Otherwise the rounds' keys are arguments of the kernel, which its instructions read as they
// are: 40 products, which run at half rate, and 20 other operations a call, where keys that are made in the kernel cost 20 more.
template <bool STATE>
struct Philox {
    const uint32_t *keys;
    uint32_t k0 = 0, k1 = 0, c2, c3;
    __device__ __forceinline__ explicit Philox(const Dropping &d) : keys(d.keys) {
        uint64_t offset = d.offset;
        if constexpr (STATE) {
            k0 = d.keys[0], k1 = d.keys[1];
            if (d.on && d.state) {
                const uint64_t seed = (uint64_t)d.state[0];
                k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32), offset = (uint64_t)d.state[1];
            }
        }
        c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    }
    __device__ __forceinline__ uint4 call(uint64_t block) const {
        uint32_t a = (uint32_t)block, b = (uint32_t)(block >> 32), c = c2, d = c3;
#pragma unroll
        for (int r = 0; r < 10; ++r) {
            const uint64_t p = (uint64_t)a * PHILOX_M0, q = (uint64_t)c * PHILOX_M1;
            const uint32_t x0 = STATE ? k0 + r * PHILOX_W0 : keys[2 * r], x1 = STATE ? k1 + r * PHILOX_W1 : keys[2 * r + 1];
            a = (uint32_t)(q >> 32) ^ b ^ x0, b = (uint32_t)q;
            c = (uint32_t)(p >> 32) ^ d ^ x1, d = (uint32_t)p;
        }
        return make_uint4(a, b, c, d);
    }
    // The words of units u .. u + VN - 1, two in each of (VN + 1) / 2, low halves first; u is a multiple of VN, which divides 8.
    // Kept: (word << 16) > over, for a high half word > over.
    template <int VN>
    __device__ __forceinline__ void words(uint64_t u, uint32_t *out) const {
        const uint4 w = call(u >> 3);
        if constexpr (VN == 8) {
            out[0] = w.x, out[1] = w.y, out[2] = w.z, out[3] = w.w;
        } else if constexpr (VN == 4) {
            out[0] = u & 4 ? w.z : w.x, out[1] = u & 4 ? w.w : w.y;
        } else {
            out[0] = u & 4 ? (u & 2 ? w.w : w.z) : (u & 2 ? w.y : w.x);
            if (VN == 1 && (u & 1)) out[0] >>= 16;
        }
    }
};

}  // namespace pcx
