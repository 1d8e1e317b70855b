// Shared by the kernels over the paged 8-bit key/value cache: where a call's
// integers (table entries, slots, starts, lengths, all of them device memory
// that the host never sees) may lead, and the codes as matrix operands.
#pragma once

#include "kf_common.h"

namespace kf {
namespace {

// ---------------------------------------------------------------------------
// Bounds.  Every address the kernels form from device integers goes through
// these; they compile for the host too, where the tests call them.
// ---------------------------------------------------------------------------
constexpr int kMaxContext = INT32_MAX - 255;  // positions and tiles stay in 32 bits

// log2 of a block size, or -1 where it is not one.
inline int block_shift(int64_t block_tokens) {
    for (int s = 4; s <= 7; ++s)
        if (block_tokens == (int64_t)1 << s) return s;
    return -1;
}

// The block a slot lies in, or -1 for a slot outside the cache.
__host__ __device__ __forceinline__ int64_t block_of_slot(int64_t slot, int64_t capacity, int shift) {
    return slot >= 0 && slot < capacity ? slot >> shift : -1;
}

// The block of a request's 16-token group, or -1 where its table (width
// entries, at least one) names none of the cache's: first what the table holds,
// then, when that has arrived, whether it is a block.
__host__ __device__ __forceinline__ int entry_of_group(const int* table, int width, int shift, int group) {
    const int entry = group >> (shift - 4);
    return table[entry < width ? entry : width - 1];
}
__host__ __device__ __forceinline__ int block_of_entry(int id, int width, int blocks, int shift, int group) {
    return group >> (shift - 4) < width && id >= 0 && id < blocks ? id : -1;
}

// One request's place in a call of `tokens` tokens.
struct Request {
    int q0, n;  // first token and number of queries, inside the call
    int ctx;    // cached tokens
};

__host__ __device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

__host__ __device__ __forceinline__ Request request_at(const int* starts, const int* context, int b, int tokens) {
    Request r;
    r.q0 = starts ? clamp_int(starts[b], 0, tokens) : b;
    r.n = starts ? clamp_int(starts[b + 1], r.q0, tokens) - r.q0 : 1;
    r.ctx = clamp_int(context[b], 0, kMaxContext);
    return r;
}

// Keys that query i of a request sees.
__host__ __device__ __forceinline__ int keys_seen(const Request& r, int i, bool causal) {
    const int seen = causal ? r.ctx - r.n + i + 1 : r.ctx;
    return seen > 0 ? seen : 0;
}

// ---------------------------------------------------------------------------
// Codes as operands of the 16-bit matrix products.  Every e4m3 and int8 value
// is exact in bf16 and in f16.
// ---------------------------------------------------------------------------

template <typename T, int CT> struct Codes;

template <typename T> __device__ __forceinline__ typename V<T>::x8 join4(u32x4 r) {
    return __builtin_bit_cast(typename V<T>::x8, r);
}

// e4m3: two codes an instruction (v_cvt_scalef32_pk_*_fp8, scale 1).
template <> struct Codes<bf16, KF_CACHE_E4M3> {
    static __device__ __forceinline__ V<bf16>::x8 x8(uint32_t lo, uint32_t hi) {
        u32x4 r;
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
        return join4<bf16>(r);
    }
};
template <> struct Codes<f16, KF_CACHE_E4M3> {
    static __device__ __forceinline__ V<f16>::x8 x8(uint32_t lo, uint32_t hi) {
        u32x4 r;
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
        return join4<f16>(r);
    }
};

// int8 to f16: code + 128 in the low byte of 0x64xx is 1024 + 128 + code in
// f16; subtracting 1152 is exact.  One permute and one packed add a pair.
template <> struct Codes<f16, KF_CACHE_INT8> {
    static __device__ __forceinline__ uint32_t pair(uint32_t biased, uint32_t select) {
        typedef f16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 x = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, biased, select));
        return __builtin_bit_cast(uint32_t, (f16x2)(x - (f16x2){(f16)1152.0f, (f16)1152.0f}));
    }
    static __device__ __forceinline__ V<f16>::x8 x8(uint32_t lo, uint32_t hi) {
        const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
        u32x4 r = {pair(a, 0x04010400u), pair(a, 0x04030402u), pair(b, 0x04010400u), pair(b, 0x04030402u)};
        return join4<f16>(r);
    }
};
// int8 to bf16 goes through fp32: bf16's 8 bits of significand hold no bias.
template <> struct Codes<bf16, KF_CACHE_INT8> {
    static __device__ __forceinline__ V<bf16>::x8 x8(uint32_t lo, uint32_t hi) {
        V<bf16>::x8 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r[i] = (bf16)(float)(int8_t)(lo >> (8 * i));
            r[4 + i] = (bf16)(float)(int8_t)(hi >> (8 * i));
        }
        return r;
    }
};

}  // namespace
}  // namespace kf
