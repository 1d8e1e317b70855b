// Attention over the paged 8-bit key/value cache: what its two kernels share.
// (Layout of the cache: paged_cache.hip.)
//
// With P the probabilities of a row and S its scores,
//   S_j = scale ks_j <q, kcode_j>,  O = sum_j exp(S_j - max) vs_j vcode_j / sum_j exp(S_j - max),
// ks and vs the scales of key j's block.  Codes enter the matrix products as
// 16-bit floats without rounding; a block's key scale multiplies the fp32
// score and its value scale the fp32 probability.
//
// P is rounded once, to f16 whatever q's type, as p * vs / vref * 2^k with vref
// the largest value scale seen so far and 2^k what keeps the product at most
// 2^15: f16 rounds by at most 2^-11 where bf16 would by 2^-8, and terms stay
// normal numbers down to 2^-29 (2^k = 2^15) or 2^-26 (2^12) of the largest.
// Maxima, sums and accumulators are fp32.
#pragma once

#include "fa_common.h"
#include "paged_common.h"

namespace kf {

// Named (not in an unnamed namespace): the kernels' launchers pass it between files.
struct PagedParams {
    const void* q;
    const uint8_t* kc;
    const uint8_t* vc;
    const float* ks;
    const float* vs;
    const int* tables;
    const int* context;
    const int* starts;  // null: one query a request
    void* out;
    float* lse;
    int64_t q_ts, q_hs;
    int tokens, B, blocks, width, Hq, Hkv, G, D, shift;
    int max_q;
    float c;  // scale * log2(e)
    int few;  // rows (queries x heads of a group) of the requests that the few-rows kernel takes
    bool causal;
    int clear_rest;  // rows behind the last request: 1 out, 2 lse
};

// A partial result's place.
struct Partials {
    float* o;    // [parts][rows][D]
    float2* ml;  // [parts][rows]: running maximum (log2 units) and sum
};

// The prompts' kernel (paged_prompt.hip): requests of more than p.few rows.
struct PromptPlan {
    int64_t units;  // workgroups before splitting
    int splits;
    int64_t bytes;
};
int64_t prompt_units(int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv);
PromptPlan prompt_plan(int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_ctx);
int launch_prompt(const PagedParams& p, const PromptPlan& w, void* workspace, int dtype, int cache_dtype,
                  hipStream_t stream);

namespace {

constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126

__device__ __forceinline__ Request request(const PagedParams& p, int b) {
    return request_at(p.starts, p.context, b, p.tokens);
}

// The same for a b that is one for the wavefront: its values in scalar registers.
__device__ __forceinline__ Request uniform_request(const PagedParams& p, int b) {
    Request r = request(p, __builtin_amdgcn_readfirstlane(b));
    r.q0 = __builtin_amdgcn_readfirstlane(r.q0);
    r.n = __builtin_amdgcn_readfirstlane(r.n);
    r.ctx = __builtin_amdgcn_readfirstlane(r.ctx);
    return r;
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x);
    return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32 | lo);
}

__device__ __forceinline__ int reach(const PagedParams& p, const Request& r, int i) {
    return keys_seen(r, i, p.causal);
}

// Keys of a request to go through: one past the table at most, since that key
// already makes the rows that see it NaN.
__device__ __forceinline__ int keys_to_scan(const PagedParams& p, int seen) {
    return (int)min((int64_t)seen, ((int64_t)p.width << p.shift) + 1);
}

// Every step-th token's rows of `heads` query heads, all to one value (what: 1
// out, 2 lse).
template <typename T>
__device__ __forceinline__ void fill_rows(const PagedParams& p, int from, int to, int step, int head, int heads,
                                          int what, float value, float lse) {
    const int vecs = p.D >> 3;
    Vec16<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.v[i] = (T)value;
    for (int64_t tok = from; tok < to; tok += step) {
        const int64_t row = tok * p.Hq + head;
        if (what & 1)
            for (int64_t i = threadIdx.x; i < (int64_t)heads * vecs; i += blockDim.x)
                *(Vec16<T>*)((T*)p.out + row * p.D + 8 * i) = v;
        if (p.lse && (what & 2))
            for (int g = threadIdx.x; g < heads; g += blockDim.x) p.lse[(int64_t)(head + g) * p.tokens + tok] = lse;
    }
}

// Joins the parts of one row and writes it.  LANES threads hold its columns, eight
// each, and WAYS sets of them take every WAYS-th part (place(k) of `from`); the
// sets meet in LDS.  The order of the additions follows from the
// lengths alone.  Called by all of a workgroup's 256 threads.
template <typename T, int LANES, int WAYS, typename Place>
__device__ __forceinline__ void join_parts(const PagedParams& p, const Partials& from, bool live, int way, int col,
                                           int parts, const Place& place, const Request& r, int head, int row) {
    __shared__ f32x4 s_o[2][256];
    __shared__ float2 s_ml[256];
    const int tid = threadIdx.x;
    float m = -__builtin_inff(), l = 0.0f;
    f32x4 o0 = {0.0f, 0.0f, 0.0f, 0.0f}, o1 = o0;
    if (live) {
#pragma unroll 8
        for (int k = way; k < parts; k += WAYS) {
            const int64_t at = place(k);
            const float2 one = from.ml[at];
            const float* o = from.o + at * p.D + col;
            const f32x4 y0 = *(const f32x4*)o, y1 = *(const f32x4*)(o + 4);
            const float now = fmaxf(m, one.x);
            const float base = now == -__builtin_inff() ? 0.0f : now;
            const float a = __builtin_amdgcn_exp2f(m - base), f = __builtin_amdgcn_exp2f(one.x - base);
            l = l * a + one.y * f;
            o0 = o0 * a + y0 * f;
            o1 = o1 * a + y1 * f;
            m = now;
        }
    }
    float best = m;
    if constexpr (WAYS > 1) {
        s_o[0][tid] = o0;
        s_o[1][tid] = o1;
        s_ml[tid] = make_float2(m, l);
        __syncthreads();
        if (!live || way != 0) return;
#pragma unroll
        for (int k = 1; k < WAYS; ++k) best = fmaxf(best, s_ml[tid + k * LANES].x);
        const float base = best == -__builtin_inff() ? 0.0f : best;
        l = 0.0f;
        o0 = o1 = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < WAYS; ++k) {
            const float2 one = s_ml[tid + k * LANES];
            const float f = __builtin_amdgcn_exp2f(one.x - base);
            l += one.y * f;
            o0 += s_o[0][tid + k * LANES] * f;
            o1 += s_o[1][tid + k * LANES] * f;
        }
    }
    if (!live) return;
    const int i = row / p.G, token = r.q0 + i, h = head * p.G + row % p.G;
    const bool none = reach(p, r, i) <= 0;
    Vec16<T> v;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v.v[k] = (T)(none ? 0.0f : o0[k] / l);
        v.v[4 + k] = (T)(none ? 0.0f : o1[k] / l);
    }
    *(Vec16<T>*)((T*)p.out + ((int64_t)token * p.Hq + h) * p.D + col) = v;
    if (p.lse && col == 0) p.lse[(int64_t)h * p.tokens + token] = none ? __builtin_inff() : (best + log2f(l)) * kLn2;
}

}  // namespace
}  // namespace kf
