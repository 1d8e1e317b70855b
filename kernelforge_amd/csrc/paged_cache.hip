// The paged 8-bit key/value cache's bookkeeping and writes for gfx950.
//
// Layout, with T = block_tokens: key[blocks, Hkv, T, D], value[blocks, Hkv,
// T/16, D, 16] (the 16 tokens of a group innermost, so that the attention
// reads the transposed operand of its second product as whole 16-byte
// vectors), fp32 key_scale and value_scale [blocks, Hkv].
#include "paged_common.h"

namespace kf {
namespace {

constexpr int kMaxBatch = 4096;      // requests whose sums fit the workgroup's LDS
constexpr int kTableThreads = 512;
constexpr int kTokensPerThread = 4;

// ---------------------------------------------------------------------------
// Block tables and slots.
//
// With o tokens cached and n new ones, a request's new blocks are the block
// indices ceil(o/T) .. ceil((o+n)/T) - 1.  A fresh block's first slot always
// belongs to one of the call's tokens, so the token that stands there writes
// the table entry and nothing has to loop over blocks.  Every workgroup sums
// all lengths for itself (two scans over B values that the L2 holds) and then
// handles its own tokens, four a thread so that a step of 2048 tokens is one
// workgroup and may change the counts in place: one launch, no workspace.  Bound
// by the latency of the lengths, the scans and the entries: 4.8 us for 64 requests
// of one token, 5.9 us for 60000 tokens of 48 prompts.
// ---------------------------------------------------------------------------
struct TableParams {
    int* tables;
    const int* context;
    const int* queries;
    const int* free_blocks;
    const int* free_used;
    int* starts;
    int* context_out;
    int64_t* slots;
    int* used_out;
    int64_t total, free_count;
    int B, width, shift;
    bool write_slots, write_state;
};

// Exclusive prefix sum of one value a thread over the workgroup; `sum` is the
// total.  scratch: one value a wavefront.
__device__ __forceinline__ int64_t block_exclusive_sum(int64_t x, int64_t* scratch, int64_t* sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t incl = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t other = __shfl_up((long long)incl, off, 64);
        if (lane >= off) incl += other;
    }
    if (lane == 63) scratch[wave] = incl;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kTableThreads / 64; ++w) {
        const int64_t v = scratch[w];
        if (w < wave) before += v;
        all += v;
    }
    __syncthreads();
    *sum = all;
    return before + incl - x;
}

__global__ __launch_bounds__(kTableThreads) void paged_tables_kernel(TableParams p) {
    __shared__ int s_start[kMaxBatch + 1];
    __shared__ int s_first[kMaxBatch];  // blocks that earlier requests take
    __shared__ int s_old[kMaxBatch];
    __shared__ int64_t s_scratch[kTableThreads / 64];
    const int tid = threadIdx.x;
    const int T = 1 << p.shift;
    const int per = (p.B + kTableThreads - 1) / kTableThreads;
    const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
    const int64_t used = *p.free_used;

    int64_t mine = 0, all;
    for (int b = b0; b < b1; ++b) mine += max(p.queries[b], 0);
    int64_t at = block_exclusive_sum(mine, s_scratch, &all);
    // Tokens past the call's buffer are not taken: the starts stop at `total`.
    int64_t need = 0;
    for (int b = b0; b < b1; ++b) {
        const int64_t begin = min(at, p.total);
        at += max(p.queries[b], 0);
        const int n = (int)(min(at, p.total) - begin);
        // A count that leaves no room for the new tokens in 32 bits is held there.
        const int old = min(max(p.context[b], 0), INT_MAX - n - T);
        s_start[b] = (int)begin;
        s_old[b] = old;
        need += ((old + n + T - 1) >> p.shift) - ((old + T - 1) >> p.shift);
    }
    if (tid == 0) s_start[p.B] = (int)min(all, p.total);
    int64_t taken;
    int64_t first = block_exclusive_sum(need, s_scratch, &taken);
    for (int b = b0; b < b1; ++b) {
        const int n = (b + 1 < b1 ? s_start[b + 1] : (int)min(at, p.total)) - s_start[b];
        const int old = s_old[b];
        s_first[b] = (int)min(first, (int64_t)INT_MAX);
        first += ((old + n + T - 1) >> p.shift) - ((old + T - 1) >> p.shift);
    }
    __syncthreads();

    // After the barrier above nothing reads `context` or `free_used` any more,
    // so a single workgroup may write them in place.
    if (blockIdx.x == 0) {
        if (p.write_slots)
            for (int b = tid; b <= p.B; b += kTableThreads) p.starts[b] = s_start[b];
        if (p.write_state) {
            for (int b = tid; b < p.B; b += kTableThreads) p.context_out[b] = s_old[b] + s_start[b + 1] - s_start[b];
            if (tid == 0) *p.used_out = (int)min(used + taken, (int64_t)INT_MAX);
        }
    }
    if (!p.write_slots) return;

    const int64_t t0 = ((int64_t)blockIdx.x * kTableThreads + tid) * kTokensPerThread;
    if (t0 >= p.total) return;
    // The last request that starts at or before t0.
    int b = 0;
    for (int lo = 0, hi = p.B; lo < hi;) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= t0) {
            b = mid;
            lo = mid + 1;
        } else {
            hi = mid;
        }
    }
#pragma unroll
    for (int i = 0; i < kTokensPerThread; ++i) {
        const int64_t t = t0 + i;
        if (t >= p.total) return;
        int64_t slot = -1;
        if (t < s_start[p.B]) {
            while (t >= s_start[b + 1]) ++b;
            const int old = s_old[b];
            const int pos = old + (int)(t - s_start[b]);
            const int j = pos >> p.shift, held = (old + T - 1) >> p.shift;
            int* entry = p.tables + (int64_t)b * p.width + j;
            int id = -1;
            if (j < p.width) {
                if (j < held) {
                    id = *entry;
                } else {
                    const int64_t take = used + s_first[b] + (j - held);
                    if (take >= 0 && take < p.free_count) id = p.free_blocks[take];
                    if ((pos & (T - 1)) == 0) *entry = id;
                }
            }
            if (id >= 0) slot = ((int64_t)id << p.shift) + (pos & (T - 1));
        }
        p.slots[t] = slot;
    }
}

// ---------------------------------------------------------------------------
// Writes into the cache.
//
// One workgroup handles the runs that begin in its slice of the tokens, one after
// the other: consecutive tokens of the call whose slots lie in one block, found by
// ballots over the slots of 64 tokens.  A unit is the block's keys or values of
// one head, and each of its 16-token groups has a wavefront, so a unit's elements
// stay in registers between the maximum that sets the scale and the rounding: the
// call reads its inputs once and writes the codes once.  17300 tokens of 8 heads
// of 128 in blocks of 16 (107 MB) take 30 us, 3.5 TB/s, against 20 at a copy's
// rate: a run's loads wait for the one before it.  64 tokens of 64 requests take
// 6 us, which is latency (slots, scale, tokens, maximum).
//
// The scale is the least power of two s >= 2^-126 with max|x| <= M s (M the
// largest code, 448 or 127) and never shrinks while the block fills.  x / s is
// then exact and a code is rounded once; when the scale grows, the codes the
// block holds are multiplied by a power of two, which loses nothing of an e4m3
// code above its subnormals and half a step of an int8 code.
// ---------------------------------------------------------------------------
struct AppendParams {
    const void* x[2];  // key, value
    uint8_t* codes[2];
    float* scales[2];
    int token_stride[2];
    int64_t head_stride[2];
    const int64_t* slots;
    int64_t tokens, capacity;  // capacity: slots of the cache
    int Hkv, D, shift, slice;
};

template <int CT> struct Code;
template <> struct Code<KF_CACHE_E4M3> {
    static constexpr float kMost = 448.0f;
    static constexpr uint32_t kMantissa = 0x600000u;  // 448 = 1.75 * 2^8
    static constexpr int kExponent = 8;
    // Four values of at most kMost as codes, in order from the low byte.
    static __device__ __forceinline__ uint32_t pack(const float* x) {
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], r, true);
    }
    static __device__ __forceinline__ void unpack(uint32_t c, float* x) {
        x[0] = __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8((int)c, 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8((int)c, 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8((int)c, 3);
    }
};
template <> struct Code<KF_CACHE_INT8> {
    static constexpr float kMost = 127.0f;
    static constexpr uint32_t kMantissa = 0x7e0000u;  // 127 = 1.984375 * 2^6
    static constexpr int kExponent = 6;
    static __device__ __forceinline__ uint32_t pack(const float* x) {
        uint32_t r = 0;
        // Adding 1.5 * 2^23 rounds to the nearest whole number, ties to even, and
        // leaves it in the low byte.
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r |= (__float_as_uint(x[i] + 12582912.0f) & 0xffu) << (8 * i);
        return r;
    }
    static __device__ __forceinline__ void unpack(uint32_t c, float* x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(c >> (8 * i));
    }
};

// The least power of two s >= 2^-126 with a <= M s, for finite a >= 0.
template <int CT> __device__ __forceinline__ float power_of_two_scale(float a) {
    const uint32_t bits = __float_as_uint(a);
    int e = (int)(bits >> 23) - 127 - Code<CT>::kExponent + ((bits & 0x7fffffu) > Code<CT>::kMantissa ? 1 : 0);
    return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}

template <int CT> __device__ __forceinline__ uint32_t rescale(uint32_t c, float ratio) {
    float x[4];
    Code<CT>::unpack(c, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fminf(fmaxf(x[i] * ratio, -Code<CT>::kMost), Code<CT>::kMost);
    return Code<CT>::pack(x);
}

// What a unit's threads agree on before they write.
struct UnitScale {
    float inverse;  // 1 / new scale; 0 where the block is not finite
    float ratio;    // old scale / new scale
    bool finite;
};

template <int CT>
__device__ __forceinline__ UnitScale unit_scale(uint32_t magnitude, float old_scale, bool begun, float* stored) {
    UnitScale u;
    float s = 0.0f;
    u.finite = magnitude < 0x7f800000u && (begun || __builtin_isfinite(old_scale));
    if (u.finite) {
        s = power_of_two_scale<CT>(__uint_as_float(magnitude));
        if (!begun) s = fmaxf(s, old_scale);
    }
    *stored = u.finite ? s : __builtin_nanf("");
    u.inverse = u.finite ? 1.0f / s : 0.0f;
    u.ratio = u.finite && !begun ? old_scale / s : 0.0f;
    return u;
}

// The larger magnitudes of two pairs of 16-bit floats, as bits: those are ordered
// as the numbers are, with infinities and NaNs the largest.
__device__ __forceinline__ uint32_t larger_of_pairs(uint32_t most, uint32_t x) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most),
                                                                  __builtin_bit_cast(u16x2, x & 0x7fff7fffu)));
}
// The larger one's bits as fp32.
template <typename T> __device__ __forceinline__ uint32_t larger_of_pair(uint32_t most) {
    const unsigned short bits = (unsigned short)max(most & 0xffffu, most >> 16);
    return __float_as_uint((float)__builtin_bit_cast(T, bits));
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x = max(x, (uint32_t)__shfl_xor((int)x, off, 64));
    return x;
}

template <typename T> struct Pair {
    T v[2];
};

// Which of the call's tokens fills a slot of the run's block: for consecutive
// slots, as a request's tokens have, arithmetic; else a table in LDS.
struct Run {
    int first, count;   // its slots, where they are consecutive
    const int* winner;  // else the last token of the run that names a slot, or -1
    __device__ __forceinline__ int token(int slot) const {
        if (winner) return winner[slot];
        const int k = slot - first;
        return k >= 0 && k < count ? k : -1;
    }
};

// T: element type of the new keys and values; CT: the cache's; DC: the head
// dim's class (64, 128 or 256).  blockDim.x = 64 * max(4, block_tokens / 16).
template <typename T, int CT, int DC> __global__ __launch_bounds__(512) void paged_append_kernel(AppendParams p) {
    constexpr int KI = DC / 32;             // 8-element vectors of a key group per lane
    constexpr int NT = DC == 64 ? 8 : 16;   // tokens of a value group per lane
    constexpr int PI = DC == 256 ? 2 : 1;   // column pairs per lane
    __shared__ int s_winner[128];
    __shared__ uint32_t s_max[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bt = 1 << p.shift, groups = bt >> 4, D = p.D;
    const int unit = blockIdx.y * ((int)(blockDim.x >> 6) / groups) + wave / groups;
    const int g = wave % groups;
    const bool active = unit < 2 * p.Hkv;
    const int part = active && unit >= p.Hkv ? 1 : 0;
    const int head = active ? unit - part * p.Hkv : 0;
    // This lane's first key vector (token, vector of its row) and the step of 64.
    const int key_tok = lane / (D >> 3), key_col = lane - key_tok * (D >> 3);
    const int key_step_tok = 64 / (D >> 3), key_step_col = 64 - key_step_tok * (D >> 3);
    // Its columns and tokens of a value group.
    const int pairs = DC == 64 ? 32 : 64;
    const int vcol = 2 * (lane % pairs), vtok = DC == 64 ? 8 * (lane / pairs) : 0;
    const int vlane = vtok * p.token_stride[1] + vcol;

    // The slots from this workgroup's slice on, one a lane, and where runs begin.
    const int64_t t_begin = (int64_t)blockIdx.x * p.slice;
    const int in_slice = (int)min((int64_t)p.slice, p.tokens - t_begin);
    auto slot_at = [&](int64_t t) { return t >= 0 && t < p.tokens ? p.slots[t] : (int64_t)-1; };
    auto block_of = [&](int64_t slot) { return block_of_slot(slot, p.capacity, p.shift); };
    const int64_t window = slot_at(t_begin + lane);
    int64_t before = __shfl_up((long long)window, 1, 64);
    if (lane == 0) before = slot_at(t_begin - 1);
    const bool goes_on = block_of(window) >= 0 && block_of(window) == block_of(before);
    const uint64_t continues = __ballot(goes_on), steps = __ballot(goes_on && window == before + 1);
    uint64_t begins = __ballot(lane < in_slice && block_of(window) >= 0) & ~continues;

    while (begins) {
        const int at = __builtin_ctzll(begins);
        begins &= begins - 1;
        const int64_t t = t_begin + at;
        const int64_t slot = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(window >> 32), at) << 32 |
                                       (uint32_t)__builtin_amdgcn_readlane((int)window, at));
        const int64_t block = slot >> p.shift;
        // The run's length, and whether its slots are consecutive.
        const uint64_t behind = at < 63 ? ~(continues >> (at + 1)) : ~0ull;
        int length = 1 + (behind ? __builtin_ctzll(behind) : 63);
        const uint64_t inside = length > 1 ? (~0ull >> (64 - (length - 1))) << (at + 1) : 0;
        bool consecutive = (steps & inside) == inside;
        if (at + length >= 64) {  // it may go on behind the window
            for (;; length += 64) {
                const int64_t s = slot_at(t + length + lane);
                const bool in = block_of(s) == block;
                const uint64_t out = __ballot(!in), other = __ballot(in && s != slot + length + lane);
                const int here = out ? __builtin_ctzll(out) : 64;
                consecutive &= (here == 64 ? other : other & ((1ull << here) - 1)) == 0;
                if (out) {
                    length += here;
                    break;  // at the call's last token at the latest
                }
            }
        }
        Run run{(int)(slot & (bt - 1)), length, nullptr};
        if (!consecutive) {  // the same for all of the workgroup's wavefronts
            __syncthreads();
            for (int i = tid; i < bt; i += blockDim.x) s_winner[i] = -1;
            __syncthreads();
            for (int i = tid; i < length; i += blockDim.x) atomicMax(&s_winner[p.slots[t + i] & (bt - 1)], i);
            __syncthreads();
            run.winner = s_winner;
        }
        const bool begun = run.token(0) >= 0;
        // The group whole, from consecutive tokens: nothing to look up or to keep.
        const bool whole = consecutive && run.first <= g * 16 && run.first + length >= g * 16 + 16;

        const int64_t where = block * p.Hkv + head;
        const float old_scale = active ? p.scales[part][where] : 0.0f;
        const int ts = p.token_stride[part];
        const T* x = (const T*)p.x[part] + t * ts + head * p.head_stride[part];
        const T* rows = x + (int64_t)(g * 16 - run.first) * ts;  // of a whole group
        uint8_t* codes = p.codes[part] + where * bt * D + g * 16 * D;
        float stored;

        // The unit's scale from a lane's largest pair.  All of a unit's wavefronts
        // meet here.
        auto scale_of = [&](uint32_t pair) {
            uint32_t most = wave_max_u32(larger_of_pair<T>(pair));
            if (groups > 1) {
                __syncthreads();  // the run before has read its maxima
                if (lane == 0) s_max[wave] = most;
                __syncthreads();
                for (int w = 0; w < groups; ++w) most = max(most, s_max[wave - g + w]);
            }
            return unit_scale<CT>(most, old_scale, begun, &stored);
        };

        if (part == 0) {
            // Keys: vector c of the group is 8 columns of token c / (D/8).
            u32x4 kx[KI];
            uint32_t have = 0, pair = 0;
            int tok = key_tok, col = key_col;
#pragma unroll
            for (int i = 0; i < KI; ++i) {
                kx[i] = (u32x4){0u, 0u, 0u, 0u};
                if (tok < 16 && active) {
                    if (whole) {
                        kx[i] = *(const u32x4*)(rows + (int64_t)tok * ts + 8 * col);
                        have |= 1u << i;
                    } else {
                        const int w = run.token(g * 16 + tok);
                        if (w >= 0) {
                            kx[i] = *(const u32x4*)(x + (int64_t)w * ts + 8 * col);
                            have |= 1u << i;
                        }
                    }
                }
                tok += key_step_tok;
                col += key_step_col;
                if (col >= D >> 3) {
                    col -= D >> 3;
                    ++tok;
                }
            }
#pragma unroll
            for (int i = 0; i < KI; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) pair = larger_of_pairs(pair, kx[i][k]);
            const UnitScale u = scale_of(pair);
            if (!active) continue;
            const bool finite = __builtin_amdgcn_readfirstlane(u.finite);
#pragma unroll
            for (int i = 0; i < KI; ++i) {
                const int c = lane + 64 * i;
                if (c >= 2 * D) continue;
                u32x2* to = (u32x2*)(codes + 8 * c);
                u32x2 r = {0u, 0u};
                if (have >> i & 1) {
                    if (finite) {
                        float y[8];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const Pair<T> two = __builtin_bit_cast(Pair<T>, (uint32_t)kx[i][k]);
                            y[2 * k] = (float)two.v[0] * u.inverse;
                            y[2 * k + 1] = (float)two.v[1] * u.inverse;
                        }
                        r[0] = Code<CT>::pack(y);
                        r[1] = Code<CT>::pack(y + 4);
                    }
                } else if (!begun) {
                    if (u.ratio == 1.0f) continue;
                    r = *to;
                    r[0] = rescale<CT>(r[0], u.ratio);
                    r[1] = rescale<CT>(r[1], u.ratio);
                }
                *to = r;
            }
        } else {
            // Values: lane (pair, part of the group) holds two columns of NT tokens.
            uint32_t vx[PI][NT], have = (1u << NT) - 1u, pair = 0;
            if (whole) {
#pragma unroll
                for (int k = 0; k < NT; ++k)
#pragma unroll
                    for (int q = 0; q < PI; ++q)
                        vx[q][k] = vcol + 128 * q < D ? *(const uint32_t*)(rows + (int64_t)k * ts + vlane + 128 * q) : 0u;
            } else {
                have = 0;
#pragma unroll
                for (int k = 0; k < NT; ++k) {
                    const int w = run.token(g * 16 + vtok + k);
                    if (w >= 0) have |= 1u << k;
#pragma unroll
                    for (int q = 0; q < PI; ++q) {
                        vx[q][k] = 0;
                        if (w >= 0 && vcol + 128 * q < D)
                            vx[q][k] = *(const uint32_t*)(x + (int64_t)w * ts + vcol + 128 * q);
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < PI; ++q)
#pragma unroll
                for (int k = 0; k < NT; ++k) pair = larger_of_pairs(pair, vx[q][k]);
            const UnitScale u = scale_of(pair);
            const bool finite = __builtin_amdgcn_readfirstlane(u.finite), all = have == (1u << NT) - 1u;
#pragma unroll
            for (int q = 0; q < PI; ++q) {
                const int col = vcol + 128 * q;
                if (col >= D) continue;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    typedef uint32_t words __attribute__((ext_vector_type(NT / 4)));
                    words* to = (words*)(codes + (col + e) * 16 + vtok);
                    words r = {};
                    if (finite) {
#pragma unroll
                        for (int k4 = 0; k4 < NT / 4; ++k4) {
                            float y[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                y[k] = (float)__builtin_bit_cast(Pair<T>, vx[q][4 * k4 + k]).v[e] * u.inverse;
                            r[k4] = Code<CT>::pack(y);
                        }
                    }
                    if (!all) {
                        if (have == 0 && !begun && u.ratio == 1.0f) continue;
                        words held = {};
                        if (!begun) held = *to;
#pragma unroll
                        for (int k4 = 0; k4 < NT / 4; ++k4) {
                            uint32_t mine = 0;
#pragma unroll
                            for (int k = 0; k < 4; ++k) mine |= have >> (4 * k4 + k) & 1 ? 0xffu << (8 * k) : 0u;
                            const uint32_t keep = u.ratio == 1.0f || begun ? held[k4] : rescale<CT>(held[k4], u.ratio);
                            r[k4] = (r[k4] & mine) | (keep & ~mine);
                        }
                    }
                    *to = r;
                }
            }
        }
        if (g == 0 && lane == 0) p.scales[part][where] = stored;
    }
}

template <typename T, int CT> void launch_append(const AppendParams& p, dim3 grid, int threads, hipStream_t stream) {
    if (p.D <= 64)
        paged_append_kernel<T, CT, 64><<<grid, threads, 0, stream>>>(p);
    else if (p.D <= 128)
        paged_append_kernel<T, CT, 128><<<grid, threads, 0, stream>>>(p);
    else
        paged_append_kernel<T, CT, 256><<<grid, threads, 0, stream>>>(p);
}

}  // namespace
}  // namespace kf

extern "C" {

int kf_paged_block_tables(int32_t* block_tables, const int32_t* context_lens, const int32_t* query_lens,
                          const int32_t* free_blocks, const int32_t* free_used, int32_t* query_starts,
                          int32_t* context_lens_out, int64_t* slots, int32_t* free_used_out, int64_t B,
                          int64_t table_width, int64_t free_count, int64_t total_tokens, int64_t block_tokens,
                          kf_stream_t stream) {
    using namespace kf;
    clear_error();
    KF_REQUIRE(B >= 1 && table_width >= 0 && free_count >= 0 && total_tokens >= 0, KF_E_INVALID,
               "kf_paged_block_tables: bad shape");
    KF_REQUIRE(B <= kMaxBatch, KF_E_UNSUPPORTED, "kf_paged_block_tables: at most %d requests", kMaxBatch);
    const int shift = block_shift(block_tokens);
    KF_REQUIRE(shift > 0, KF_E_INVALID, "kf_paged_block_tables: block_tokens must be 16, 32, 64 or 128");
    KF_REQUIRE(table_width <= INT32_MAX && total_tokens <= INT64_C(1) << 30, KF_E_UNSUPPORTED,
               "kf_paged_block_tables: at most 2^30 tokens and a table width of 32 bits");
    KF_REQUIRE(context_lens && query_lens && free_used && query_starts && context_lens_out && free_used_out &&
                   (block_tables || table_width == 0) && (free_blocks || free_count == 0) && (slots || total_tokens == 0),
               KF_E_INVALID, "kf_paged_block_tables: null pointer");
    TableParams p{block_tables, context_lens, query_lens,    free_blocks, free_used, query_starts, context_lens_out,
                  slots,        free_used_out, total_tokens, free_count,  (int)B,    (int)table_width, shift,
                  true,         true};
    const int64_t per = (int64_t)kTableThreads * kTokensPerThread;
    const int64_t blocks = total_tokens > per ? (total_tokens + per - 1) / per : 1;
    const hipStream_t s = (hipStream_t)stream;
    // In place, the counts change only after every workgroup has read them.
    const bool apart = blocks > 1 && (context_lens_out == context_lens || free_used_out == free_used);
    p.write_state = !apart;
    paged_tables_kernel<<<dim3((unsigned)blocks), dim3(kTableThreads), 0, s>>>(p);
    int rc = check_launch("kf_paged_block_tables");
    if (rc != KF_OK || !apart) return rc;
    p.write_slots = false;
    p.write_state = true;
    paged_tables_kernel<<<dim3(1), dim3(kTableThreads), 0, s>>>(p);
    return check_launch("kf_paged_block_tables");
}

int kf_paged_cache_append(const void* key, const void* value, const int64_t* slots, void* key_cache,
                          void* value_cache, float* key_scale, float* value_scale, int64_t tokens, int64_t blocks,
                          int64_t Hkv, int64_t D, int64_t block_tokens, int64_t key_token_stride,
                          int64_t key_head_stride, int64_t value_token_stride, int64_t value_head_stride, int dtype,
                          int cache_dtype, kf_stream_t stream) {
    using namespace kf;
    clear_error();
    KF_REQUIRE(tokens >= 0 && blocks >= 1 && Hkv >= 1, KF_E_INVALID, "kf_paged_cache_append: bad shape");
    KF_REQUIRE(D >= 16 && D <= 256 && D % 16 == 0, KF_E_INVALID,
               "kf_paged_cache_append: head dim must be a multiple of 16 <= 256");
    const int shift = block_shift(block_tokens);
    KF_REQUIRE(shift > 0, KF_E_INVALID, "kf_paged_cache_append: block_tokens must be 16, 32, 64 or 128");
    KF_REQUIRE(dtype == KF_F16 || dtype == KF_BF16, KF_E_INVALID, "kf_paged_cache_append: dtype must be f16 or bf16");
    KF_REQUIRE(cache_dtype == KF_CACHE_E4M3 || cache_dtype == KF_CACHE_INT8, KF_E_INVALID,
               "kf_paged_cache_append: bad cache dtype");
    // (a launch holds less than 2^32 threads)
    KF_REQUIRE(blocks <= INT32_MAX && Hkv <= 16384 && tokens < 1 << 27, KF_E_UNSUPPORTED,
               "kf_paged_cache_append: at most 2^31-1 blocks, 2^27-1 tokens and 16384 heads");
    if (tokens == 0) return KF_OK;
    KF_REQUIRE(key && value && slots && key_cache && value_cache && key_scale && value_scale, KF_E_INVALID,
               "kf_paged_cache_append: null pointer");
    KF_REQUIRE(((uintptr_t)key | (uintptr_t)value | (uintptr_t)key_cache | (uintptr_t)value_cache) % 16 == 0 &&
                   (key_token_stride | key_head_stride | value_token_stride | value_head_stride) % 8 == 0,
               KF_E_INVALID, "kf_paged_cache_append: rows must be aligned to 16 bytes");
    KF_REQUIRE(key_token_stride >= 0 && key_token_stride < 1 << 26 && value_token_stride >= 0 &&
                   value_token_stride < 1 << 26,
               KF_E_UNSUPPORTED, "kf_paged_cache_append: token strides must be below 2^26");
    AppendParams p{{key, value},
                   {(uint8_t*)key_cache, (uint8_t*)value_cache},
                   {key_scale, value_scale},
                   {(int)key_token_stride, (int)value_token_stride},
                   {key_head_stride, value_head_stride},
                   slots,
                   tokens,
                   blocks << shift,
                   (int)Hkv,
                   (int)D,
                   shift,
                   1};
    const int bt = 1 << shift, groups = bt >> 4, waves = groups > 4 ? groups : 4;
    const int64_t gy = (2 * Hkv * groups + waves - 1) / waves;
    // Tokens of a workgroup.  Decoding gives every token a block of its own, so one
    // each spreads the runs; prompts begin a run every block_tokens tokens, and most
    // workgroups of one token find nothing.  The host cannot tell the two apart, so
    // 2048 workgroups, eight a CU, decide (8 heads of 128, T = 16, us with 1, 2, 4,
    // 8, 16 tokens each; calls below 9 us wait for the host): 256 requests 10, 10,
    // 14, 25, 45; 1024 requests 25, 23, 23, 30, 49; 4096 requests 82, 71, 67, 68, 75;
    // four prompts of 256 tokens 11, 10, 11, 8, 9; of 1000 28, 17, 15, 11, 11.  At
    // most a block, and the 64 slots that a wavefront looks at (T = 64, 16 against
    // 64 tokens: two prompts of 4000 40, 18; 2048 requests 136, 152).
    const int most = bt < 64 ? bt : 64;
    p.slice = 1;
    while (p.slice < most && p.slice * 2048 < tokens * gy) p.slice *= 2;
    const int64_t gx = (tokens + p.slice - 1) / p.slice;
    const dim3 grid((unsigned)gx, (unsigned)gy);
    const hipStream_t s = (hipStream_t)stream;
    if (dtype == KF_BF16) {
        if (cache_dtype == KF_CACHE_E4M3)
            launch_append<bf16, KF_CACHE_E4M3>(p, grid, 64 * waves, s);
        else
            launch_append<bf16, KF_CACHE_INT8>(p, grid, 64 * waves, s);
    } else {
        if (cache_dtype == KF_CACHE_E4M3)
            launch_append<f16, KF_CACHE_E4M3>(p, grid, 64 * waves, s);
        else
            launch_append<f16, KF_CACHE_INT8>(p, grid, 64 * waves, s);
    }
    return check_launch("kf_paged_cache_append");
}

}  // extern "C"
