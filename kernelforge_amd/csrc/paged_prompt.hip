// Attention over the paged cache: many rows of a request (chunks of prompts).
#include <type_traits>

#include "paged_attn.h"

namespace kf {
namespace {

constexpr float kPromptPScale = 4096.0f;  // 2^12: a probability may exceed its row's reference by 2^kRise
constexpr float kRise = 3.0f;

// ---------------------------------------------------------------------------
// Many rows: 128 (query, head) rows of one key head per workgroup, 16 for each of
// eight wavefronts, 64 keys at a time through LDS.
//
// The products and their operand layouts are those of the few-rows kernel
// (paged_attn.hip): S^T = K Q^T leaves each lane the scores of one 16-token
// group, which are the second product's operand as they are.  Here all
// wavefronts read the same keys.  Two of them load the codes of one of a tile's
// four groups, whose block, address and scales are scalars, a tile ahead into
// registers, and write them into LDS as 16-bit floats behind the first product
// of the tile before; one barrier a tile.
//
// Issue-bound: of two prompts' chunks of 2048 tokens over 8192 keys, 32 heads of
// 128 (425 GFLOP, 549 us, 774 TFLOP/s), the SIMDs issue vector instructions in
// 59% of their cycles and matrix instructions in 36%.  So the instructions for a
// key count: with the codes in LDS and a conversion by each of four wavefronts of
// 32 rows it took 592 us.  Four wavefronts of 32 rows over 16-bit tiles take 561
// (and 138 against 153 at a dim of 64), but are slower on short chunks, which have
// half as many of them to hide the loads.
//
// Keys lie in LDS as rows of 16-byte chunks (8 elements) permuted by key_swizzle,
// values as [group][column][16 tokens] with the halves of odd groups exchanged;
// both leave the operand reads without bank conflicts in 32-lane passes over
// 128 banks.
// ---------------------------------------------------------------------------
template <int DP> struct PromptShape {
    static constexpr int WAVES = 8;
    static constexpr int ROWS = 16 * WAVES;            // of a workgroup
    static constexpr int CH = DP == 96 ? 16 : DP / 8;  // 16-byte chunks of a key row in LDS
    static constexpr int BUFFERS = DP > 128 ? 1 : 2;   // two workgroups share a CU's LDS
    static constexpr int OCC = DP > 128 ? 2 : 4;       // wavefronts a SIMD
};

// The permutation of a key row's chunks.
template <int CH> __device__ __forceinline__ int key_swizzle(int key) {
    const int g = (key >> 4) & 3, e = key & 3;
    if constexpr (CH == 8) return 2 * g + (e >> 1);
    else if constexpr (CH == 16) return 2 * g + 8 * (e >> 1) + (e & 1);
    else return 2 * (4 * g + e);
}

// Integers and scales that one wavefront's lanes share, through scalar loads.
template <typename X> __device__ __forceinline__ X uniform_load(const X* p) {
    return *(const __attribute__((address_space(4))) X*)(uintptr_t)p;
}

struct PromptWork {
    Partials to;
    int units, splits;
};

// A unit's key head (fastest, so that a head's units share an XCD's cache) and
// rows.  Request b's tiles of rows begin at floor(first row / ROWS) + b, which
// leaves room for all of them.  b: -1 where the unit has none.
struct Unit {
    Request r;
    int b, head, row0;
};
template <int ROWS> __device__ __forceinline__ Unit unit_at(const PagedParams& p, int unit) {
    Unit u;
    u.head = unit % p.Hkv;
    const int index = unit / p.Hkv;
    auto tile_of = [&](int first, int b) { return (int)(((int64_t)first * p.G) / ROWS) + b; };
    // The last request whose tiles begin at or before this one, by 64ths.
    int b = 0;
    for (int count = p.B; count > 1;) {
        const int step = (count + 63) >> 6, at = b + step * (int)(threadIdx.x & 63);
        const bool in = at < b + count;
        const int first = !in ? 0 : p.starts ? clamp_int(p.starts[at], 0, p.tokens) : at;
        const int before = __builtin_popcountll(__ballot(in && tile_of(first, at) <= index));
        const int skip = step * (before > 0 ? before - 1 : 0);
        b += skip;
        count = min(count - skip, step);
    }
    u.b = __builtin_amdgcn_readfirstlane(b);
    u.r = uniform_request(p, u.b);
    const int row_tile = index - tile_of(u.r.q0, u.b);
    u.row0 = row_tile * ROWS;
    // (in 64 bits: starts that run backwards can lead to any tile)
    if ((int64_t)u.r.n * p.G <= p.few || row_tile < 0 || (int64_t)row_tile * ROWS >= min(u.r.n, p.max_q) * p.G) u.b = -1;
    return u;
}

template <typename T, int CT, int DP>
__global__ __launch_bounds__(64 * PromptShape<DP>::WAVES, PromptShape<DP>::OCC) void paged_prompt_kernel(
    PagedParams p, PromptWork w) {
    using Shape = PromptShape<DP>;
    constexpr int ROWS = Shape::ROWS, CH = Shape::CH, BUFFERS = Shape::BUFFERS;
    constexpr int KC = DP / 32, VT = DP / 16;
    constexpr int NC = (DP + 127) / 128;  // 16-byte vectors of half a group's codes a lane
    __shared__ u32x4 s_keys[BUFFERS][64 * CH];
    __shared__ u32x4 s_values[BUFFERS][64 * DP / 8];
    __shared__ float2 s_scales[BUFFERS][4];  // key scale (NaN: no such block), value scale

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, quarter = lane >> 4;
    const int group = wave >> 1;  // of a tile, this wavefront's and its neighbour's
    const int D = p.D;

    // The latest units, which see the most keys, go first.
    const Unit u = unit_at<ROWS>(p, w.units - 1 - blockIdx.x);
    const Request r = u.r;
    const int b = u.b, head = u.head, row0 = u.row0, rows = min(r.n, p.max_q) * p.G;
    if (u.b < 0) return;
    if (row0 == 0 && blockIdx.y == 0 && r.n > p.max_q)
        fill_rows<T>(p, r.q0 + p.max_q, r.q0 + r.n, 1, head * p.G, p.G, 3, __builtin_nanf(""), __builtin_nanf(""));

    // This lane's row.
    const int my_row0 = row0 + 16 * wave;
    const int row = my_row0 + m, i = row / p.G;
    const bool live = row < rows;
    const int limit = live ? reach(p, r, i) : 0;
    typename V<T>::x8 qf[KC];
    const T* q = (const T*)p.q + (int64_t)(r.q0 + i) * p.q_ts + (int64_t)(head * p.G + row % p.G) * p.q_hs;
#pragma unroll
    for (int c = 0; c < KC; ++c) {
        const int col = 32 * c + 8 * quarter;
        u32x4 v = {0u, 0u, 0u, 0u};
        if (live && col < D) v = *(const u32x4*)(q + col);
        qf[c] = __builtin_bit_cast(typename V<T>::x8, v);
    }
    auto seen_by = [&](int row) {
        return __builtin_amdgcn_readfirstlane(keys_to_scan(p, reach(p, r, min(row, rows - 1) / p.G)));
    };
    // Keys that the wavefront's rows all see.
    const int all_see = my_row0 < rows ? __builtin_amdgcn_readfirstlane(reach(p, r, my_row0 / p.G)) : 0;
    const int tiles = (seen_by(row0 + ROWS - 1) + 63) >> 6;
    const int first = (int)((int64_t)tiles * blockIdx.y / w.splits);
    const int last = (int)((int64_t)tiles * (blockIdx.y + 1) / w.splits);

    // This wavefront's group: a lane's vectors of codes and where they go.
    const int subs = (1 << (p.shift - 4)) - 1;
    const int64_t unit_bytes = (int64_t)D << p.shift;
    // The codes of a group lie as they are read; past D the query is 0 and columns
    // are not written, so any bytes of the group serve there.
    uint32_t from_k[NC], from_v[NC], to_k[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int slot = (wave & 1) * (DP / 2) + 64 * j + lane, key = slot / (DP / 16), chunk = slot % (DP / 16);
        from_k[j] = key < 16 ? key * D + (16 * chunk < D ? 16 * chunk : 0) : 0;
        from_v[j] = slot < D ? 16 * slot : 0;
        if (DP / 2 % 64 != 0 && slot >= DP) from_k[j] = from_v[j] = 0;
        to_k[j] = (16 * group + key) * CH + ((2 * chunk) ^ key_swizzle<CH>(16 * group + key));  // the other half's ^ 1
    }
    const uint32_t to_v = (group * DP + (wave & 1) * (DP / 2) + lane) * 2 + (group & 1);  // likewise
    const int* table = p.tables + (int64_t)b * p.width;
    auto entry_of = [&](int tile) {
        const int entry = (4 * tile + group) >> (p.shift - 4);
        return uniform_load(table + min(entry, p.width - 1));
    };
    auto block_of = [&](int id, int tile) {
        return __builtin_amdgcn_readfirstlane(block_of_entry(id, p.width, p.blocks, p.shift, 4 * tile + group));
    };
    u32x4 codes_k[NC], codes_v[NC];
    auto load_codes = [&](int tile, int block) {
        const int64_t at = ((int64_t)max(block, 0) * p.Hkv + head) * unit_bytes + 16 * ((4 * tile + group) & subs) * D;
        const uint8_t *k = p.kc + at, *v = p.vc + at;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            codes_k[j] = *(const u32x4*)(k + from_k[j]);
            codes_v[j] = *(const u32x4*)(v + from_v[j]);
        }
    };
    auto store_codes = [&](int buffer, int valid) {
        // Values behind the context or of no block are zeroed: what lies there may be NaN.
        if (valid < 16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int bytes = clamp_int(valid - 4 * e, 0, 4);
                const uint32_t mask = bytes == 4 ? 0xffffffffu : (1u << (8 * bytes)) - 1u;
#pragma unroll
                for (int j = 0; j < NC; ++j) codes_v[j][e] &= mask;
            }
        }
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            if (DP / 2 % 64 != 0 && 64 * j + lane >= DP / 2) continue;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const auto k = Codes<T, CT>::x8(codes_k[j][2 * h], codes_k[j][2 * h + 1]);
                const auto v = Codes<f16, CT>::x8(codes_v[j][2 * h], codes_v[j][2 * h + 1]);
                s_keys[buffer][to_k[j] ^ h] = __builtin_bit_cast(u32x4, k);
                s_values[buffer][(to_v + 128 * j) ^ h] = __builtin_bit_cast(u32x4, v);
            }
        }
    };
    auto valid_of = [&](int tile, int block) {
        return block < 0 ? 0 : clamp_int(r.ctx - (64 * tile + 16 * group), 0, 16);
    };
    auto scales_of = [&](int tile, int block) {
        const int64_t at = (int64_t)max(block, 0) * p.Hkv + head;
        const float vs = uniform_load(p.vs + at);
        // A key scale of 0 is held above it, so that a hidden key's -inf stays one.
        const float ks = uniform_load(p.ks + at) * p.c;
        float2 s = make_float2(ks < kLeastScale ? kLeastScale : ks, vs < __builtin_inff() ? vs : __builtin_nanf(""));
        if (block < 0) s = make_float2(__builtin_nanf(""), 0.0f);
        if (64 * tile + 16 * group >= r.ctx) s = make_float2(1.0f, 0.0f);  // says nothing
        return s;
    };

    f32x4 acc[VT];
    float ref = -__builtin_inff(), sum = 0.0f, vref = kLeastScale, inv_vref = 1.0f / kLeastScale;
#pragma unroll
    for (int d = 0; d < VT; ++d) acc[d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    // Operand reads: a lane's chunk of column block c, and its values' halves.
    uint32_t read_k = (16 * (m >> 2) + (m & 3)) * CH + (quarter ^ key_swizzle<CH>(16 * (m >> 2) + (m & 3)));
    const uint32_t read_v = (quarter * DP + m) * 2 + (quarter & 1);

    int block = -1, ahead = 0;
    if (first < last) {
        block = block_of(entry_of(first), first);
        load_codes(first, block);
        ahead = entry_of(min(first + 1, last - 1));
        const float2 s = scales_of(first, block);
        store_codes(0, valid_of(first, block));
        if (lane == 0) s_scales[0][group] = s;
        block = block_of(ahead, min(first + 1, last - 1));
        load_codes(min(first + 1, last - 1), block);
    }
    int now = 0;
    for (int tile = first; tile < last; ++tile) {
        __syncthreads();
        const int then = min(tile + 1, last - 1);  // the tile in the registers, the last one again at the end
        const float2 next_scales = scales_of(then, block);
        auto pass_on = [&](int buffer) {
            store_codes(buffer, valid_of(then, block));
            if (lane == 0) s_scales[buffer][group] = next_scales;
            const int after = min(tile + 2, last - 1);
            block = block_of(entry_of(after), after);
            load_codes(after, block);
        };
        const float2 mine = s_scales[now][quarter];
        const float vmax = fmaxf(fmaxf(s_scales[now][0].y, s_scales[now][1].y),
                                 fmaxf(s_scales[now][2].y, s_scales[now][3].y));
        asm volatile("" : "+v"(read_k));  // its columns' addresses are formed here, not kept
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            s[t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const auto a = __builtin_bit_cast(typename V<T>::x8, s_keys[now][(read_k ^ (4 * c)) + 4 * t * CH]);
                s[t] = mfma16x16x32(a, qf[c], s[t]);
            }
        }
        if constexpr (BUFFERS == 2) pass_on(now ^ 1);
        const int key0 = 64 * tile + 16 * quarter;  // position of this lane's first key
        const bool edge = 64 * tile + 64 > all_see;
        // The lane's keys share a scale, which is not negative: their largest
        // product is their largest score.
        float most;
        // Keys of this lane's group that its row sees.  The empty asm keeps the
        // comparisons out of the tiles that every row sees whole.
        auto seen_here = [&] {
            int n = limit - key0;
            asm volatile("" : "+v"(n));
            return n;
        };
        auto largest = [&](auto at_edge) {
            if (decltype(at_edge)::value) {
                const int n = seen_here();
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (4 * t + i >= n) s[t][i] = -__builtin_inff();
            }
            float x = s[0][0];
#pragma unroll
            for (int k = 1; k < 16; ++k) x = fmaxf(x, s[k >> 2][k & 3]);
            most = row_max4(x * mine.x);
        };
        if (edge)
            largest(std::true_type());
        else
            largest(std::false_type());
        // The references follow the rows' maxima when one has risen by 2^kRise.
        if (__any(most > ref + kRise) || vmax > vref) {
            const float shrink = vmax > vref ? vref / vmax : 1.0f;
            if (vmax > vref) {
                vref = vmax;
                inv_vref = 1.0f / vmax;
            }
            const float to = fmaxf(ref, most);
            const float alpha = to == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(ref - to);
            ref = to;
            sum *= alpha;
#pragma unroll
            for (int d = 0; d < VT; ++d) acc[d] *= alpha * shrink;
        }
        // exp2(score - reference) * factor as one exponential of one fma; the
        // sum takes the factor out again.  A factor below 2^-60 counts as 2^-60:
        // its products are 0 in f16 either way.
        const float factor = mine.y * inv_vref * kPromptPScale;
        const float least = factor < 0x1p-60f ? 0x1p-60f : factor;  // keeps a NaN
        const float lift = __builtin_amdgcn_logf(least), unlift = __builtin_amdgcn_exp2f(-lift);
        V<f16>::x8 pf[2];
        auto probabilities = [&](auto at_edge) {
            const float base = lift - (ref == -__builtin_inff() ? 0.0f : ref);
            float add = 0.0f;
            const int n = decltype(at_edge)::value ? seen_here() : 0;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], mine.x, base));
                    // A hidden key's weight is 0 whatever its block's scale.
                    if (decltype(at_edge)::value && 4 * t + i >= n) e = 0.0f;
                    add += e;
                    pf[t >> 1][4 * (t & 1) + i] = (f16)e;
                }
            sum += add == 0.0f ? 0.0f : add * unlift;  // rows that see no key of a NaN scale
        };
        if (edge)
            probabilities(std::true_type());
        else
            probabilities(std::false_type());
#pragma unroll
        for (int d = 0; d < VT; ++d)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const auto a = __builtin_bit_cast(V<f16>::x8, s_values[now][(read_v ^ h) + 32 * d]);
                acc[d] = mfma16x16x32(a, pf[h], acc[d]);
            }
        if constexpr (BUFFERS == 1) {
            __syncthreads();
            pass_on(0);
        } else {
            now ^= 1;
        }
    }

    const float l = row_sum4(sum);
    if (!live) return;
    const int token = r.q0 + i, h = head * p.G + row % p.G;
    if (w.splits > 1) {
        const int64_t at = ((int64_t)blockIdx.x * w.splits + blockIdx.y) * ROWS + (row - row0);
        if (quarter == 0) w.to.ml[at] = make_float2(ref, l);
#pragma unroll
        for (int d = 0; d < VT; ++d)
            if (16 * d < D)
                *(f32x4*)(w.to.o + at * D + 16 * d + 4 * quarter) = acc[d] * (1.0f / kPromptPScale) * vref;
        return;
    }
    const bool none = limit <= 0;
#pragma unroll
    for (int d = 0; d < VT; ++d) {
        if (16 * d >= D) continue;
        const f32x4 o = acc[d] * (1.0f / kPromptPScale) * vref;
        typename V<T>::x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(none ? 0.0f : o[e] / l);
        *(typename V<T>::x4*)((T*)p.out + ((int64_t)token * p.Hq + h) * D + 16 * d + 4 * quarter) = v;
    }
    if (p.lse && quarter == 0)
        p.lse[(int64_t)h * p.tokens + token] = none ? __builtin_inff() : (ref + log2f(l)) * kLn2;
}

// Joins a unit's splits, in order: LANES threads with eight columns each a row.
template <typename T, int ROWS, int LANES>
__global__ __launch_bounds__(256) void paged_prompt_join_kernel(PagedParams p, PromptWork w) {
    const Unit u = unit_at<ROWS>(p, w.units - 1 - blockIdx.x);
    if (u.b < 0) return;
    const int tid = threadIdx.x, col = 8 * (tid % LANES);
    const int x = blockIdx.y * (256 / LANES) + tid / LANES, row = u.row0 + x;
    const bool live = row < min(u.r.n, p.max_q) * p.G && col < p.D;
    join_parts<T, LANES, 1>(
        p, w.to, live, 0, col, w.splits,
        [&](int k) { return ((int64_t)blockIdx.x * w.splits + k) * ROWS + x; }, u.r, u.head, row);
}

template <typename T, int CT, int DP>
int launch_shape(const PagedParams& p, const PromptWork& w, hipStream_t s) {
    constexpr int ROWS = PromptShape<DP>::ROWS;
    const dim3 grid((unsigned)w.units, (unsigned)w.splits), threads(64 * PromptShape<DP>::WAVES);
    paged_prompt_kernel<T, CT, DP><<<grid, threads, 0, s>>>(p, w);
    int rc = check_launch("kf_paged_attention (prompts)");
    if (rc != KF_OK || w.splits == 1) return rc;
    constexpr int LANES = DP == 96 ? 16 : DP / 8;  // of a row's columns
    paged_prompt_join_kernel<T, ROWS, LANES><<<dim3((unsigned)w.units, ROWS * LANES / 256), 256, 0, s>>>(p, w);
    return check_launch("kf_paged_attention (prompts' join)");
}

template <typename T, int CT> int launch_dim(const PagedParams& p, const PromptWork& w, hipStream_t s) {
    if (p.D <= 64) return launch_shape<T, CT, 64>(p, w, s);
    if (p.D <= 96) return launch_shape<T, CT, 96>(p, w, s);
    if (p.D <= 128) return launch_shape<T, CT, 128>(p, w, s);
    return launch_shape<T, CT, 256>(p, w, s);
}

constexpr int kUnitRows = PromptShape<128>::ROWS;

}  // namespace

int64_t prompt_units(int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv) {
    return (tokens * (Hq / Hkv) / kUnitRows + B) * Hkv;
}

PromptPlan prompt_plan(int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_ctx) {
    PromptPlan w;
    const int64_t rows = kUnitRows;
    w.units = prompt_units(tokens, B, Hq, Hkv);
    // Two workgroups a CU fit; fewer units than CUs have their keys split over two
    // a CU (us, split against whole, 32/8 heads of 128: 36 tokens over 30000 keys
    // 66, 850; 512 over 30000 304, 764; 200 over 2000 33, 69).  260 units at a dim
    // of 256 take 214 in two parts and 178 whole.  The parts are counted for units
    // that are full, in one round of workgroups (200 tokens over 2000 keys, 9 parts
    // of 56 units 33, 10 parts 41; four of 100 over 1000, 4 parts of 104 31, 5 parts
    // 39; 12 ragged requests of 1 to 700, 2 parts of 188 94, 3 parts 92).
    const int64_t full = ((tokens > 0 ? tokens : 1) * (Hq / Hkv) + rows - 1) / rows * Hkv;
    int64_t splits = w.units >= device_cu_count() ? 1 : 2 * device_cu_count() / full;
    // A part has at least so many keys (64 tokens over 1000 keys with 128, 256, 512:
    // 18, 23, 35 us; at a dim of 256 300 tokens over 1000 keys 39, 33, 50).
    const int64_t most = max_ctx / (D > 128 ? 256 : 128);
    if (splits > most) splits = most;
    // Requests of few rows leave units empty: not more than 4 a CU, which bounds the
    // workspace.
    if (splits > 4 * device_cu_count() / w.units) splits = 4 * device_cu_count() / w.units;
    w.splits = splits > 1 ? (int)splits : 1;
    w.bytes = w.splits > 1 ? w.units * w.splits * rows * (D * 4 + 8) : 0;
    return w;
}

int launch_prompt(const PagedParams& p, const PromptPlan& plan, void* workspace, int dtype, int cache_dtype,
                  hipStream_t stream) {
    PromptWork w;
    w.to.o = (float*)workspace;
    w.to.ml = (float2*)(w.to.o + plan.units * plan.splits * kUnitRows * p.D);
    w.units = (int)plan.units;
    w.splits = plan.splits;
    const bool e4m3 = cache_dtype == KF_CACHE_E4M3;
    if (dtype == KF_BF16)
        return e4m3 ? launch_dim<bf16, KF_CACHE_E4M3>(p, w, stream) : launch_dim<bf16, KF_CACHE_INT8>(p, w, stream);
    return e4m3 ? launch_dim<f16, KF_CACHE_E4M3>(p, w, stream) : launch_dim<f16, KF_CACHE_INT8>(p, w, stream);
}

}  // namespace kf
