// Attention over the paged 8-bit key/value cache (layout: paged_cache.hip).
//
// With P the probabilities of a row and S its scores,
//   S_j = scale ks_j <q, kcode_j>,  O = sum_j exp(S_j - max) vs_j vcode_j / sum_j exp(S_j - max),
// ks and vs the scales of key j's block.  Codes enter the matrix products as
// 16-bit floats without rounding; a block's key scale multiplies the fp32
// score and its value scale the fp32 probability.
//
// P is rounded once, to f16 whatever q's type: p * vs / vref * 2^15 with vref
// the largest value scale seen so far, so the product is at most 2^15 and
// stays a normal number down to 2^-29 of the largest term (f16 rounds by at most
// 2^-11 where bf16 would by 2^-8).  Maxima, sums and accumulators are fp32.
#include "paged_common.h"

namespace kf {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kPScale = 32768.0f;  // 2^15, the largest f16 operand of the second product
constexpr int kMaxSplits = 64;
constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126

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
    float2* ml;   // [tokens * Hq][splits]: running maximum (log2 units) and sum
    float* part;  // [splits][tokens * Hq][D]
    int64_t q_ts, q_hs;
    int tokens, B, blocks, width, Hq, Hkv, G, D, shift;
    int max_q, row_tiles, splits;
    float c;  // scale * log2(e)
    bool causal;
    int clear_rest;  // rows behind the last request: 1 out, 2 lse
};

__device__ __forceinline__ Request request(const PagedParams& p, int b) {
    return request_at(p.starts, p.context, b, p.tokens);
}

__device__ __forceinline__ int reach(const PagedParams& p, const Request& r, int i) {
    return keys_seen(r, i, p.causal);
}

// The rows of tokens [from, to) of one key head, all to one value.
// (what: 1 out, 2 lse).
template <typename T>
__device__ __forceinline__ void fill_rows(const PagedParams& p, int head, int from, int to, int what, float value,
                                          float lse) {
    const int vecs = p.D >> 3;
    Vec16<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.v[i] = (T)value;
    for (int tok = from; tok < to; ++tok) {
        const int64_t row = (int64_t)tok * p.Hq + head * p.G;
        if (what & 1)
            for (int i = threadIdx.x; i < p.G * vecs; i += blockDim.x)
                *(Vec16<T>*)((T*)p.out + row * p.D + 8 * i) = v;
        if (p.lse && (what & 2))
            for (int g = threadIdx.x; g < p.G; g += blockDim.x)
                p.lse[(int64_t)(head * p.G + g) * p.tokens + tok] = lse;
    }
}

// ---------------------------------------------------------------------------
// Few rows: 16 * RT (query, head) rows of one key head per workgroup, keys
// split over its 4 wavefronts and over workgroups.
//
// A wavefront takes 64 keys at a time, as four 16-token groups.  S^T = K Q^T
// with K as the A operand: tile t's row m' is token 4t + m'%4 of group m'/4,
// so the D layout (column = row of Q = lane%16, rows 4*(lane/16)+i) leaves lane
// (row, quarter) with all 16 scores of its quarter's group: one key scale and
// one value scale a lane, and exactly the B operand O^T = V^T P^T wants when
// V^T's lane (column, quarter) holds the same 16 tokens of its column, which
// is 16 contiguous bytes of the value cache.  Nothing passes through LDS and
// every load is 16 bytes a lane.
// ---------------------------------------------------------------------------
template <typename T, int CT, int DP, int RT>
__global__ __launch_bounds__(256, DP * RT > 128 ? 1 : 2) void paged_rows_kernel(PagedParams p) {
    constexpr int KC = DP / 64;   // 64-column chunks of a key row
    constexpr int VT = DP / 16;   // 16-column tiles of the output
    constexpr int OC = DP < 128 ? DP : 128;  // columns joined at a time
    constexpr int PITCH = OC + 4;
    __shared__ float s_acc[4][16][PITCH];
    __shared__ float s_m[4][16 * RT], s_l[4][16 * RT];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int m = lane & 15, quarter = lane >> 4;
    const int b = blockIdx.x / p.row_tiles, tile_of_rows = blockIdx.x % p.row_tiles;
    const int head = blockIdx.y, split = blockIdx.z;
    const Request r = request(p, b);
    const int D = p.D;

    if (split == 0 && tile_of_rows == 0 && p.starts) {
        if (r.n > p.max_q)
            fill_rows<T>(p, head, r.q0 + p.max_q, r.q0 + r.n, 3, __builtin_nanf(""), __builtin_nanf(""));
        if (b == p.B - 1) fill_rows<T>(p, head, r.q0 + r.n, p.tokens, p.clear_rest, 0.0f, __builtin_inff());
    }
    const int row0 = tile_of_rows * 16 * RT, rows = min(r.n, p.max_q) * p.G;
    if (row0 >= rows) return;

    // This lane's rows (columns of S^T).
    int limit[RT];
    typename V<T>::x8 qf[RT][KC][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = row0 + 16 * rt + m, i = row / p.G;
        const bool live = row < rows;
        limit[rt] = live ? reach(p, r, i) : 0;
        const T* q = (const T*)p.q + (int64_t)(r.q0 + i) * p.q_ts + (int64_t)(head * p.G + row % p.G) * p.q_hs;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int col = 64 * c + 16 * quarter + 8 * h;
                u32x4 v = {0u, 0u, 0u, 0u};
                if (live && col < D) v = *(const u32x4*)(q + col);
                qf[rt][c][h] = __builtin_bit_cast(typename V<T>::x8, v);
            }
    }
    // Keys that every row sees, and that any row sees (one past the table at
    // most: that key already makes the row NaN).
    const int all_see = reach(p, r, row0 / p.G);
    const int64_t table_keys = ((int64_t)p.width << p.shift) + 1;
    const int any_sees = (int)min((int64_t)reach(p, r, (min(row0 + 16 * RT, rows) - 1) / p.G), table_keys);
    const int tiles = (any_sees + 63) >> 6;
    const int per_split = (tiles + p.splits - 1) / p.splits;
    const int first = split * per_split, last = min(first + per_split, tiles);
    const int per_wave = max((last - first + 3) / 4, 0);
    const int t0 = first + wave * per_wave, t1 = min(t0 + per_wave, last);

    const int* table = p.tables + (int64_t)b * p.width;
    const int subs = (1 << (p.shift - 4)) - 1;  // groups of a block - 1
    const int64_t unit = (int64_t)D << p.shift;  // bytes of a block's keys of one head
    auto id_of = [&](int group) { return block_of_group(table, p.width, p.blocks, p.shift, group); };
    u32x4 kr[4][KC], vr[VT];
    auto load_keys = [&](int tile, int id) {
        const int sub = (4 * tile + (m >> 2)) & subs;
        const uint8_t* base = p.kc + ((int64_t)max(id, 0) * p.Hkv + head) * unit + (16 * sub + (m & 3)) * D;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const int col = 64 * c + 16 * quarter;  // past D: any bytes, the query is 0 there
                kr[t][c] = *(const u32x4*)(base + 4 * t * D + (col < D ? col : 0));
            }
    };
    auto load_values = [&](int tile, int id) {
        const int sub = (4 * tile + quarter) & subs;
        const uint8_t* base = p.vc + ((int64_t)max(id, 0) * p.Hkv + head) * unit + 16 * sub * D;
#pragma unroll
        for (int d = 0; d < VT; ++d)
            if (16 * d < D) vr[d] = *(const u32x4*)(base + (16 * d + m) * 16);
    };

    f32x4 acc[RT][VT];
    float top[RT], sum[RT], vref = kLeastScale, inv_vref = 1.0f / kLeastScale;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        top[rt] = -__builtin_inff();
        sum[rt] = 0.0f;
#pragma unroll
        for (int d = 0; d < VT; ++d) acc[rt][d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }

    int idk = -1, idv = -1, next_idk = -1, next_idv = -1;
    float ks = 0.0f, vs = 0.0f;
    auto load_scales = [&](int id) {
        const int64_t at = (int64_t)max(id, 0) * p.Hkv + head;
        ks = p.ks[at];
        vs = p.vs[at];
    };
    if (t0 < t1) {
        idk = id_of(4 * t0 + (m >> 2));
        idv = id_of(4 * t0 + quarter);
        load_scales(idv);
        load_keys(t0, idk);
        load_values(t0, idv);
        if (t0 + 1 < t1) {
            next_idk = id_of(4 * t0 + 4 + (m >> 2));
            next_idv = id_of(4 * t0 + 4 + quarter);
        }
    }
    for (int tile = t0; tile < t1; ++tile) {
        f32x4 s[RT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][t] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const auto a = Codes<T, CT>::x8(kr[t][c][2 * h], kr[t][c][2 * h + 1]);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) s[rt][t] = mfma16x16x32(a, qf[rt][c][h], s[rt][t]);
                }
        }
        const int group0 = tile * 64 + 16 * quarter;  // position of this lane's first key
        const bool bad = idv < 0 && group0 < r.ctx;
        const bool edge = tile * 64 + 64 > all_see || __any(idv < 0);
        const float kscale = bad ? __builtin_nanf("") : ks * p.c;
        // Blocks behind the context say nothing; an infinite scale is a NaN, which
        // only the rows that see its block take on.
        const float vscale = idv < 0 || group0 >= r.ctx ? 0.0f : vs < __builtin_inff() ? vs : __builtin_nanf("");
        const int idv_now = idv;
        if (tile + 1 < t1) {
            idk = next_idk;
            idv = next_idv;
            load_scales(idv);
            load_keys(tile + 1, idk);
            if (tile + 2 < t1) {
                next_idk = id_of(4 * tile + 8 + (m >> 2));
                next_idv = id_of(4 * tile + 8 + quarter);
            }
        }

        // The largest value scale so far, the same on every lane.
        float vmax = fmaxf(vscale, __shfl_xor(vscale, 16, 64));
        vmax = fmaxf(vmax, __shfl_xor(vmax, 32, 64));
        float shrink = 1.0f;
        if (vmax > vref) {
            shrink = vref / vmax;
            vref = vmax;
            inv_vref = 1.0f / vmax;
        }
        const float factor = vscale * inv_vref * kPScale;

        V<f16>::x8 pf[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float most = -__builtin_inff();
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float x = s[rt][t][i] * kscale;
                    if (edge && group0 + 4 * t + i >= limit[rt]) x = -__builtin_inff();
                    s[rt][t][i] = x;
                    most = fmaxf(most, x);
                }
            most = fmaxf(most, __shfl_xor(most, 16, 64));
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            const float now = fmaxf(top[rt], most);
            const float base = now == -__builtin_inff() ? 0.0f : now;
            const float alpha = __builtin_amdgcn_exp2f(top[rt] - base);
            top[rt] = now;
            float add = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f(s[rt][t][i] - base);
                    add += e;
                    // A hidden key's weight is 0 whatever its block's scale.
                    const float w = edge && group0 + 4 * t + i >= limit[rt] ? 0.0f : e * factor;
                    pf[rt][t >> 1][4 * (t & 1) + i] = (f16)w;
                }
            sum[rt] = sum[rt] * alpha + add;
            const float keep = alpha * shrink;
            if (__any(keep != 1.0f)) {
#pragma unroll
                for (int d = 0; d < VT; ++d) acc[rt][d] *= keep;
            }
        }
        if (edge) {
            // Codes behind the context or of no block are not looked at.
            const int valid = idv_now < 0 ? 0 : min(max(r.ctx - group0, 0), 16);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int bytes = min(max(valid - 4 * k, 0), 4);
                const uint32_t mask = bytes == 4 ? 0xffffffffu : (1u << (8 * bytes)) - 1u;
#pragma unroll
                for (int d = 0; d < VT; ++d) vr[d][k] &= mask;
            }
        }
#pragma unroll
        for (int d = 0; d < VT; ++d)
            if (16 * d < D) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const auto a = Codes<f16, CT>::x8(vr[d][2 * h], vr[d][2 * h + 1]);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) acc[rt][d] = mfma16x16x32(a, pf[rt][h], acc[rt][d]);
                }
            }
        if (tile + 1 < t1) load_values(tile + 1, idv);
    }

    // Join the four wavefronts, 16 rows and OC columns at a time.
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        sum[rt] += __shfl_xor(sum[rt], 16, 64);
        sum[rt] += __shfl_xor(sum[rt], 32, 64);
        if (quarter == 0) {
            s_m[wave][16 * rt + m] = top[rt];
            s_l[wave][16 * rt + m] = sum[rt];
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int d0 = 0; d0 < DP; d0 += OC) {
            __syncthreads();
#pragma unroll
            for (int d = 0; d < OC / 16; ++d)
                *(f32x4*)&s_acc[wave][m][16 * d + 4 * quarter] =
                    acc[rt][d0 / 16 + d] * (1.0f / kPScale) * vref;
            __syncthreads();
            const int x = threadIdx.x >> 4, col = 8 * (threadIdx.x & 15);
            const int row = row0 + 16 * rt + x;
            if (row >= rows || col >= OC || d0 + col >= D) continue;
            float best = s_m[0][16 * rt + x];
#pragma unroll
            for (int w = 1; w < 4; ++w) best = fmaxf(best, s_m[w][16 * rt + x]);
            float l = 0.0f, o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float lw = s_l[w][16 * rt + x];
                if (lw == 0.0f) continue;
                const float f = __builtin_amdgcn_exp2f(s_m[w][16 * rt + x] - best);
                l += f * lw;
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] += f * s_acc[w][x][col + k];
            }
            const int i = row / p.G;
            const int64_t at = (int64_t)(r.q0 + i) * p.Hq + head * p.G + row % p.G;
            if (p.splits > 1) {
                if (d0 == 0 && col == 0) p.ml[at * p.splits + split] = make_float2(best, l);
                if (l != 0.0f) {
                    float* to = p.part + ((int64_t)split * p.tokens * p.Hq + at) * D + d0 + col;
                    *(f32x4*)to = (f32x4){o[0], o[1], o[2], o[3]};
                    *(f32x4*)(to + 4) = (f32x4){o[4], o[5], o[6], o[7]};
                }
                continue;
            }
            const bool none = reach(p, r, i) <= 0;
            Vec16<T> v;
#pragma unroll
            for (int k = 0; k < 8; ++k) v.v[k] = (T)(none ? 0.0f : o[k] / l);
            *(Vec16<T>*)((T*)p.out + at * D + d0 + col) = v;
            if (p.lse && d0 == 0 && col == 0)
                p.lse[(int64_t)(head * p.G + row % p.G) * p.tokens + r.q0 + i] =
                    none ? __builtin_inff() : (best + log2f(l)) * kLn2;
        }
}

// Joins the splits' partial results in order: 16 rows of one key head per
// workgroup, 8 columns a thread.
template <typename T> __global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p, int tiles16) {
    const int b = blockIdx.x / tiles16, head = blockIdx.y;
    const Request r = request(p, b);
    const int rows = min(r.n, p.max_q) * p.G;
    const int row = (blockIdx.x % tiles16) * 16 + (threadIdx.x >> 4);
    if (row >= rows) return;
    const int i = row / p.G;
    const int64_t at = (int64_t)(r.q0 + i) * p.Hq + head * p.G + row % p.G;
    const float2* ml = p.ml + at * p.splits;
    float best = -__builtin_inff();
    for (int s = 0; s < p.splits; ++s) best = fmaxf(best, ml[s].x);
    const bool none = reach(p, r, i) <= 0;
    for (int col = 8 * (threadIdx.x & 15); col < p.D; col += 128) {
        float l = 0.0f, o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < p.splits; ++s) {
            const float2 one = ml[s];
            if (one.y == 0.0f) continue;
            const float f = __builtin_amdgcn_exp2f(one.x - best);
            l += f * one.y;
            const float* from = p.part + ((int64_t)s * p.tokens * p.Hq + at) * p.D + col;
            const f32x4 x = *(const f32x4*)from, y = *(const f32x4*)(from + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[k] += f * x[k];
                o[4 + k] += f * y[k];
            }
        }
        Vec16<T> v;
#pragma unroll
        for (int k = 0; k < 8; ++k) v.v[k] = (T)(none ? 0.0f : o[k] / l);
        *(Vec16<T>*)((T*)p.out + at * p.D + col) = v;
        if (p.lse && col == 0)
            p.lse[(int64_t)(head * p.G + row % p.G) * p.tokens + r.q0 + i] =
                none ? __builtin_inff() : (best + log2f(l)) * kLn2;
    }
}

struct Plan {
    int rt, row_tiles, splits;
    int64_t bytes;
};

Plan plan(int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q, int64_t max_ctx) {
    Plan r;
    const int64_t rows = max_q * (Hq / Hkv);
    r.rt = rows <= 16 || D > 128 ? 1 : 2;
    r.row_tiles = (int)((rows + 16 * r.rt - 1) / (16 * r.rt));
    const int64_t groups = B * r.row_tiles * Hkv;
    const int64_t want = (4 * device_cu_count() + groups - 1) / (groups > 0 ? groups : 1);
    const int64_t most = (max_ctx + 255) / 256;  // a tile for each wavefront
    int64_t splits = want < most ? want : most;
    if (splits > kMaxSplits) splits = kMaxSplits;
    r.splits = splits > 1 ? (int)splits : 1;
    const int64_t n = tokens * Hq * r.splits;
    r.bytes = r.splits > 1 ? n * 8 + n * D * 4 : 0;
    return r;
}

template <typename T, int CT> void launch(const PagedParams& p, const Plan& w, hipStream_t s) {
    const dim3 grid((unsigned)(p.B * w.row_tiles), (unsigned)p.Hkv, (unsigned)w.splits);
    if (p.D <= 64) {
        if (w.rt == 1)
            paged_rows_kernel<T, CT, 64, 1><<<grid, 256, 0, s>>>(p);
        else
            paged_rows_kernel<T, CT, 64, 2><<<grid, 256, 0, s>>>(p);
    } else if (p.D <= 128) {
        if (w.rt == 1)
            paged_rows_kernel<T, CT, 128, 1><<<grid, 256, 0, s>>>(p);
        else
            paged_rows_kernel<T, CT, 128, 2><<<grid, 256, 0, s>>>(p);
    } else {
        paged_rows_kernel<T, CT, 256, 1><<<grid, 256, 0, s>>>(p);
    }
}

int check_shape(int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q, int64_t max_ctx) {
    KF_REQUIRE(tokens >= 0 && B >= 1 && Hq >= 1 && Hkv >= 1 && max_q >= 1 && max_ctx >= 0, KF_E_INVALID,
               "kf_paged_attention: bad shape");
    KF_REQUIRE(Hq % Hkv == 0, KF_E_INVALID, "kf_paged_attention: Hq must be a multiple of Hkv");
    KF_REQUIRE(D >= 16 && D <= 256 && D % 16 == 0, KF_E_INVALID,
               "kf_paged_attention: head dim must be a multiple of 16 <= 256");
    KF_REQUIRE(tokens <= INT32_MAX / 2 && B <= INT32_MAX / 2 && Hkv <= 65535 && Hq <= INT32_MAX / 2 &&
                   max_q * (Hq / Hkv) <= INT32_MAX / 2 && B * ((max_q * (Hq / Hkv) + 15) / 16) <= INT32_MAX / 2,
               KF_E_UNSUPPORTED, "kf_paged_attention: too many rows");
    return KF_OK;
}

}  // namespace
}  // namespace kf

extern "C" {

int64_t kf_paged_attention_workspace_bytes(int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                                           int64_t max_query_len, int64_t max_context_len) {
    using namespace kf;
    clear_error();
    if (check_shape(tokens, B, Hq, Hkv, D, max_query_len, max_context_len) != KF_OK) return -1;
    return plan(tokens, B, Hq, Hkv, D, max_query_len, max_context_len).bytes;
}

int kf_paged_attention(const void* q, const void* key_cache, const void* value_cache, const float* key_scale,
                       const float* value_scale, const int32_t* block_tables, const int32_t* context_lens,
                       const int32_t* query_starts, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                       int64_t tokens, int64_t B, int64_t blocks, int64_t table_width, int64_t Hq, int64_t Hkv,
                       int64_t D, int64_t block_tokens, int64_t q_token_stride, int64_t q_head_stride,
                       int64_t max_query_len, int64_t max_context_len, float scale, int causal, int clear_rest,
                       int dtype, int cache_dtype, kf_stream_t stream) {
    using namespace kf;
    clear_error();
    int rc = check_shape(tokens, B, Hq, Hkv, D, max_query_len, max_context_len);
    if (rc != KF_OK) return rc;
    const int shift = block_shift(block_tokens);
    KF_REQUIRE(shift > 0, KF_E_INVALID, "kf_paged_attention: block_tokens must be 16, 32, 64 or 128");
    KF_REQUIRE(blocks >= 1 && blocks <= INT32_MAX && table_width >= 1 && table_width <= INT32_MAX, KF_E_INVALID,
               "kf_paged_attention: the cache and the tables must hold a block");
    KF_REQUIRE(query_starts || tokens == B, KF_E_INVALID,
               "kf_paged_attention: without query_starts every request has one token");
    KF_REQUIRE(dtype == KF_F16 || dtype == KF_BF16, KF_E_INVALID, "kf_paged_attention: dtype must be f16 or bf16");
    KF_REQUIRE(cache_dtype == KF_CACHE_E4M3 || cache_dtype == KF_CACHE_INT8, KF_E_INVALID,
               "kf_paged_attention: bad cache dtype");
    KF_REQUIRE(scale > 0.0f && __builtin_isfinite(scale), KF_E_INVALID,
               "kf_paged_attention: scale must be finite and positive");
    if (tokens == 0) return KF_OK;
    KF_REQUIRE(q && key_cache && value_cache && key_scale && value_scale && block_tables && context_lens && out,
               KF_E_INVALID, "kf_paged_attention: null pointer");
    KF_REQUIRE(((uintptr_t)q | (uintptr_t)key_cache | (uintptr_t)value_cache | (uintptr_t)out | (uintptr_t)workspace) %
                           16 == 0 &&
                   (q_token_stride | q_head_stride) % 8 == 0,
               KF_E_INVALID, "kf_paged_attention: rows must be aligned to 16 bytes");
    const Plan w = plan(tokens, B, Hq, Hkv, D, max_query_len, max_context_len);
    KF_REQUIRE(w.bytes == 0 || (workspace && workspace_bytes >= w.bytes), KF_E_WORKSPACE,
               "kf_paged_attention: workspace of %lld bytes needed", (long long)w.bytes);
    PagedParams p;
    p.q = q;
    p.kc = (const uint8_t*)key_cache;
    p.vc = (const uint8_t*)value_cache;
    p.ks = key_scale;
    p.vs = value_scale;
    p.tables = block_tables;
    p.context = context_lens;
    p.starts = query_starts;
    p.out = out;
    p.lse = lse;
    p.part = (float*)workspace;
    p.ml = (float2*)((float*)workspace + tokens * Hq * w.splits * D);
    p.q_ts = q_token_stride;
    p.q_hs = q_head_stride;
    p.tokens = (int)tokens;
    p.B = (int)B;
    p.blocks = (int)blocks;
    p.width = (int)table_width;
    p.Hq = (int)Hq;
    p.Hkv = (int)Hkv;
    p.G = (int)(Hq / Hkv);
    p.D = (int)D;
    p.shift = shift;
    p.max_q = (int)max_query_len;
    p.row_tiles = w.row_tiles;
    p.splits = w.splits;
    p.c = scale * kLog2e;
    p.causal = causal != 0;
    p.clear_rest = clear_rest;
    const hipStream_t s = (hipStream_t)stream;
    const bool e4m3 = cache_dtype == KF_CACHE_E4M3;
    if (dtype == KF_BF16)
        e4m3 ? launch<bf16, KF_CACHE_E4M3>(p, w, s) : launch<bf16, KF_CACHE_INT8>(p, w, s);
    else
        e4m3 ? launch<f16, KF_CACHE_E4M3>(p, w, s) : launch<f16, KF_CACHE_INT8>(p, w, s);
    rc = check_launch("kf_paged_attention");
    if (rc != KF_OK || w.splits == 1) return rc;
    const int64_t tiles16 = (max_query_len * p.G + 15) / 16;
    const dim3 grid((unsigned)(B * tiles16), (unsigned)Hkv);
    if (dtype == KF_BF16)
        paged_join_kernel<bf16><<<grid, 256, 0, s>>>(p, (int)tiles16);
    else
        paged_join_kernel<f16><<<grid, 256, 0, s>>>(p, (int)tiles16);
    return check_launch("kf_paged_attention (join)");
}

// Where device integers lead (paged_common.h), on the host: for the tests.
int kfm_paged_block_of_group(const int32_t* table, int width, int blocks, int shift, int group) {
    return kf::block_of_group(table, width, blocks, shift, group);
}

int64_t kfm_paged_block_of_slot(int64_t slot, int64_t capacity, int shift) {
    return kf::block_of_slot(slot, capacity, shift);
}

// result: {first token, queries, context, keys the query sees}
void kfm_paged_request(const int32_t* starts, const int32_t* context, int b, int tokens, int query, int causal,
                       int32_t* result) {
    const kf::Request r = kf::request_at(starts, context, b, tokens);
    result[0] = r.q0;
    result[1] = r.n;
    result[2] = r.ctx;
    result[3] = kf::keys_seen(r, query, causal != 0);
}

}  // extern "C"
