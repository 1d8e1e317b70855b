// Attention over the paged cache: few rows of a request (decoding, drafts), and
// the entry point.
#include <type_traits>

#include "paged_attn.h"

namespace kf {
namespace {

constexpr float kPScale = 32768.0f;  // 2^15, the largest f16 operand of the second product

// ---------------------------------------------------------------------------
// Few rows: 16 * RT (query, head) rows of one key head are a unit of work, whose
// keys the 4 wavefronts of a workgroup split.
//
// A wavefront takes 16 * NT keys at a time.  S^T = K Q^T with K as the A
// operand: of tile t, row m' is the key 4 NT (m'/4) + 4 t + m'%4, so the D layout
// (column = row of Q = lane%16, rows 4*(lane/16)+i) leaves lane (row, quarter)
// with the scores of 4 NT consecutive keys, all of one 16-token group: one key
// scale and one value scale a lane, and exactly the B operand that
// O^T = V^T P^T wants when V^T's lane (column, quarter) holds the same tokens
// of its column, which are contiguous bytes of the value cache.  Nothing passes
// through LDS before a unit's end, and every load is 16 (NT = 2: 8 for values)
// bytes a lane.
//
// Bound by HBM, so the loop is built around the loads in flight: a wavefront
// asks for the next turn's keys as soon as the products have used the
// registers, for its values likewise, for its table entries a turn earlier, and
// goes on to its next unit's without a pause.  Measured: 32 requests of 8192
// keys, 8 key heads of 128 in e4m3 (537 MB), 106 us with the join, 5.1 TB/s,
// two requests of 100001 and 60000 keys (401 MB) 82 us, 4.9 TB/s; a pass costs 12 us
// besides 5.9 TB/s (starting, the last units, the join).
// ---------------------------------------------------------------------------
template <int DP, int RT> struct RowsShape {
    // 16-key tiles of a turn: what two wavefronts a SIMD have registers for.
    static constexpr int NT = DP * RT > 128 ? 2 : 4;
    static constexpr int KEYS = 16 * NT;            // keys a wavefront takes in a turn
    static constexpr int ROWS = 16 * RT;            // rows of a unit
    static constexpr int OC = DP < 128 ? DP : 128;  // columns joined at a time
};

// The work is a line of turns: for each request its units (row tile, key head),
// for each unit its keys in turns.  Every workgroup takes an equal share of the
// line, one round of workgroups for the GPU.  The device alone knows the
// lengths, so every workgroup sums the requests' turns for itself.  Requests of
// any mixture of lengths then end together.  Where the contexts are short
// (`aligned`) the line counts units and no unit is cut, so nothing is left to
// join.
struct Whole {
    int q0, n, ctx;  // request
    int row_tile, head;
    int parts, part;  // how many (0: there is no such unit), the first one's place
    int unused;
};
struct Shares {
    Partials to;  // two of a workgroup, its first and last segment's
    Whole* whole; // [workgroups]: the unit that begins there and does not end
    int least;    // turns of a workgroup at least
    bool aligned;
};

// A request's units and the steps of the line that each takes.
template <int KEYS, int ROWS>
__device__ __forceinline__ int2 steps_and_units(const PagedParams& p, const Request& r, bool aligned) {
    const int keys = keys_to_scan(p, r.ctx);
    // Requests of more rows are the prompts' kernel's.
    const int rows = (int64_t)r.n * p.G > p.few ? 0 : min(r.n, p.max_q) * p.G;
    return make_int2(aligned ? 1 : max((keys + KEYS - 1) / KEYS, 1), (rows + ROWS - 1) / ROWS * p.Hkv);
}

// a / b for b > 0; the 64-bit division only where it is needed (0.3 us of a
// workgroup's start each).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if ((a | b) >> 32 == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
    return a / b;
}

// A workgroup's stretch of one unit.
struct Segment {
    int b, q0, n, ctx;  // request
    int row_tile, head;
    int first, last;  // turns
    int part;         // where its partial result goes; -1: it is the whole unit
    int unit;
};
constexpr int kSegments = 64;  // of a workgroup at a time

template <int DP, int RT> struct RowsShared {
    float acc[4][16][RowsShape<DP, RT>::OC + 4];
    float m[4][16 * RT], l[4][16 * RT];
    Segment list[kSegments];
    int64_t sum[4], units[4];
    int64_t unit0, unit1, behind;  // global indexes of the share's first and last unit; the line behind the list
    Whole whole;
};

// Exclusive prefix sums over the workgroup's 4 wavefronts; *total their sum.
__device__ __forceinline__ int64_t prefix_of(int64_t mine, int64_t* scratch, int64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t incl = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t other = __shfl_up((long long)incl, off, 64);
        if (lane >= off) incl += other;
    }
    if (lane == 63) scratch[wave] = incl;
    __syncthreads();
    int64_t before = incl - mine, all = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (k < wave) before += scratch[k];
        all += scratch[k];
    }
    *total = uniform64(all);
    return before;
}

template <typename T, int CT, int DP, int RT, bool EXACT>
__global__ __launch_bounds__(256, 2) void paged_rows_kernel(PagedParams p, Shares w) {
    using Shape = RowsShape<DP, RT>;
    constexpr int NT = Shape::NT, KEYS = Shape::KEYS, ROWS = Shape::ROWS, OC = Shape::OC;
    constexpr int KC = DP / 64;  // 64-column chunks of a key row
    constexpr int VT = DP / 16;  // 16-column tiles of the output
    constexpr int PC = NT / 2;   // 32-key products of a turn
    __shared__ RowsShared<DP, RT> sh;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m = lane & 15, quarter = lane >> 4;
    const int D = EXACT ? DP : p.D;

    // This workgroup's share of the line.  Where no unit is cut and every request
    // has one token, all have the same number of units and a unit's request follows
    // by a division; else every workgroup sums over the requests.
    const bool uniform = w.aligned && !p.starts;
    const int units_each = steps_and_units<KEYS, ROWS>(p, Request{0, 1, 0}, true).y;
    const int per = (p.B + 255) / 256;
    const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
    // A thread's first request, most often its only one, stays in registers.
    Request r0{0, 0, 0};
    auto my_request = [&](int b) { return b == b0 ? r0 : request(p, b); };
    int64_t steps_before = 0, units_before = 0, total = (int64_t)p.B * units_each;
    if (!uniform) {
        r0 = request(p, min(b0, p.B - 1));
        int64_t my_steps = 0, my_units = 0, all_units;
        for (int b = b0; b < b1; ++b) {
            const int2 su = steps_and_units<KEYS, ROWS>(p, my_request(b), w.aligned);
            my_steps += (int64_t)su.x * su.y;
            my_units += su.y;
        }
        steps_before = prefix_of(my_steps, sh.sum, &total);
        units_before = prefix_of(my_units, sh.units, &all_units);
    }
    const int64_t share = max(quotient(total + gridDim.x - 1, gridDim.x), (int64_t)w.least);
    const int64_t begin = blockIdx.x * share, end = min(begin + share, total);
    if (p.starts) {  // tokens behind the last request
        const Request r = request(p, p.B - 1);
        fill_rows<T>(p, r.q0 + r.n + blockIdx.x, p.tokens, gridDim.x, 0, p.Hq, p.clear_rest, 0.0f, __builtin_inff());
    }
    if (tid == 0) sh.whole.parts = 0;

    const int subs = (1 << (p.shift - 4)) - 1;   // groups of a block - 1
    const int64_t unit_bytes = (int64_t)D << p.shift;  // a block's keys of one head
    const int kgroup = 4 * NT * (m >> 2), vgroup = 4 * NT * quarter;  // first key of this lane's in a turn
    typename V<T>::x8 qf[RT][KC][2];
    u32x4 kr[NT][KC];
    uint32_t vr[VT][NT];
    float ks = 0.0f, vs = 0.0f;
    auto load_queries = [&](const Segment& g) {
        const int rows = min(g.n, p.max_q) * p.G;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int row = g.row_tile * ROWS + 16 * rt + m, i = row / p.G;
            const T* q = (const T*)p.q + (int64_t)(g.q0 + i) * p.q_ts + (int64_t)(g.head * p.G + row % p.G) * p.q_hs;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = 64 * c + 16 * quarter + 8 * h;
                    u32x4 v = {0u, 0u, 0u, 0u};
                    if (row < rows && col < D) v = *(const u32x4*)(q + col);
                    qf[rt][c][h] = __builtin_bit_cast(typename V<T>::x8, v);
                }
        }
    };
    // A table entry is looked at only when its turn comes: a check right behind its
    // load would wait for every load issued before it, the next keys among them.
    auto entry_of = [&](int b, int key) {
        return entry_of_group(p.tables + (int64_t)b * p.width, p.width, p.shift, key >> 4);
    };
    auto block_of = [&](int id, int key) { return block_of_entry(id, p.width, p.blocks, p.shift, key >> 4); };
    auto load_keys = [&](int head, int turn, int idk, int idv) {
        const int64_t at = (int64_t)max(idv, 0) * p.Hkv + head;
        ks = p.ks[at];
        vs = p.vs[at];
        __builtin_amdgcn_sched_barrier(0);
        const int key = KEYS * turn + kgroup;
        const uint8_t* from = p.kc + ((int64_t)max(idk, 0) * p.Hkv + head) * unit_bytes +
                              (16 * ((key >> 4) & subs) + (key & 15) + (m & 3)) * D;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const int col = 64 * c + 16 * quarter;  // past D: any bytes, the query is 0 there
                kr[t][c] = *(const u32x4*)(from + 4 * t * D + (col < D ? col : 0));
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    auto load_values = [&](int head, int turn, int id) {
        const int key = KEYS * turn + vgroup;
        const uint8_t* from =
            p.vc + ((int64_t)max(id, 0) * p.Hkv + head) * unit_bytes + 16 * ((key >> 4) & subs) * D + (key & 15);
#pragma unroll
        for (int d = 0; d < VT; ++d) {
            const int col = 16 * d < D ? 16 * d : 0;  // past D: columns that are not written
            if constexpr (NT == 4) {
                const u32x4 v = *(const u32x4*)(from + (col + m) * 16);
#pragma unroll
                for (int k = 0; k < 4; ++k) vr[d][k] = v[k];
            } else {
                const u32x2 v = *(const u32x2*)(from + (col + m) * 16);
                vr[d][0] = v[0];
                vr[d][1] = v[1];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    auto segment_at = [&](int k) {
        Segment g = sh.list[k];
        int* x = (int*)&g;
#pragma unroll
        for (int e = 0; e < (int)(sizeof(Segment) / 4); ++e) x[e] = __builtin_amdgcn_readfirstlane(x[e]);
        return g;
    };
    // This wavefront's turns of a segment: a quarter of them.  One without a turn
    // of its own goes through the first with every key hidden.
    auto turns_of = [&](const Segment& g) {
        const int per_wave = (g.last - g.first + 3) >> 2, t0 = g.first + wave * per_wave;
        return t0 < g.last ? make_int2(t0, min(t0 + per_wave, g.last)) : make_int2(g.first, g.first + 1);
    };

    // Unit u of request b, its steps [x, y) of the line out of [unit_begin, unit_end).
    auto segment_of = [&](int b, const Request& r, int u, int64_t x, int64_t y, int64_t unit_begin, int64_t unit_end) {
        Segment g;
        g.b = b;
        g.q0 = r.q0;
        g.n = r.n;
        g.ctx = r.ctx;
        g.unit = u;
        g.row_tile = u / p.Hkv;
        g.head = u - g.row_tile * p.Hkv;
        const int rows = min(r.n, p.max_q) * p.G;
        const int sees = keys_to_scan(p, reach(p, r, (min((g.row_tile + 1) * ROWS, rows) - 1) / p.G));
        const int turns = (sees + KEYS - 1) / KEYS;
        g.first = w.aligned ? 0 : (int)(x - unit_begin);
        g.last = w.aligned ? turns : min((int)(y - unit_begin), turns);
        g.part = -1;
        if (x != unit_begin || y != unit_end) {
            g.part = 2 * blockIdx.x + (x == begin ? 0 : 1);
            if (x == unit_begin)
                sh.whole = Whole{r.q0, r.n, r.ctx, g.row_tile, g.head,
                                 (int)quotient(unit_end - 1, share) - (int)blockIdx.x + 1, g.part, 0};
        }
        return g;
    };

    for (int64_t from = begin; from < end;) {
        // The next segments of the share, in order.
        int count;
        __syncthreads();
        if (uniform) {
            count = (int)min(end - from, (int64_t)kSegments);
            if (tid < count) {
                const int64_t at = from + tid;
                const int b = (int)quotient(at, units_each);
                sh.list[tid] = segment_of(b, request(p, b), (int)(at - (int64_t)b * units_each), at, at + 1, at, at + 1);
            }
            if (tid == 0) sh.behind = from + count;
        } else {
            int64_t base = steps_before, unit_base = units_before;
            for (int b = b0; b < b1; ++b) {
                const int2 su = steps_and_units<KEYS, ROWS>(p, my_request(b), w.aligned);
                const int64_t after = base + (int64_t)su.x * su.y;
                if (from >= base && from < after) sh.unit0 = unit_base + quotient(from - base, su.x);
                if (end - 1 >= base && end - 1 < after) sh.unit1 = unit_base + quotient(end - 1 - base, su.x);
                base = after;
                unit_base += su.y;
            }
            __syncthreads();
            const int64_t unit0 = uniform64(sh.unit0), unit1 = uniform64(sh.unit1);
            count = (int)min(unit1 - unit0 + 1, (int64_t)kSegments);
            base = steps_before;
            unit_base = units_before;
            for (int b = b0; b < b1; ++b) {
                const Request r = my_request(b);
                const int2 su = steps_and_units<KEYS, ROWS>(p, r, w.aligned);
                const int u0 = (int)min(max(unit0 - unit_base, (int64_t)0), (int64_t)su.y);
                const int u1 = (int)max(min(unit0 + count - unit_base, (int64_t)su.y), (int64_t)0);
                for (int u = u0; u < u1; ++u) {
                    const int64_t unit_begin = base + (int64_t)u * su.x, unit_end = unit_begin + su.x;
                    const int64_t x = max(from, unit_begin), y = min(end, unit_end);
                    const int at = (int)(unit_base + u - unit0);
                    sh.list[at] = segment_of(b, r, u, x, y, unit_begin, unit_end);
                    if (at == count - 1) sh.behind = y;
                }
                base += (int64_t)su.x * su.y;
                unit_base += su.y;
            }
        }
        __syncthreads();
        from = uniform64(sh.behind);

        // The registers hold the keys and values of (cur, turn); next_id* are the
        // table entries of the turn behind it, of this segment or of the next.  The
        // loads of a turn are issued in one order everywhere (scales, keys, entries,
        // values) and whether or not there is a turn to come (the last one's are
        // repeated): a wait for the oldest of them then leaves the others in flight.
        Segment cur = segment_at(0), nxt = segment_at(min(1, count - 1));
        int2 turns = turns_of(cur), next_turns = turns_of(nxt);
        int turn = turns.x;
        int next_idk, next_idv;
        auto load_entries = [&](int b, int at) {
            next_idk = entry_of(b, KEYS * at + kgroup);
            next_idv = entry_of(b, KEYS * at + vgroup);
            __builtin_amdgcn_sched_barrier(0);
        };
        load_entries(cur.b, turn);
        load_queries(cur);
        int idk = block_of(next_idk, KEYS * turn + kgroup), idv = block_of(next_idv, KEYS * turn + vgroup);
        __builtin_amdgcn_sched_barrier(0);
        load_keys(cur.head, turn, idk, idv);
        load_entries(turn + 1 < turns.y ? cur.b : nxt.b, turn + 1 < turns.y ? turn + 1 : next_turns.x);
        load_values(cur.head, turn, idv);
        for (int k = 0; k < count; ++k) {
            const Request r{cur.q0, cur.n, cur.ctx};
            const Segment later = segment_at(min(k + 2, count - 1));
            const int2 later_turns = turns_of(later);
            const int row0 = cur.row_tile * ROWS, rows = min(r.n, p.max_q) * p.G;
            if (cur.row_tile == 0 && cur.first == 0 && r.n > p.max_q)
                fill_rows<T>(p, r.q0 + p.max_q, r.q0 + r.n, 1, cur.head * p.G, p.G, 3, __builtin_nanf(""),
                             __builtin_nanf(""));
            // This lane's rows (columns of S^T).
            const bool idle = cur.first + wave * ((cur.last - cur.first + 3) >> 2) >= cur.last;
            int limit[RT];
            f32x4 acc[RT][VT];
            float top[RT], sum[RT], vref = kLeastScale, inv_vref = 1.0f / kLeastScale;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int row = row0 + 16 * rt + m;
                limit[rt] = row < rows && !idle ? reach(p, r, row / p.G) : 0;
                top[rt] = -__builtin_inff();
                sum[rt] = 0.0f;
#pragma unroll
                for (int d = 0; d < VT; ++d) acc[rt][d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
            }
            const int all_see = idle ? 0 : reach(p, r, row0 / p.G);  // keys that every row sees

            for (; turn < turns.y; ++turn) {
                f32x4 s[RT][NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
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
                const int key0 = turn * KEYS + vgroup;  // position of this lane's first key
                const bool bad = idv < 0 && key0 < r.ctx;
                const bool edge = turn * KEYS + KEYS > all_see || __any(idv < 0);
                const float kscale = bad ? __builtin_nanf("") : ks * p.c;
                // Blocks behind the context say nothing; an infinite scale is a NaN, which
                // only the rows that see its block take on.
                const float vscale = idv < 0 || key0 >= r.ctx ? 0.0f : vs < __builtin_inff() ? vs : __builtin_nanf("");
                const int idv_now = idv;
                const bool same = turn + 1 < turns.y;
                const int then = same ? turn + 1 : next_turns.x, then_head = same ? cur.head : nxt.head;
                idk = block_of(next_idk, KEYS * then + kgroup);
                idv = block_of(next_idv, KEYS * then + vgroup);
                if (!same) load_queries(nxt);
                load_keys(then_head, then, idk, idv);
                {
                    const bool inside = turn + 2 < turns.y, behind = next_turns.x + 1 < next_turns.y;
                    load_entries(inside ? cur.b : same || behind ? nxt.b : later.b,
                                 inside ? turn + 2 : same ? next_turns.x : behind ? next_turns.x + 1 : later_turns.x);
                }

                // The largest value scale so far, the same on every lane.
                const float vmax = row_max4(vscale);
                float shrink = 1.0f;
                if (vmax > vref) {
                    shrink = vref / vmax;
                    vref = vmax;
                    inv_vref = 1.0f / vmax;
                }
                const float factor = vscale * inv_vref * kPScale;

                V<f16>::x8 pf[RT][PC];
                auto softmax = [&](auto at_edge) {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        float most = -__builtin_inff();
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float x = s[rt][t][i] * kscale;
                                if (decltype(at_edge)::value && key0 + 4 * t + i >= limit[rt]) x = -__builtin_inff();
                                s[rt][t][i] = x;
                                most = fmaxf(most, x);
                            }
                        most = row_max4(most);
                        const float now = fmaxf(top[rt], most);
                        const float ref = now == -__builtin_inff() ? 0.0f : now;
                        const float alpha = __builtin_amdgcn_exp2f(top[rt] - ref);
                        top[rt] = now;
                        float add = 0.0f;
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float e = __builtin_amdgcn_exp2f(s[rt][t][i] - ref);
                                add += e;
                                // A hidden key's weight is 0 whatever its block's scale.
                                const float x =
                                    decltype(at_edge)::value && key0 + 4 * t + i >= limit[rt] ? 0.0f : e * factor;
                                pf[rt][t >> 1][4 * (t & 1) + i] = (f16)x;
                            }
                        sum[rt] = sum[rt] * alpha + add;
                        const float keep = alpha * shrink;
                        // Always: a way around the products would keep two copies of them.
#pragma unroll
                        for (int d = 0; d < VT; ++d) acc[rt][d] *= keep;
                    }
                };
                if (edge)
                    softmax(std::true_type());
                else
                    softmax(std::false_type());
                // Codes behind the context or of no block are not looked at.
                const int valid = idv_now < 0 ? 0 : min(max(r.ctx - key0, 0), 4 * NT);
                uint32_t mask[NT];
#pragma unroll
                for (int e = 0; e < NT; ++e) {
                    const int bytes = min(max(valid - 4 * e, 0), 4);
                    mask[e] = bytes == 4 ? 0xffffffffu : (1u << (8 * bytes)) - 1u;
                }
#pragma unroll
                for (int d = 0; d < VT; ++d)
#pragma unroll
                    for (int h = 0; h < PC; ++h) {
                        const auto a = Codes<f16, CT>::x8(vr[d][2 * h] & mask[2 * h], vr[d][2 * h + 1] & mask[2 * h + 1]);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) acc[rt][d] = mfma16x16x32(a, pf[rt][h], acc[rt][d]);
                    }
                load_values(then_head, then, idv);
            }

            // Join the four wavefronts, 16 rows and OC columns at a time.
            __syncthreads();  // the segment before has read its sums
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                sum[rt] = row_sum4(sum[rt]);
                if (quarter == 0) {
                    sh.m[wave][16 * rt + m] = top[rt];
                    sh.l[wave][16 * rt + m] = sum[rt];
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int d0 = 0; d0 < DP; d0 += OC) {
                    if (rt + d0 > 0) __syncthreads();
#pragma unroll
                    for (int d = 0; d < OC / 16; ++d)
                        *(f32x4*)&sh.acc[wave][m][16 * d + 4 * quarter] = acc[rt][d0 / 16 + d] * (1.0f / kPScale) * vref;
                    __syncthreads();
                    const int x = tid >> 4, col = 8 * (tid & 15);
                    const int row = row0 + 16 * rt + x;
                    if (row >= rows || col >= OC || d0 + col >= D) continue;
                    float best = sh.m[0][16 * rt + x];
#pragma unroll
                    for (int k = 1; k < 4; ++k) best = fmaxf(best, sh.m[k][16 * rt + x]);
                    const float ref = best == -__builtin_inff() ? 0.0f : best;
                    float l = 0.0f, o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float lk = sh.l[k][16 * rt + x];
                        if (lk == 0.0f) continue;
                        const float f = __builtin_amdgcn_exp2f(sh.m[k][16 * rt + x] - ref);
                        l += f * lk;
#pragma unroll
                        for (int e = 0; e < 8; ++e) o[e] += f * sh.acc[k][x][col + e];
                    }
                    if (cur.part >= 0) {
                        const int64_t at = (int64_t)cur.part * ROWS + 16 * rt + x;
                        if (d0 == 0 && col == 0) w.to.ml[at] = make_float2(best, l);
                        float* to = w.to.o + at * D + d0 + col;
                        *(f32x4*)to = (f32x4){o[0], o[1], o[2], o[3]};
                        *(f32x4*)(to + 4) = (f32x4){o[4], o[5], o[6], o[7]};
                        continue;
                    }
                    const int i = row / p.G;
                    const int64_t at = (int64_t)(r.q0 + i) * p.Hq + cur.head * p.G + row % p.G;
                    const bool none = reach(p, r, i) <= 0;
                    Vec16<T> v;
#pragma unroll
                    for (int e = 0; e < 8; ++e) v.v[e] = (T)(none ? 0.0f : o[e] / l);
                    *(Vec16<T>*)((T*)p.out + at * D + d0 + col) = v;
                    if (p.lse && d0 == 0 && col == 0)
                        p.lse[(int64_t)(cur.head * p.G + row % p.G) * p.tokens + r.q0 + i] =
                            none ? __builtin_inff() : (best + log2f(l)) * kLn2;
                }
            cur = nxt;
            nxt = later;
            turns = next_turns;
            next_turns = later_turns;
            turn = turns.x;
        }
    }
    if (!w.aligned) {
        __syncthreads();
        if (tid == 0) w.whole[blockIdx.x] = sh.whole;
    }
}

// Joins the parts of the unit that begins in workgroup blockIdx.x's share: its
// own part and the first part of each workgroup behind it.  LANES threads hold a
// row's columns, eight each, and WAYS sets of them take every WAYS-th part; the
// sets meet in LDS.  The order of the additions follows from the lengths alone.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedParams p, Shares w, int unit_rows) {
    constexpr int WAYS = 128 / LANES;  // two rows a workgroup
    const Whole whole = w.whole[blockIdx.x];
    if (whole.parts == 0) return;
    const int tid = threadIdx.x, col = 8 * (tid % LANES), way = tid / LANES % WAYS;
    const int x = blockIdx.y * 2 + tid / 128;  // row of the unit
    const Request r{whole.q0, whole.n, whole.ctx};
    const int row = whole.row_tile * unit_rows + x;
    const bool live = row < min(r.n, p.max_q) * p.G && col < p.D;
    join_parts<T, LANES, WAYS>(
        p, w.to, live, way, col, whole.parts,
        [&](int k) { return (int64_t)(k == 0 ? whole.part : 2 * ((int)blockIdx.x + k)) * unit_rows + x; }, r,
        whole.head, row);
}

struct Plan {
    int rt, few;
    bool aligned;
    int64_t groups, bytes;  // of the few-rows kernel
    bool prompts;
    PromptPlan prompt;
};

// Requests of up to this many rows go to the few-rows kernel, which reads the
// keys once for each 32 of them and spreads them over the GPU.  The prompts'
// kernel takes 128 rows in about the time of any fewer (e4m3, us, few-rows kernel
// against prompts'; 32 requests of 500 to 8192 keys, 8 key heads of 128: 64 rows
// 142 against 279, 128 rows 240 against 303, 192 rows 341 against 311; one of
// 30000 keys: 128 rows 58 against 65, 192 rows 75 against 67; 16 of 500 to 4096,
// 2 heads of 256: 128 rows 66 against 73, 192 rows 88 against 75).
constexpr int kFewRows = 128;

Plan plan(int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q, int64_t max_ctx) {
    Plan r;
    int64_t rows = max_q * (Hq / Hkv);
    r.prompts = rows > kFewRows;
    r.few = r.prompts ? kFewRows : INT32_MAX;
    if (r.prompts) rows = kFewRows;
    r.rt = rows <= 16 || D > 128 ? 1 : 2;
    const int64_t units = B * ((rows + 16 * r.rt - 1) / (16 * r.rt)) * Hkv;
    // A second launch joins the parts of cut units (5 us).  Whole units take less
    // where the contexts are short (us, whole against cut): of one tile of rows and
    // a dim of 128, one request of 2000 keys 17.6 against 18.2, of 4000 27 against
    // 18, 64 of 2000 52 against 56, 128 of 500 to 4000 153 against 122; with two
    // tiles or a dim of 256 a turn takes longer: one request of 1000 keys 20.4
    // against 18.4, of 750 17.9 against 17.9, 16 of 1000 21 against 25.
    r.aligned = max_ctx <= (r.rt == 1 && D <= 128 ? 2048 : 1024);
    // One workgroup a CU streams fastest (two requests of 100000 keys, 16 units: 82
    // us against 86 with two, which fit); a second hides the ends of the first's
    // units where each workgroup may have several (32 requests of 500 to 8192 keys,
    // 256 units: 73 us against 77; 64 of 100 to 2048: 49 against 55).
    r.groups = device_cu_count() * (units >= device_cu_count() ? 2 : 1);
    if (r.aligned && units < r.groups) r.groups = units;
    r.bytes = r.aligned ? 0 : r.groups * (2 * 16 * r.rt * (D * 4 + 8) + sizeof(Whole));
    r.prompt.bytes = 0;
    if (r.prompts) r.prompt = prompt_plan(tokens, B, Hq, Hkv, D, max_ctx);
    return r;
}

template <typename T, int CT, int DP, int RT>
void launch_rows(const PagedParams& p, const Plan& w, const Shares& sh, hipStream_t s) {
    if (p.D == DP)
        paged_rows_kernel<T, CT, DP, RT, true><<<dim3((unsigned)w.groups), 256, 0, s>>>(p, sh);
    else
        paged_rows_kernel<T, CT, DP, RT, false><<<dim3((unsigned)w.groups), 256, 0, s>>>(p, sh);
}

template <typename T, int CT> void launch(const PagedParams& p, const Plan& w, const Shares& sh, hipStream_t s) {
    if (p.D <= 64)
        w.rt == 1 ? launch_rows<T, CT, 64, 1>(p, w, sh, s) : launch_rows<T, CT, 64, 2>(p, w, sh, s);
    else if (p.D <= 128)
        w.rt == 1 ? launch_rows<T, CT, 128, 1>(p, w, sh, s) : launch_rows<T, CT, 128, 2>(p, w, sh, s);
    else
        launch_rows<T, CT, 256, 1>(p, w, sh, s);
}

template <typename T> void launch_join(const PagedParams& p, const Plan& w, const Shares& sh, hipStream_t s) {
    const int unit_rows = 16 * w.rt;
    const int64_t most = (int64_t)p.max_q * p.G, rows = most < unit_rows ? most : unit_rows;
    const dim3 grid((unsigned)w.groups, (unsigned)((rows + 1) / 2));
    if (p.D <= 64)
        paged_join_kernel<T, 8><<<grid, 256, 0, s>>>(p, sh, unit_rows);
    else if (p.D <= 128)
        paged_join_kernel<T, 16><<<grid, 256, 0, s>>>(p, sh, unit_rows);
    else
        paged_join_kernel<T, 32><<<grid, 256, 0, s>>>(p, sh, unit_rows);
}

int check_shape(int64_t tokens, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q, int64_t max_ctx) {
    KF_REQUIRE(tokens >= 0 && B >= 1 && Hq >= 1 && Hkv >= 1 && max_q >= 1 && max_ctx >= 0, KF_E_INVALID,
               "kf_paged_attention: bad shape");
    KF_REQUIRE(Hq % Hkv == 0, KF_E_INVALID, "kf_paged_attention: Hq must be a multiple of Hkv");
    KF_REQUIRE(D >= 16 && D <= 256 && D % 16 == 0, KF_E_INVALID,
               "kf_paged_attention: head dim must be a multiple of 16 <= 256");
    KF_REQUIRE(tokens <= INT32_MAX / 2 && Hq <= INT32_MAX / 2 && B <= INT32_MAX / 2 && max_q <= INT32_MAX / 2 &&
                   tokens * Hq <= INT32_MAX / 2 && Hkv <= 65535 && max_q * (Hq / Hkv) <= INT32_MAX / 2,
               KF_E_UNSUPPORTED, "kf_paged_attention: too many rows");
    // The prompts' kernel has a workgroup for each of its units, and a launch holds
    // less than 2^32 threads.
    KF_REQUIRE(max_q * (Hq / Hkv) <= kFewRows || prompt_units(tokens, B, Hq, Hkv) < 1 << 23,
               KF_E_UNSUPPORTED, "kf_paged_attention: too many requests of many rows");
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
    const Plan w = plan(tokens, B, Hq, Hkv, D, max_query_len, max_context_len);
    return w.bytes > w.prompt.bytes ? w.bytes : w.prompt.bytes;
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
    // The two kernels run one after the other and share the workspace.
    const int64_t bytes = w.bytes > w.prompt.bytes ? w.bytes : w.prompt.bytes;
    KF_REQUIRE(bytes == 0 || (workspace && workspace_bytes >= bytes), KF_E_WORKSPACE,
               "kf_paged_attention: workspace of %lld bytes needed", (long long)bytes);
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
    p.few = w.few;
    p.c = scale * kLog2e;
    p.causal = causal != 0;
    p.clear_rest = clear_rest;
    Shares sh;
    sh.to.o = (float*)workspace;
    sh.to.ml = (float2*)(sh.to.o + w.groups * 2 * 16 * w.rt * D);
    sh.whole = (Whole*)(sh.to.ml + w.groups * 2 * 16 * w.rt);
    sh.least = w.aligned ? 1 : 4;  // a turn for each wavefront
    sh.aligned = w.aligned;
    const hipStream_t s = (hipStream_t)stream;
    const bool e4m3 = cache_dtype == KF_CACHE_E4M3;
    if (dtype == KF_BF16)
        e4m3 ? launch<bf16, KF_CACHE_E4M3>(p, w, sh, s) : launch<bf16, KF_CACHE_INT8>(p, w, sh, s);
    else
        e4m3 ? launch<f16, KF_CACHE_E4M3>(p, w, sh, s) : launch<f16, KF_CACHE_INT8>(p, w, sh, s);
    rc = check_launch("kf_paged_attention");
    if (rc != KF_OK) return rc;
    if (!w.aligned) {
        if (dtype == KF_BF16)
            launch_join<bf16>(p, w, sh, s);
        else
            launch_join<f16>(p, w, sh, s);
        rc = check_launch("kf_paged_attention (join)");
        if (rc != KF_OK) return rc;
    }
    return w.prompts ? launch_prompt(p, w.prompt, workspace, dtype, cache_dtype, s) : KF_OK;
}

// Where device integers lead (paged_common.h), on the host: for the tests.
int kfm_paged_block_of_group(const int32_t* table, int width, int blocks, int shift, int group) {
    return kf::block_of_entry(kf::entry_of_group(table, width, shift, group), width, blocks, shift, group);
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
