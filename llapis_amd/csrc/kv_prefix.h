// kv_prefix.h -- attention over the prefix that the sequences of a group share (one
// instance per cache type, query type and head size; kv_prefix_*.hip).
//
// Work.  A group's rows are the query heads of all its sequences' new tokens; every row
// sees every key of the prefix.  An item is (group, kv head, tile of KvpShape::ROWS rows),
// its keys are units of UNIT, and the items' units lie in one line that the runs share
// out evenly, as in kv_attn.h; a run is a workgroup, as many as the card holds at once.
// Every piece writes its maximum, sum and unnormalised output, which k_kv_prefix_join
// adds to what kv_attn.h's kernel makes of the sequences' own keys.  For that kernel the
// sequences are written anew without the prefix: their lengths, and their page table's
// rows from the prefix's end on.
//
// A unit's K and V are staged in LDS once for all rows, eight waves with 16 or 32 rows
// each: loaded into registers while the unit before it is computed, written to the other
// half of LDS behind it, one barrier a unit.  A wave forms S^T = K Q^T for its rows with
// Q^T in registers, keeps maximum, sum and P in its lanes, and adds O^T += V^T P^T: K's rows lie in
// LDS in the order that makes a lane's scores those of 8 consecutive keys, P's operand.
// Rows of LDS are 16 bytes longer than their values, so that 16 rows' reads of a column
// meet every bank once.
//
// Rounding is kv_attn.h's: fp32 scores, maxima and sums, 16-bit parts of q and p; q8_0
// values are staged as an fp16 value and its exact remainder.
#pragma once

#include "kv_attn.h"

namespace llapis {

constexpr int KVP_GROUPS = 256;                         // groups of a call

struct KvPrefix {
    KvSeqs b;
    const uint8_t * k;
    const uint8_t * v;
    uint64_t k_stride, v_stride;
    int n_pages, page_shift, n_kv, group;
    float scale;
    int type;
    const void * q;
    int64_t q_stride;
    const int32_t * groups;                              // [n_group + 1] first sequences
    const int32_t * prefix;                              // [n_group] tokens
    int n_group;
    int runs, slots;
    int64_t max_steps;                                   // of the line, for row starts in order
    // the sequences without their prefixes
    int32_t * lens;                                      // [n_seq]
    int32_t * table;                                     // [n_seq][max_pages]
    // for the join: each sequence's group (-1: no prefix), a group's places in the line
    int32_t * seq_group;                                 // [n_seq]
    struct KvGroup * plan;                               // [n_group]
    int32_t * total;                                     // steps
    float * ml;                                          // [slots][ROWS][2]
    float * acc;                                         // [slots][ROWS][head_dim]
};

// a group's rows and place: steps from `base`, items from `item`
struct KvGroup { int32_t base, item, row0, rows, units, lead, eff, pad; };

// Rows of a wave and waves of a workgroup, by what 256 registers (512 at head size 512,
// a wave a SIMD) hold of the output, Q's parts and P's
constexpr int kvp_nt(int ct_half, int wide, int hd) { return hd <= 96 || (hd == 128 && (ct_half || !wide)) ? 2 : 1; }
constexpr int kvp_waves(int hd) { return hd > 256 ? 4 : 8; }
constexpr int kvp_unit(int hd) { return hd > 256 ? 32 : 64; }
constexpr int kvp_rows(int ct_half, int wide, int hd) { return 16 * kvp_nt(ct_half, wide, hd) * kvp_waves(hd); }

hipError_t launch_kv_prefix_f16(const KvPrefix & p, int head_dim, hipStream_t s);
hipError_t launch_kv_prefix_bf16(const KvPrefix & p, int head_dim, hipStream_t s);
hipError_t launch_kv_prefix_q8(const KvPrefix & p, int head_dim, hipStream_t s);

namespace dev {

template <int CT, bool WIDE, int HD>
struct KvpShape {
    static constexpr bool HALF = CT != KV_BF16, Q8 = CT == KV_Q8;
    static constexpr int PQ = HALF ? (WIDE ? 2 : 1) : (WIDE ? 3 : 2);
    static constexpr int PP = HALF ? 2 : (WIDE ? 3 : 2);
    static constexpr int WAVES = kvp_waves(HD), WGT = 64 * WAVES, NT = kvp_nt(HALF, WIDE, HD), ROWS = 16 * NT * WAVES;
    static constexpr int UNIT = kvp_unit(HD), NB = UNIT / 32, NK = UNIT / 16, NC = HD / 32, NV = HD / 16;
    static constexpr int KP = 2 * HD + 16, VP = 2 * UNIT + 16;           // bytes from a row of LDS to the next
    static constexpr int PART = UNIT * KP + HD * VP;                     // K and V of a unit
    static constexpr int LDS = 2 * PART;                                 // two units, q8_0: a unit's values and remainders
    // 16-byte loads of a thread
    static constexpr int KL = UNIT * HD / (Q8 ? 16 : 8), KPT = (KL + WGT - 1) / WGT, VPT = KPT;
};

// exclusive sums over the workgroup's threads in order, and the whole
template <int WAVES>
__device__ __forceinline__ int64_t kvp_scan(int64_t x, int64_t * s_part, int64_t & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t v = x;
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(v, o, 64);
        if (lane >= o) v += y;
    }
    if (lane == 63) s_part[wave] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) before += s_part[w];
        total += s_part[w];
    }
    return before + v - x;
}

// the last i < n with at[i] <= x, where at[0] <= x
template <class F>
__device__ __forceinline__ int kvp_find(int n, int x, F at) {
    int lo = 0;
    for (int hi = n; hi - lo > 1;) {
        const int mid = (lo + hi) >> 1;
        if (at(mid) <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <int CT, bool WIDE, int HD>
__global__ __launch_bounds__(64 * kvp_waves(HD), kvp_waves(HD) / 4) void k_kv_prefix(const KvPrefix p) {
    using Sh = KvpShape<CT, WIDE, HD>;
    constexpr bool HALF = Sh::HALF, Q8 = Sh::Q8;
    constexpr int PQ = Sh::PQ, PP = Sh::PP, NT = Sh::NT, NC = Sh::NC, NV = Sh::NV, NB = Sh::NB, NK = Sh::NK;
    constexpr int WAVES = Sh::WAVES, WGT = Sh::WGT, ROWS = Sh::ROWS, UNIT = Sh::UNIT, KP = Sh::KP, VP = Sh::VP, PART = Sh::PART;
    constexpr int KPT = Sh::KPT, VPT = Sh::VPT, KL = Sh::KL;
    constexpr float P_SHIFT = HALF ? 15.0f : 0.0f;                // log2 of p's scale
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int s_first[KVP_GROUPS + 1], s_eff[KVP_GROUPS], s_lead[KVP_GROUPS];
    __shared__ KvGroup s_plan[KVP_GROUPS];
    __shared__ int64_t s_part[2][WAVES];

    const int tid = threadIdx.x, lane = tid & 63, wave = same(tid >> 6);
    const int lm = lane & 15, lg = lane >> 4;
    const int page = 1 << p.page_shift, page_mask = page - 1, cap = p.b.max_pages << p.page_shift;
    const int type = WIDE ? (int)T_F32 : p.type;

    // ---- the groups: their first sequence with new tokens, and what all of those have before them
    for (int g = tid; g <= p.n_group; g += WGT) {
        s_first[g] = min(max(p.groups[g], 0), p.b.n_seq);
        if (g < p.n_group) {
            s_eff[g] = 0x7FFFFFFF;
            s_lead[g] = 0x7FFFFFFF;
        }
    }
    __syncthreads();
    auto group_of = [&](int s) {
        if (s < s_first[0]) return -1;
        const int g = kvp_find(p.n_group, s, [&](int i) { return s_first[i]; });
        return s < s_first[g + 1] ? g : -1;
    };
    for (int s = tid; s < p.b.n_seq; s += WGT) {
        const SeqRows r = seq_rows(p.b, s);
        const int g = r.n > 0 ? group_of(s) : -1;
        if (g >= 0) {
            atomicMin(&s_eff[g], max(r.len - r.n, 0));
            atomicMin(&s_lead[g], s);
        }
    }
    __syncthreads();
    // thread g counts group g
    KvGroup mine = {};
    int64_t steps = 0, items = 0, n_steps_all, n_items;
    if (tid < p.n_group && s_lead[tid] != 0x7FFFFFFF) {
        const int align = max(page, 64);
        mine.lead = s_lead[tid];
        mine.eff = min(min(max(p.prefix[tid], 0), s_eff[tid]), cap) & ~(align - 1);
        mine.units = mine.eff / UNIT;
        const int end = p.b.start ? p.b.start[s_first[tid + 1]] : s_first[tid + 1];
        mine.row0 = min(max(p.b.start ? p.b.start[s_first[tid]] : s_first[tid], 0), p.b.n_tokens);
        mine.rows = mine.eff > 0 ? max(min(end, p.b.n_tokens) - mine.row0, 0) * p.group : 0;
        items = (int64_t)((mine.rows + ROWS - 1) / ROWS) * p.n_kv;
        steps = items * item_steps(mine.units);
    }
    const int64_t base_step = kvp_scan<WAVES>(steps, s_part[0], n_steps_all), base_item = kvp_scan<WAVES>(items, s_part[1], n_items);
    if (tid < p.n_group) {
        mine.base = (int)base_step;
        mine.item = (int)base_item;
        s_plan[tid] = mine;
        if (blockIdx.x == 0) p.plan[tid] = mine;
    }
    __syncthreads();
    // (row starts that are not in order may give groups more rows than there are: no prefix then)
    const int n_steps = same(n_steps_all <= p.max_steps ? (int)n_steps_all : 0), n_runs = runs_of(p.runs, n_steps);
    if (blockIdx.x == 0 && tid == 0) p.total[0] = n_steps;
    // ---- the sequences without their prefix, a wave each
    for (int s = blockIdx.x * WAVES + wave; s < p.b.n_seq; s += gridDim.x * WAVES) {
        const int g = same(group_of(s)), eff = g >= 0 ? same(s_plan[g].eff) : 0, len = min(max(p.b.lens[s], 0), 0x7FFFFFFF);
        const int32_t * from = p.b.table + s * p.b.table_stride;
        const int skip = eff >> p.page_shift;
        if (lane == 0) {
            p.lens[s] = len - min(eff, len);
            p.seq_group[s] = eff > 0 ? g : -1;
        }
        // entries to the end of the last unit, which its loads ask for
        const int n = (min(len, cap) - min(eff, len) + kv_unit(HD)) / page + 1;
        for (int i = lane; i < min(n, p.b.max_pages); i += 64)
            p.table[(int64_t)s * p.b.max_pages + i] = i + skip < p.b.max_pages ? from[i + skip] : -1;
    }
    // consecutive runs on one XCD: they read the same head's keys, for the next rows or further on
    const int run = (blockIdx.x & 7) * (p.runs >> 3) + (blockIdx.x >> 3);
    if (run >= n_runs) return;
    const Runs runs(n_steps, n_runs);
    const int hi = runs.begin(run + 1);
    int step = runs.begin(run);

    struct Piece {
        int g, head, tile, item, u0, n_u;
        const int32_t * row;                              // of the page table
        uint64_t part;                                    // a head's part of a page
    };
    auto next_piece = [&](Piece & c) {
        while (step < hi) {
            // (groups without items have the next one's base)
            const int g = same(kvp_find(p.n_group, step, [&](int i) { return s_plan[i].base; }));
            const KvGroup & gr = s_plan[g];
            const int units = same(gr.units), each = item_steps(units), base = same(gr.base), tiles = (same(gr.rows) + ROWS - 1) / ROWS;
            const int i = (step - base) / each, first = base + i * each;
            const int u0 = units_before(step - first), u1 = units_before(min(hi - first, each));
            step = min(hi, first + each);
            if (u1 <= u0) continue;
            c.g = g;
            c.head = i / tiles;
            c.tile = i - c.head * tiles;
            c.item = same(gr.item) + i;
            c.u0 = u0;
            c.n_u = u1 - u0;
            c.row = p.b.table + same(gr.lead) * p.b.table_stride;
            c.part = (uint64_t)c.head * page * (Q8 ? HD + HD / 16 : 2 * HD);
            return true;
        }
        return false;
    };

    // ---- a unit's K and V, from memory to registers and from there to LDS
    u4 kf[KPT], vf[VPT];
    u4 vd[Q8 ? VPT : 1][2];
    uint32_t kd[Q8 ? KPT : 1];
    int k_pg[KPT], v_pg, m_pg;
    auto has_page = [&](int pg) { return (uint32_t)pg < (uint32_t)p.n_pages; };
    constexpr int KC = Q8 ? HD / 16 : HD / 8;             // loads of a key's row
    constexpr int VO = Q8 ? UNIT / 16 : UNIT / 8;         // ... of a column
    auto load_pages = [&](const int32_t * row, int key) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) k_pg[i] = row[(key + min((tid + WGT * i) / KC, UNIT - 1)) >> p.page_shift];
        v_pg = row[(key + (tid % VO) * (Q8 ? 16 : 8)) >> p.page_shift];
        m_pg = row[(key + lane % UNIT) >> p.page_shift];
    };
    auto load_unit = [&](uint64_t part, int key) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int j = tid + WGT * i, kk = min(j / KC, UNIT - 1), c = j % KC, slot = (key + kk) & page_mask;
            const uint8_t * a = p.k + part + (uint64_t)(has_page(k_pg[i]) ? k_pg[i] : 0) * p.k_stride;
            kf[i] = *(const u4 *)(a + slot * HD * (Q8 ? 1 : 2) + 16 * c);
            if constexpr (Q8) kd[i] = ((const uint16_t *)(a + page * HD))[(c / 2) * page + slot];
        }
        const uint8_t * a = p.v + part + (uint64_t)(has_page(v_pg) ? v_pg : 0) * p.v_stride;
        const int slot = (key + (tid % VO) * (Q8 ? 16 : 8)) & page_mask;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int col = min((tid + WGT * i) / VO, HD - 1);
            vf[i] = *(const u4 *)(a + (col * page + slot) * (Q8 ? 1 : 2));
            if constexpr (Q8) {
                const u4 * d = (const u4 *)(a + page * HD + ((col / 32) * page + slot) * 2);
                vd[i][0] = d[0];
                vd[i][1] = d[1];
            }
        }
    };
    // a key's row in LDS
    auto k_place = [&](int kk) { return (kk & ~31) + 16 * ((kk >> 2) & 1) + ((kk & 31) >> 3) * 4 + (kk & 3); };
    auto store_unit = [&](uint8_t * to) {
        const u4 zero = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int j = tid + WGT * i, kk = j / KC, c = j % KC;
            if (KL % WGT && j >= KL) continue;
            const bool ok = has_page(k_pg[i]);
            uint8_t * w = to + k_place(kk) * KP;
            if constexpr (Q8) {
                const uint32_t d = kd[i] | kd[i] << 16;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    u4 a, b;
                    times_scale(i8_to_half(u2{kf[i][2 * h], kf[i][2 * h + 1]}), u4{d, d, d, d}, a, b);
                    *(u4 *)(w + 32 * c + 16 * h) = ok ? a : zero;
                    *(u4 *)(w + PART + 32 * c + 16 * h) = ok ? b : zero;
                }
            } else {
                *(u4 *)(w + 16 * c) = ok ? kf[i] : zero;
            }
        }
        const bool ok = has_page(v_pg);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int j = tid + WGT * i, col = j / VO;
            if (KL % WGT && j >= KL) continue;
            uint8_t * w = to + UNIT * KP + col * VP + (tid % VO) * (Q8 ? 32 : 16);
            if constexpr (Q8) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    u4 a, b;
                    times_scale(i8_to_half(u2{vf[i][2 * h], vf[i][2 * h + 1]}), vd[i][h], a, b);
                    *(u4 *)(w + 16 * h) = ok ? a : zero;
                    *(u4 *)(w + PART + 16 * h) = ok ? b : zero;
                }
            } else {
                *(u4 *)w = ok ? vf[i] : zero;
            }
        }
    };

    Piece cur, then;
    if (!next_piece(cur)) return;
    load_pages(cur.row, cur.u0 * UNIT);
    load_unit(cur.part, cur.u0 * UNIT);
    store_unit(lds);
    uint64_t keys_ok = __ballot(has_page(m_pg));
    __syncthreads();
    int buf = 0;
    for (;;) {
        const KvGroup & gr = s_plan[cur.g];
        const int n_rows = min(same(gr.rows) - cur.tile * ROWS, ROWS), row0 = same(gr.row0);
        // ---- the wave's queries as B operands: 16 rows from 16 (wave + WAVES nt) on
        u4 qf[PQ][NT][NC];
        float q_scale[NT], m[NT], l[NT];
        f4v acc[NT][NV];
        const int n_pq = !HALF && !WIDE && type == T_BF16 ? 1 : PQ;    // bf16 queries are one part
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = 16 * (wave + WAVES * nt) + lm, rr = cur.tile * ROWS + r, tok = rr / p.group;
            const int64_t from = (int64_t)(row0 + tok) * p.q_stride + (int64_t)(cur.head * p.group + rr - tok * p.group) * HD + 8 * lg;
            float qx[NC][8], amax = 0.0f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
#pragma unroll
                for (int j = 0; j < 8; ++j) qx[c][j] = 0.0f;
                if (r < n_rows) load8(p.q, type, from + 32 * c, qx[c]);
                if (HALF)
#pragma unroll
                    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(qx[c][j]));
            }
            q_scale[nt] = p.scale * KV_LOG2E;
            int ex = 0;
            if (HALF) {
                // the row's largest to [2^13, 2^14): exact, and undone with the scale (0 and non-finite: left)
                amax = over_groups(amax, [](float a, float b) { return fmaxf(a, b); });
                ex = amax > 0.0f && amax < __builtin_inff() ? 14 - __builtin_amdgcn_frexp_expf(amax) : 0;
                q_scale[nt] = __builtin_ldexpf(q_scale[nt], -ex);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if (HALF)
#pragma unroll
                    for (int j = 0; j < 8; ++j) qx[c][j] = __builtin_ldexpf(qx[c][j], ex);
                u4 part[PQ];
                split8<HALF, PQ>(qx[c], part);
#pragma unroll
                for (int q = 0; q < PQ; ++q) qf[q][nt][c] = part[q];
            }
            m[nt] = -__builtin_inff();
            l[nt] = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v) acc[nt][v] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const bool more = next_piece(then);
        const int key_begin = cur.u0 * UNIT, key_end = key_begin + cur.n_u * UNIT;
        const bool busy = 16 * wave < n_rows;
        for (int key = key_begin; key < key_end; key += UNIT) {
            const bool last = key + UNIT >= key_end, ahead = !last || more;
            const int next = last ? then.u0 * UNIT : key + UNIT;
            const uint64_t ok = keys_ok;
            if (ahead) {
                load_pages(last ? then.row : cur.row, next);
                load_unit(last ? then.part : cur.part, next);
            }
            const uint8_t * lk = lds + (Q8 ? 0 : buf * PART), * lv = lk + UNIT * KP;
            if (busy) {
                // ---- S^T of the wave's rows
                f4v sc[NT][NK];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < NK; ++j) sc[nt][j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int j = 0; j < NK; ++j) {
                        const uint8_t * a = lk + (16 * j + lm) * KP + 64 * c + 16 * lg;
                        const u4 k = *(const u4 *)a;
                        u4 k_lo;
                        if constexpr (Q8) k_lo = *(const u4 *)(a + PART);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int q = 0; q < PQ; ++q)
                                if (q < 1 || q < n_pq) sc[nt][j] = mfma16<HALF>(k, qf[q][nt][c], sc[nt][j]);
                            if constexpr (Q8) sc[nt][j] = mfma16<HALF>(k_lo, qf[0][nt][c], sc[nt][j]);
                        }
                    }
                // ---- softmax: the lane's scores 2 b + t are those of keys 32 b + 8 lg + 4 t + (0 .. 3)
                u4 part[NT][NB][PP];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float top = -__builtin_inff();
#pragma unroll
                    for (int j = 0; j < NK; ++j) {
                        sc[nt][j] *= q_scale[nt];
                        if (~ok & (~0ull >> (64 - UNIT))) {
                            const uint32_t bits = (uint32_t)(ok >> (32 * (j >> 1) + 8 * lg + 4 * (j & 1)));
#pragma unroll
                            for (int i = 0; i < 4; ++i) sc[nt][j][i] = bits >> i & 1 ? sc[nt][j][i] : -__builtin_inff();
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[nt][j][i]);
                    }
                    const float now = fmaxf(m[nt], over_groups(top, [](float a, float b) { return fmaxf(a, b); }));
                    const float ref = now == -__builtin_inff() ? 0.0f : now;
                    if (__any(now != m[nt])) {
                        const float f = __builtin_amdgcn_exp2f(m[nt] - ref);
                        l[nt] *= f;
#pragma unroll
                        for (int v = 0; v < NV; ++v) acc[nt][v] *= f;
                        m[nt] = now;
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            x[i] = __builtin_amdgcn_exp2f(sc[nt][2 * b + (i >> 2)][i & 3] - (ref - P_SHIFT));
                            l[nt] += x[i];
                        }
                        split8<HALF, PP>(x, part[nt][b]);
                    }
                }
                // ---- O^T
#pragma unroll
                for (int v = 0; v < NV; ++v)
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint8_t * a = lv + (16 * v + lm) * VP + 64 * b + 16 * lg;
                        const u4 hi_v = *(const u4 *)a;
                        u4 lo_v;
                        if constexpr (Q8) lo_v = *(const u4 *)(a + PART);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int q = 0; q < PP; ++q) acc[nt][v] = mfma16<HALF>(hi_v, part[nt][b][q], acc[nt][v]);
                            if constexpr (Q8) acc[nt][v] = mfma16<HALF>(lo_v, part[nt][b][0], acc[nt][v]);
                        }
                    }
            }
            if (Q8) __syncthreads();                      // the one unit in LDS has been read
            if (ahead) {
                store_unit(lds + (Q8 ? 0 : (buf ^ 1) * PART));
                keys_ok = __ballot(has_page(m_pg));
            }
            __syncthreads();
            buf ^= 1;
        }
        // ---- the piece's part of the result
        const int64_t slot = (int64_t)cur.item + run;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float sum = over_groups(l[nt], [](float a, float b) { return a + b; });
            const int r = 16 * (wave + WAVES * nt) + lm;
            if (r >= n_rows || slot >= p.slots) continue;
            float * a = p.acc + (slot * ROWS + r) * HD;
#pragma unroll
            for (int v = 0; v < NV; ++v) *(f4v *)(a + 16 * v + 4 * lg) = acc[nt][v];
            if (lg == 0) {
                p.ml[(slot * ROWS + r) * 2] = m[nt];
                p.ml[(slot * ROWS + r) * 2 + 1] = sum;
            }
        }
        if (!more) return;
        cur = then;
    }
}

template <int CT, bool WIDE, int HD>
hipError_t launch_kv_prefix_one(const KvPrefix & p, hipStream_t s) {
    using Sh = KvpShape<CT, WIDE, HD>;
    hipLaunchKernelGGL((k_kv_prefix<CT, WIDE, HD>), dim3(p.runs), dim3(Sh::WGT), (Sh::LDS), s, p);
    return hipGetLastError();
}

template <int CT, bool WIDE>
hipError_t launch_kv_prefix_hd(const KvPrefix & p, int head_dim, hipStream_t s) {
    switch (head_dim) {
        case 64: return launch_kv_prefix_one<CT, WIDE, 64>(p, s);
        case 96: return launch_kv_prefix_one<CT, WIDE, 96>(p, s);
        case 128: return launch_kv_prefix_one<CT, WIDE, 128>(p, s);
        case 192: return launch_kv_prefix_one<CT, WIDE, 192>(p, s);
        case 256: return launch_kv_prefix_one<CT, WIDE, 256>(p, s);
        case 512: return launch_kv_prefix_one<CT, WIDE, 512>(p, s);
    }
    return hipErrorInvalidValue;
}

template <int CT>
hipError_t launch_kv_prefix_type(const KvPrefix & p, int head_dim, hipStream_t s) {
    return p.type == T_F32 ? launch_kv_prefix_hd<CT, true>(p, head_dim, s) : launch_kv_prefix_hd<CT, false>(p, head_dim, s);
}

}  // namespace dev
}  // namespace llapis
