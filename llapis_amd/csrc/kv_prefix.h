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
// each (four of 16 at head size 512).  A wave forms S^T = K Q^T for its rows with Q^T in registers,
// keeps maximum, sum and P in its lanes, and adds O^T += V^T P^T: K's rows lie in LDS in the order that
// makes a lane's scores those of 8 consecutive keys, P's operand.  Rows of LDS are 16 bytes longer than their
// values, so that 16 rows' reads of a column meet every bank once.
//
// Bound by the issue of matrix and vector instructions, not by memory: 64 sequences of 32 heads of 128 (8 kv heads)
// behind 32768 tokens, bf16, are 34 GFLOP (52 with P in two parts) and 134 MB, and take 74 us, 465 TFLOP/s.  The
// VALU is busy for 52 % of the time and the matrix cores for 40; q8_0 (16 sequences behind each of three prefixes, 99 us)
// 52 and 53.  A third of the waves' cycles wait for an instruction to be issued, a third for memory, LDS or a barrier.
// What carries it, with what it measured there (the whole call):
//  - the workgroup's two halves work half a unit apart, one at products while the other forms P and
//    stages, so that a SIMD's matrix cores and VALU work at once: 142 to 119 us with the next two
//  - sums are products with ones, P is split in two instructions a pair (split_p), and sums and output are scaled anew
//    only when a row's maximum grows by more than P_SLACK
//  - loads from memory stay in flight over barriers, and none is under a condition, which would have all of them waited for
//  - a second tile of a wave's rows where one leaves rows over: the same 64 sequences 114 us, with one tile 120, 33 of
//    them 93 and 99 (q8_0 111 and 130); 32, whose 128 rows one tile of each wave holds, 91 with two and 76 with one
// One part of P would take 10 us off and add 2^-9 to the error of its weights: it keeps kv_attn.h's instead.
//
// Rounding is kv_attn.h's: fp32 scores, maxima and sums, 16-bit parts of q and p, a pair of p's bf16 parts good to 2^-17 (cut
// off instead of rounded they took as long and were good to 2^-16); q8_0 values are staged as an fp16 value and its
// exact remainder.  A row's maximum is rounded up to a whole number, in base 2: what it is taken from or scaled by is exact.
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
    int tiles;                                           // of 16 rows a wave
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

// Waves of a workgroup, keys of a unit, and the most tiles of 16 rows that a wave's 256
// registers (512 at head size 512, a wave a SIMD) hold the output, Q's parts and P's of
constexpr int kvp_waves(int hd) { return hd > 256 ? 4 : 8; }
constexpr int kvp_unit(bool q8, int hd) { return hd > (q8 ? 128 : 256) ? 32 : 64; }
constexpr int kvp_q_parts(bool half, int type) { return half ? (type == T_F32 ? 2 : 1) : (type == T_F32 ? 3 : type == T_F16 ? 2 : 1); }
constexpr int kvp_p_parts(bool half, int type) { return !half && type == T_F32 ? 3 : 2; }
constexpr int kvp_most_tiles(bool half, int type, int hd) {
    return hd / 4 + kvp_q_parts(half, type) * hd / 8 + 8 * kvp_p_parts(half, type) <= 64 ? 2 : 1;
}
// tiles of a wave for groups of `rows` rows: a second one where one a wave leaves rows over
constexpr int kvp_tiles(bool half, int type, int hd, int64_t rows) { return rows > 16 * kvp_waves(hd) ? kvp_most_tiles(half, type, hd) : 1; }

hipError_t launch_kv_prefix_f16(const KvPrefix & p, int head_dim, hipStream_t s);
hipError_t launch_kv_prefix_bf16(const KvPrefix & p, int head_dim, hipStream_t s);
hipError_t launch_kv_prefix_q8(const KvPrefix & p, int head_dim, hipStream_t s);

namespace dev {

// QT: the queries' type; 16-bit ones are one part, but for F16 in two BF16 parts
template <int CT, int QT, int HD, int TILES>
struct KvpShape {
    static constexpr bool HALF = CT != KV_BF16, Q8 = CT == KV_Q8, WIDE = QT == T_F32;
    static constexpr int PQ = kvp_q_parts(HALF, QT), PP = kvp_p_parts(HALF, QT);
    static constexpr int WAVES = kvp_waves(HD), WGT = 64 * WAVES, NT = TILES, ROWS = 16 * NT * WAVES;
    static constexpr int UNIT = kvp_unit(Q8, HD), NB = UNIT / 32, NK = UNIT / 16, NC = HD / 32, NV = HD / 16;
    static constexpr int KP = 2 * HD + 16, VP = 2 * UNIT + 16;           // bytes from a row of LDS to the next
    static constexpr bool TWO = WAVES == 8;                              // groups of waves
    // Where a unit's loads are issued: before its products, where these are the shorter half of its work (64 sequences
    // behind 32768 tokens, bf16: 77.5 to 73.6 us; fp32 queries over fp16 1 to 2 % of a call), else behind the
    // stores (Q8_0, 48 sequences: 122 us a call and 126; three parts of q at head size 256: 77 and 84)
    static constexpr bool LATE = !Q8 && PQ <= 2;
    static constexpr int BUFS = TWO ? 2 : 1, PARTS = Q8 ? 2 : 1;         // units in LDS; q8_0: values and remainders
    static constexpr int KB = UNIT * KP, VB = HD * VP;                   // bytes of a part of K, of V
    static constexpr int LDS = BUFS * PARTS * (KB + VB);
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

// split8 with fewer instructions: the remainder of an fp16 part is taken and rounded in one, a pair of bf16 parts
// rounded once
template <bool HALF, int PARTS>
__device__ __forceinline__ void split_p(const float (&x)[8], u4 (&out)[PARTS]) {
    if constexpr (HALF) {
        static_assert(PARTS == 2, "two fp16 parts");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const h2v h = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
            const uint32_t w = __builtin_bit_cast(uint32_t, h);
            uint32_t r;
            // x - h, rounded to fp16
            asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(x[2 * i]));
            asm("v_fma_mixhi_f16 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(r) : "v"(w), "v"(x[2 * i + 1]));
            out[0][i] = w;
            out[1][i] = r;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const b2v h = {(__bf16)a, (__bf16)b};
                uint32_t w = __builtin_bit_cast(uint32_t, h);
                out[p][i] = w;
                if (p + 1 < PARTS) {
                    asm("" : "+v"(w));                     // (else the low half is rounded once more, alone)
                    a -= __builtin_bit_cast(float, w << 16);
                    b -= __builtin_bit_cast(float, w & 0xFFFF0000u);
                }
            }
        }
    }
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

template <int CT, int QT, int HD, int TILES>
__global__ __launch_bounds__(64 * kvp_waves(HD), kvp_waves(HD) / 4) void k_kv_prefix(const KvPrefix p) {
    using Sh = KvpShape<CT, QT, HD, TILES>;
    constexpr bool HALF = Sh::HALF, Q8 = Sh::Q8;
    constexpr int PQ = Sh::PQ, PP = Sh::PP, NT = Sh::NT, NC = Sh::NC, NV = Sh::NV, NB = Sh::NB, NK = Sh::NK;
    constexpr int WAVES = Sh::WAVES, WGT = Sh::WGT, ROWS = Sh::ROWS, UNIT = Sh::UNIT, KP = Sh::KP, VP = Sh::VP, KB = Sh::KB, VB = Sh::VB;
    constexpr int BUFS = Sh::BUFS, PARTS = Sh::PARTS;
    constexpr bool TWO = Sh::TWO;
    constexpr int KPT = Sh::KPT, VPT = Sh::VPT, KL = Sh::KL;
    // log2 of p's scale, and how far a row's scores may pass the maximum that its sums are
    // taken against before these are scaled anew: p stays below 2^16, fp16's end
    constexpr float KV_P_SHIFT = HALF ? 15.0f : 0.0f, P_SHIFT = HALF ? 13.0f : 0.0f, P_SLACK = HALF ? 2.75f : 16.0f;
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int s_first[KVP_GROUPS + 1], s_eff[KVP_GROUPS], s_lead[KVP_GROUPS];
    __shared__ KvGroup s_plan[KVP_GROUPS];
    __shared__ int64_t s_part[2][WAVES];

    const int tid = threadIdx.x, lane = tid & 63, wave = same(tid >> 6);
    const int lm = lane & 15, lg = lane >> 4;
    const int page = 1 << p.page_shift, page_mask = page - 1, cap = p.b.max_pages << p.page_shift;

    // ---- the groups: their first sequence with new tokens, and what all of those have before them
    // (a thread's first sequence is read beside the groups)
    const SeqRows ahead_rows = tid < p.b.n_seq ? seq_rows(p.b, tid) : SeqRows{0, 0, 0};
    const int wanted = tid < p.n_group ? p.prefix[tid] : 0;
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
        const SeqRows r = s == tid ? ahead_rows : seq_rows(p.b, s);
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
        mine.eff = min(min(max(wanted, 0), s_eff[tid]), cap) & ~(align - 1);
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
    // (row starts that are not in order may give groups more rows than there are: nothing is attended of them then)
    const int n_steps = same(n_steps_all <= p.max_steps ? (int)n_steps_all : 0), n_runs = runs_of(p.runs, n_steps);
    if (blockIdx.x == 0 && tid == 0) p.total[0] = n_steps;
    // ---- the sequences without their prefix, a wave each; last, when their loads hold up nothing
    auto write_rest = [&]() {
        for (int s = blockIdx.x * WAVES + wave; s < p.b.n_seq; s += gridDim.x * WAVES) {
            const int g = same(group_of(s)), eff = g >= 0 ? same(s_plan[g].eff) : 0, len = min(max(p.b.lens[s], 0), 0x7FFFFFFF);
            const int32_t * from = p.b.table + s * p.b.table_stride;
            const int skip = eff >> p.page_shift;
            if (lane == 0) {
                p.lens[s] = len - min(eff, len);
                p.seq_group[s] = eff > 0 ? g : -1;
            }
            // entries to the end of the last unit that k_kv_attn asks for: it knows the table's end, but not
            // that the table begins at the prefix's, so that the last `skip` entries have no page
            const int n = (min(len - min(eff, len), cap) + kv_unit(HD)) / page + 1;
            for (int i = lane; i < min(n, p.b.max_pages); i += 64)
                p.table[(int64_t)s * p.b.max_pages + i] = i + skip < p.b.max_pages ? from[i + skip] : -1;
        }
    };
    // consecutive runs on one XCD: they read the same head's keys, for the next rows or further on
    const int run = (blockIdx.x & 7) * (p.runs >> 3) + (blockIdx.x >> 3);
    if (run >= n_runs) {
        write_rest();
        return;
    }
    const Runs runs(n_steps, n_runs);
    const int lo = same(runs.begin(run)), hi = same(runs.begin(run + 1));

    struct Piece {
        int g, head, tile, item, u0, n_u;
        const int32_t * row;                              // of the page table
        uint64_t part;                                    // a head's part of a page
    };
    // (what is the same in every lane is said to be: it stays in scalar registers)
    auto next_piece = [&](int & step, Piece & c) {
        while (step < hi) {
            // (groups without items have the next one's base)
            const int g = same(kvp_find(p.n_group, step, [&](int i) { return s_plan[i].base; }));
            const KvGroup & gr = s_plan[g];
            const int units = same(gr.units), each = item_steps(units), base = same(gr.base), tiles = (same(gr.rows) + ROWS - 1) / ROWS;
            const int i = same((step - base) / each), first = base + i * each;
            const int u0 = units_before(step - first), u1 = units_before(min(hi - first, each));
            step = same(min(hi, first + each));
            if (u1 <= u0) continue;
            c.g = g;
            c.head = same(i / tiles);
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
    auto has_page = [&](int x) { return (uint32_t)x < (uint32_t)p.n_pages; };
    constexpr int KC = Q8 ? HD / 16 : HD / 8;             // loads of a key's row
    constexpr int VO = Q8 ? UNIT / 16 : UNIT / 8;         // ... of a column
    struct Unit { const int32_t * row; uint64_t part; int key; };
    u4 kf[KPT], vf[VPT], vd[Q8 ? VPT : 1][2];
    uint32_t kd[Q8 ? KPT : 1];
    const uint8_t * k_at[KPT];                            // places of the K loads, and of their scales
    const uint16_t * kd_at[Q8 ? KPT : 1];
    auto place_k = [&](const Unit & u, const int (&pg)[KPT]) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int j = tid + WGT * i, kk = min(j / KC, UNIT - 1), c = j % KC, slot = (u.key + kk) & page_mask;
            const uint8_t * a = p.k + u.part + (uint64_t)(has_page(pg[i]) ? pg[i] : 0) * p.k_stride;
            k_at[i] = a + slot * HD * (Q8 ? 1 : 2) + 16 * c;
            if constexpr (Q8) kd_at[i] = (const uint16_t *)(a + page * HD) + (c / 2) * page + slot;
        }
    };
    auto load_k = [&]() {
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            kf[i] = *(const u4 *)k_at[i];
            if constexpr (Q8) kd[i] = *kd_at[i];
        }
    };
    auto load_v = [&](const Unit & u, int pg) {
        const uint8_t * a = p.v + u.part + (uint64_t)(has_page(pg) ? pg : 0) * p.v_stride;
        const int slot = (u.key + (tid % VO) * (Q8 ? 16 : 8)) & page_mask;
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
    const u4 zero = {0, 0, 0, 0};
    auto store_k = [&](uint8_t * to, uint32_t ok) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int j = tid + WGT * i, kk = j / KC, c = j % KC;
            if (KL % WGT && j >= KL) continue;
            // the key's row in LDS
            const int r = (kk & ~31) + 16 * ((kk >> 2) & 1) + ((kk & 31) >> 3) * 4 + (kk & 3);
            uint8_t * w = to + r * KP;
            if constexpr (Q8) {
                const uint32_t d = kd[i] | kd[i] << 16;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    u4 a, b;
                    times_scale(i8_to_half(u2{kf[i][2 * h], kf[i][2 * h + 1]}), u4{d, d, d, d}, a, b);
                    *(u4 *)(w + 32 * c + 16 * h) = ok >> i & 1 ? a : zero;
                    *(u4 *)(w + KB + 32 * c + 16 * h) = ok >> i & 1 ? b : zero;
                }
            } else {
                *(u4 *)(w + 16 * c) = ok >> i & 1 ? kf[i] : zero;
            }
        }
    };
    auto store_v = [&](uint8_t * to, bool ok) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int j = tid + WGT * i;
            if (KL % WGT && j >= KL) continue;
            uint8_t * w = to + (j / VO) * VP + (tid % VO) * (Q8 ? 32 : 16);
            if constexpr (Q8) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    u4 a, b;
                    times_scale(i8_to_half(u2{vf[i][2 * h], vf[i][2 * h + 1]}), vd[i][h], a, b);
                    *(u4 *)(w + 16 * h) = ok ? a : zero;
                    *(u4 *)(w + VB + 16 * h) = ok ? b : zero;
                }
            } else {
                *(u4 *)w = ok ? vf[i] : zero;
            }
        }
    };
    uint8_t * const lds_k = lds, * const lds_v = lds + BUFS * PARTS * KB;

    // ---- the staging of the run's units in their order: K of a unit and V of the one
    // before it are stored, the next of each loaded, and the pages behind them asked for.
    // Behind the last unit it goes on with that one, which nothing reads: a load that is not always
    // issued would have the others waited for.  For the same reason the pages are used before loads are issued
    int ahead = lo, ahead_unit = 0;
    Piece ahead_piece;
    ahead_piece.n_u = 0;
    Unit id_unit, k_unit;
    int id_k[KPT], id_v = 0, id_m = 0, v_page = 0;
    uint32_t k_ok = 0;
    bool v_ok = false;
    int k_buf = 0, v_buf = 0;
    uint64_t missing[3] = {0, 0, 0};                      // keys without a page: of the unit whose K was loaded last, and those before
    auto ask = [&]() {
        if (ahead_unit == ahead_piece.n_u) {
            Piece next;
            if (next_piece(ahead, next)) {
                ahead_piece = next;
                ahead_unit = 0;
            } else {
                --ahead_unit;
            }
        }
        id_unit = {ahead_piece.row, ahead_piece.part, (ahead_piece.u0 + ahead_unit++) * UNIT};
#pragma unroll
        for (int i = 0; i < KPT; ++i) id_k[i] = id_unit.row[(id_unit.key + min((tid + WGT * i) / KC, UNIT - 1)) >> p.page_shift];
        id_v = id_unit.row[(id_unit.key + (tid % VO) * (Q8 ? 16 : 8)) >> p.page_shift];
        id_m = id_unit.row[(id_unit.key + lane % UNIT) >> p.page_shift];
    };
    // the unit of the pages asked for last is the next whose K is loaded
    uint32_t next_ok = 0;
    int next_v = 0;
    auto take_pages = [&]() {
        missing[2] = missing[1];
        missing[1] = missing[0];
        missing[0] = ~__ballot(has_page(id_m)) & (~0ull >> (64 - UNIT));
        place_k(id_unit, id_k);
        next_ok = 0;
#pragma unroll
        for (int i = 0; i < KPT; ++i) next_ok |= (uint32_t)has_page(id_k[i]) << i;
        next_v = id_v;
    };
    auto load_next_k = [&]() {
        load_k();
        k_unit = id_unit;
        k_ok = next_ok;
        v_page = next_v;
    };
    constexpr bool LATE = Sh::LATE;
    auto load = [&]() {
        load_v(k_unit, v_page);
        v_ok = has_page(v_page);
        load_next_k();
        ask();
        if (LATE) __builtin_amdgcn_sched_barrier(0);
    };
    auto stage = [&](bool with_v) {
        take_pages();
        __builtin_amdgcn_sched_barrier(0);
        store_k(lds_k + k_buf * PARTS * KB, k_ok);
        k_buf = (k_buf + 1) % BUFS;
        if (with_v) {
            store_v(lds_v + v_buf * PARTS * VB, v_ok);
            v_buf = (v_buf + 1) % BUFS;
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!LATE) load();
    };
    // LDS is written and read as barriers order it; loads from memory stay in flight
    auto barrier = [&]() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

    // ---- a wave's rows
    u4 qf[PQ][NT][NC];
    f4v acc[NT][NV], sc[NT][NK];
    u4 part[NT][NB][PP];
    f4v sum[NT];                                          // of p, the same in each of its values
    float q_scale[NT], m[NT];
    auto load_q = [&](const Piece & c, int n_rows) {
        const int row0 = same(s_plan[c.g].row0);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            // (a row behind the last is the last again)
            const int r = min(16 * (wave + WAVES * nt) + lm, n_rows - 1), rr = c.tile * ROWS + r, tok = rr / p.group;
            const int64_t from = (int64_t)(row0 + tok) * p.q_stride + (int64_t)(c.head * p.group + rr - tok * p.group) * HD + 8 * lg;
            float qx[NC][8], amax = 0.0f;
#pragma unroll
            for (int c32 = 0; c32 < NC; ++c32) load8(p.q, QT, from + 32 * c32, qx[c32]);
#pragma unroll
            for (int c32 = 0; c32 < NC; ++c32) {
                if (HALF)
#pragma unroll
                    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(qx[c32][j]));
            }
            // (the scale's sign is q's: the largest product is then the largest score)
            const float sign = p.scale < 0.0f ? -1.0f : 1.0f;
            q_scale[nt] = fabsf(p.scale) * KV_LOG2E;
            int ex = 0;
            if (HALF) {
                // the row's largest to [2^13, 2^14): exact, and undone with the scale (0 and non-finite: left)
                amax = over_groups(amax, [](float a, float b) { return fmaxf(a, b); });
                ex = amax > 0.0f && amax < __builtin_inff() ? 14 - __builtin_amdgcn_frexp_expf(amax) : 0;
                q_scale[nt] = __builtin_ldexpf(q_scale[nt], -ex);
            }
            q_scale[nt] = fmaxf(q_scale[nt], 1.17549435e-38f);         // 0 times a masked score's -infinity is none
#pragma unroll
            for (int c32 = 0; c32 < NC; ++c32) {
#pragma unroll
                for (int j = 0; j < 8; ++j) qx[c32][j] = sign * (HALF ? __builtin_ldexpf(qx[c32][j], ex) : qx[c32][j]);
                u4 parts[PQ];
                split8<HALF, PQ>(qx[c32], parts);
#pragma unroll
                for (int q = 0; q < PQ; ++q) qf[q][nt][c32] = parts[q];
            }
            m[nt] = -__builtin_inff();
            sum[nt] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int v = 0; v < NV; ++v) acc[nt][v] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        }
    };
    // Each of the loops over a unit's operands in LDS has RING of them on their way.
    constexpr int RING = Q8 ? 2 : 4;
    auto scores = [&](const uint8_t * lk) {
        constexpr int N = NC * NK;
        u4 f[RING][PARTS];
        auto get = [&](int i) {
            const uint8_t * a = lk + (16 * (i % NK) + lm) * KP + 64 * (i / NK) + 16 * lg;
            f[i % RING][0] = *(const u4 *)a;
            if constexpr (Q8) f[i % RING][1] = *(const u4 *)(a + KB);
        };
#pragma unroll
        for (int i = 0; i < RING; ++i) get(i);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < NK; ++j) sc[nt][j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = i / NK, j = i % NK;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int q = 0; q < PQ; ++q) sc[nt][j] = mfma16<HALF>(f[i % RING][0], qf[q][nt][c], sc[nt][j]);
                if constexpr (Q8) sc[nt][j] = mfma16<HALF>(f[i % RING][1], qf[0][nt][c], sc[nt][j]);
            }
            if (i + RING < N) get(i + RING);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // the lane's scores 2 b + t are those of keys 32 b + 8 lg + 4 t + (0 .. 3)
    auto softmax = [&](uint64_t none) {
        if (none) {
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                const uint32_t bits = (uint32_t)(none >> (32 * (j >> 1) + 8 * lg + 4 * (j & 1)));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[nt][j][i] = bits >> i & 1 ? -__builtin_inff() : sc[nt][j][i];
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float top = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[nt][j][i]);
            top = over_groups(top, [](float a, float b) { return fmaxf(a, b); }) * q_scale[nt];
            if (__any(top > m[nt] + P_SLACK)) {
                // (a whole number: it and what it is added to are exact, and scaling by it is)
                const float now = fmaxf(m[nt], ceilf(top));
                const float f = now == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m[nt] - now);
                sum[nt] *= f;
#pragma unroll
                for (int v = 0; v < NV; ++v) acc[nt][v] *= f;
                m[nt] = now;
            }
            const float shift = P_SHIFT - (m[nt] == -__builtin_inff() ? 0.0f : m[nt]);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[nt][2 * b + (i >> 2)][i & 3], q_scale[nt], shift));
                split_p<HALF, PP>(x, part[nt][b]);
            }
        }
    };
    auto products = [&](const uint8_t * lv) {
        constexpr int N = NV * NB;
        // sums as products with ones: the matrix cores have the time, the VALU does not
        const uint32_t one = HALF ? 0x3C003C00u : 0x3F803F80u;
        u4 f[RING][PARTS];
        auto get = [&](int i) {
            const uint8_t * a = lv + (16 * (i / NB) + lm) * VP + 64 * (i % NB) + 16 * lg;
            f[i % RING][0] = *(const u4 *)a;
            if constexpr (Q8) f[i % RING][1] = *(const u4 *)(a + VB);
        };
#pragma unroll
        for (int i = 0; i < RING; ++i) get(i);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int q = 0; q < PP; ++q)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) sum[nt] = mfma16<HALF>(u4{one, one, one, one}, part[nt][b][q], sum[nt]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int v = i / NB, b = i % NB;
#pragma unroll
            for (int q = 0; q < PP; ++q)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[nt][v] = mfma16<HALF>(f[i % RING][0], part[nt][b][q], acc[nt][v]);
            if constexpr (Q8)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[nt][v] = mfma16<HALF>(f[i % RING][1], part[nt][b][0], acc[nt][v]);
            if (i + RING < N) get(i + RING);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto rows_of = [&](const Piece & c) { return min(same(s_plan[c.g].rows) - c.tile * ROWS, ROWS); };
    // the piece's part of the result
    auto write = [&](const Piece & c) {
        const int64_t slot = (int64_t)c.item + run;
        const int n_rows = rows_of(c);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = 16 * (wave + WAVES * nt) + lm;
            if (r >= n_rows || slot >= p.slots) continue;
            float * a = p.acc + (slot * ROWS + r) * HD;
#pragma unroll
            for (int v = 0; v < NV; ++v) *(f4v *)(a + 16 * v + 4 * lg) = acc[nt][v];
            if (lg == 0) {
                p.ml[(slot * ROWS + r) * 2] = m[nt] + (KV_P_SHIFT - P_SHIFT);      // as if its p had kv_attn.h's scale
                p.ml[(slot * ROWS + r) * 2 + 1] = sum[nt][0];
            }
        }
    };

    // ---- the units.  Half of the waves form products (of the last unit's P and V, of Q
    // and this unit's K) while the others, half a unit behind, form P and stage: a SIMD's two
    // waves keep its matrix cores and its VALU busy at once.  At the end of half step 2 u + 1
    // both have stored K of unit u + 1 and V of unit u: the first waves in that half step, the others
    // in the one before, and what lay in those places was read last before that.
    const bool second = TWO && same(wave >= WAVES / 2);
    Piece cur, past;
    int step = lo, unit = 0, i = 0;
    bool busy = false;                                    // the wave has rows
    bool more = next_piece(step, cur);
    if (!more) {
        write_rest();
        return;
    }
    ask();
    load_q(cur, rows_of(cur));                            // (its loads beside the pages')
    busy = same(16 * wave < rows_of(cur));
    take_pages();
    load_next_k();
    ask();
    stage(false);
    barrier();
    if (second) {
        if constexpr (LATE) load();
        stage(true);
        barrier();
    }
    for (;; ++unit) {
        if constexpr (LATE) load();
        if (unit > 0 && busy) products(lds_v + ((unit - 1) % BUFS) * PARTS * VB);
        if (i == 0 && unit > 0) {
            write(past);
            const int n_rows = rows_of(cur);
            load_q(cur, n_rows);
            busy = same(16 * wave < n_rows);
        }
        if (busy) {
            scores(lds_k + (unit % BUFS) * PARTS * KB);
        } else {                                          // (no old values to keep)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < NK; ++j) sc[nt][j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        }
        barrier();
        if (busy) {
            softmax(second ? missing[2] : missing[1]);
        } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int q = 0; q < PP; ++q) part[nt][b][q] = zero;
        }
        stage(true);
        if (++i == cur.n_u) {
            past = cur;
            more = next_piece(step, cur);
            i = 0;
        }
        barrier();
        if (!more) break;
    }
    if (busy) products(lds_v + (unit % BUFS) * PARTS * VB);
    write(past);
    write_rest();
    if (TWO && !second) barrier();                        // the other waves' last one
}

template <int CT, int QT, int HD, int TILES>
hipError_t launch_kv_prefix_tiles(const KvPrefix & p, hipStream_t s) {
    using Sh = KvpShape<CT, QT, HD, TILES>;
    hipLaunchKernelGGL((k_kv_prefix<CT, QT, HD, TILES>), dim3(p.runs), dim3(Sh::WGT), (Sh::LDS), s, p);
    return hipGetLastError();
}

template <int CT, int QT, int HD>
hipError_t launch_kv_prefix_one(const KvPrefix & p, hipStream_t s) {
    if constexpr (kvp_most_tiles(CT != KV_BF16, QT, HD) == 2)
        if (p.tiles == 2) return launch_kv_prefix_tiles<CT, QT, HD, 2>(p, s);
    return launch_kv_prefix_tiles<CT, QT, HD, 1>(p, s);
}

template <int CT, int QT>
hipError_t launch_kv_prefix_hd(const KvPrefix & p, int head_dim, hipStream_t s) {
    switch (head_dim) {
        case 64: return launch_kv_prefix_one<CT, QT, 64>(p, s);
        case 96: return launch_kv_prefix_one<CT, QT, 96>(p, s);
        case 128: return launch_kv_prefix_one<CT, QT, 128>(p, s);
        case 192: return launch_kv_prefix_one<CT, QT, 192>(p, s);
        case 256: return launch_kv_prefix_one<CT, QT, 256>(p, s);
        case 512: return launch_kv_prefix_one<CT, QT, 512>(p, s);
    }
    return hipErrorInvalidValue;
}

template <int CT>
hipError_t launch_kv_prefix_type(const KvPrefix & p, int head_dim, hipStream_t s) {
    if (p.type == T_F32) return launch_kv_prefix_hd<CT, T_F32>(p, head_dim, s);
    return p.type == T_F16 ? launch_kv_prefix_hd<CT, T_F16>(p, head_dim, s) : launch_kv_prefix_hd<CT, T_BF16>(p, head_dim, s);
}

}  // namespace dev
}  // namespace llapis
