// kv_attn.h -- attention of new tokens over the paged cache, the kernel (one
// instance per cache type, query type, head size and row tiles; kv_attn_*.hip).
//
// Work.  A sequence's keys are units of 128 or 64; an item is (sequence, kv
// head).  The items' units lie in one line, of which every run of workgroups
// takes an equal part: long and short sequences share the card alike, and no
// count of splits has to be chosen.  A workgroup holds the kv head's query heads
// of every new token, up to 32 rows, and reads K and V once for all of them; more
// rows are tiles of 32 in workgroups of the same run, eight apart and so on one
// XCD, where they walk the same keys at the same time.  (Tiles of 16 in two
// workgroups instead of 32 in one measured 3.6 against 5.3 TB/s at head size 128:
// they do not stay close enough for the L2.)  A run that covers an item writes
// its result; parts of an item go to the workspace as (maximum, sum, unnormalised
// output) and k_kv_join adds them.  The split is a function of the lengths alone.
//
// A workgroup's waves take a unit together.  For its 32 (16) keys a wave forms
//   S^T = K Q^T     A = K (16 keys x 32 values), B = Q^T from LDS
// and with the row maxima of all waves its P, which goes to LDS; for its share
// of the values' columns and all keys of the unit it then adds
//   O^T += V^T P^T  A = V^T (16 values x 32 keys), B = P^T
// (v_mfma_f32_16x16x32).  A lane's column is query row l % 16 in both products,
// so the running maximum, the sum and the rescaling stay in the lane, and P is
// written as it is read: K's rows are assigned to the first product such that a
// lane's scores belong to the keys that are consecutive in its V^T operand.  K
// and V go from memory to the operands' registers, each once in the workgroup:
// V is loaded ahead of the unit's first product, the next unit's K behind it.
//
// Rounding.  Scores, maxima and sums are fp32.  The products take 16-bit
// operands: the cache's values are exact in them; q and p are split into parts
// whose sum is the fp32 value to 2^-22 (two fp16 parts) or 2^-24 (three bf16
// parts).  16-bit queries are exact in one fp16 or two bf16 parts, and their p in
// two bf16 parts (2^-17) is far below out's rounding.  fp16 parts keep their
// exponent range by powers of two: q's row is scaled to a maximum in [2^13,
// 2^14), p by 2^15.  q8_0: an
// int8 value times its scale is exact in two fp16 parts (18 bits), K's and V's alike
// for results of every type: fp16's 11 bits alone would be rounded a second time
// where one key carries a row.  Past 65504 the first part is infinite and the second
// of the other sign, so that such a value is NaN (a remainder kept finite takes two
// more instructions for two values, 7 % of a long cache's time, and sums of its own
// for the remainders 2.5 % and spilled registers at three head sizes).
//
// q8_0's loads are 16 bytes a lane too: of a K row the lane's 16 values go to two
// products, and of a V column 16 keys, so that the products' order of values and
// of keys is another (Q and P are laid out to it).
//
// What bounds it.  Long caches: memory.  TB/s of K and V (a kernel that only reads
// reaches 6.2): head size 64 5.5, 128 5.6 (pages of 16 tokens 5.4), 256 5.4, 512
// 5.3; with two row tiles 5.3, at 512 4.5; q8_0 4.8 to 5.2, at 512 4.65 (its
// conversions keep the VALU busy for 60 % of the time).  Short ones: the chain of
// lengths, page table, K, scores, V, result, each a memory latency: 7.6 us for 700
// keys, and 24.6 us for 11203 keys of head size 512, of which a workgroup's unit is
// 256 KB.  What the choices were worth, and cost (us of the kernel):
//   the line in half units, a half for each piece    48 ragged sequences   49 -> 45
//   eight waves instead of four at head size 512     11203 keys            29 -> 25
//   q8_0: two fp16 parts instead of three bf16       2 x 131072 keys     203 -> 172
//   q8_0: 16-byte loads instead of 8                                     172 -> 118
//   q8_0: V's second part for 16-bit results too, all else as it is      107 -> 116
// As many runs as the card holds at once are enough: twice or three times as many
// took 129 and 142 us instead of 124 for the 131072 keys.  Units are not parted
// between runs: ends at a half of one (a quarter) took 55 to 59 (65) us instead of 53
// for the 48 sequences with their join, since what a part of a unit costs is its chain
// of latencies.
#pragma once

#include <type_traits>

#include "kv.h"

namespace llapis {
namespace dev {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef float f2v __attribute__((ext_vector_type(2)));

enum { KV_F16 = 0, KV_BF16 = 1, KV_Q8 = 2 };

template <bool HALF>
__device__ __forceinline__ f4v mfma16(u4 a, u4 b, f4v c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8v, a), __builtin_bit_cast(h8v, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}

// eight fp32 values as PARTS 16-bit operands whose sum they are
template <bool HALF, int PARTS>
__device__ __forceinline__ void split8(const float (&x)[8], u4 (&out)[PARTS]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            if constexpr (HALF) {
                const h2v h = {(_Float16)a, (_Float16)b};
                out[p][i] = __builtin_bit_cast(uint32_t, h);
                if (p + 1 < PARTS) { a -= (float)h[0]; b -= (float)h[1]; }
            } else {
                const b2v h = {(__bf16)a, (__bf16)b};
                const uint32_t w = __builtin_bit_cast(uint32_t, h);
                out[p][i] = w;
                if (p + 1 < PARTS) {
                    a -= __builtin_bit_cast(float, w << 16);
                    b -= __builtin_bit_cast(float, w & 0xFFFF0000u);
                }
            }
        }
    }
}

// eight int8 values as fp16: 1024 + (q + 128) by its bits, less 1152
__device__ __forceinline__ u4 i8_to_half(u2 q) {
    u4 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t w = q[i] ^ 0x80808080u;
        const h2v off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        const h2v a = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
        const h2v b = __builtin_bit_cast(h2v, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
        r[2 * i] = __builtin_bit_cast(uint32_t, a);
        r[2 * i + 1] = __builtin_bit_cast(uint32_t, b);
    }
    return r;
}

// int8 values (as fp16) times their scales: the product's rounding and what it leaves
__device__ __forceinline__ void times_scale(u4 q, u4 d, u4 & hi, u4 & lo) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2v a = __builtin_bit_cast(h2v, (uint32_t)q[i]), b = __builtin_bit_cast(h2v, (uint32_t)d[i]);
        const h2v p = a * b;
        hi[i] = __builtin_bit_cast(uint32_t, p);
        lo[i] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(a, b, -p));
    }
}

// the value of lane l ^ 16 / l ^ 32 combined with this lane's
template <class F>
__device__ __forceinline__ float over_groups(float x, F f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = f(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    const uint32_t w = __builtin_bit_cast(uint32_t, x);
    const auto c = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return f(__builtin_bit_cast(float, (uint32_t)c[0]), __builtin_bit_cast(float, (uint32_t)c[1]));
}

__device__ __forceinline__ void load8(const void * p, int type, int64_t at, float (&x)[8]) {
    if (type == T_F32) {
        const f4v * f = (const f4v *)((const float *)p + at);
        const f4v a = f[0], b = f[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
    } else {
        const u4 w = *(const u4 *)((const uint16_t *)p + at);
        if (type == T_F16) {
            const h8v h = __builtin_bit_cast(h8v, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                x[i] = __builtin_bit_cast(float, (i & 1) ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
        }
    }
}

__device__ __forceinline__ void store4(void * p, int type, int64_t at, f4v x) {
    if (type == T_F32) {
        *(f4v *)((float *)p + at) = x;
    } else {
        u2 w;
        if (type == T_F16) {
            const h2v a = {(_Float16)x[0], (_Float16)x[1]}, b = {(_Float16)x[2], (_Float16)x[3]};
            w = u2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
        } else {
            const b2v a = {(__bf16)x[0], (__bf16)x[1]}, b = {(__bf16)x[2], (__bf16)x[3]};
            w = u2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
        }
        *(u2 *)((uint16_t *)p + at) = w;
    }
}

// a sequence's keys as its items see them
struct SeqUnits {
    SeqRows r;
    int k0, kend;          // keys [k0, kend), k0 a multiple of KV_BLOCK
    int units;             // of an item
};

__device__ __forceinline__ SeqUnits seq_units(const KvSeqs & b, int s, int page_shift, int window, int unit) {
    SeqUnits u;
    u.r = seq_rows(b, s);
    u.kend = min(u.r.len, b.max_pages << page_shift);
    u.k0 = window > 0 ? min(max(u.r.len - u.r.n - window + 1, 0), u.kend) & ~(KV_BLOCK - 1) : 0;
    u.units = u.r.n > 0 ? max((u.kend - u.k0 + unit - 1) / unit, 1) : 0;   // a row without keys is written too
    return u;
}

__device__ __forceinline__ int same(int x) { return __builtin_amdgcn_readfirstlane(x); }

// ... of a sequence that is the same in every lane, held in scalar registers
__device__ __forceinline__ SeqUnits uniform_units(const SeqUnits & v) {
    SeqUnits u;
    u.r.row0 = same(v.r.row0);
    u.r.n = same(v.r.n);
    u.r.len = same(v.r.len);
    u.k0 = same(v.k0);
    u.kend = same(v.kend);
    u.units = same(v.units);
    return u;
}

// The line that runs share out, in halves of a unit: an item has one half more
// than its units, for what a piece costs beside them (its queries, its first
// loads, its results).
__device__ __forceinline__ int item_steps(int units) { return units > 0 ? 2 * units + 1 : 0; }
// Runs over `total` steps: the first total % n take one more.
struct Runs {
    int q, more;
    __device__ __forceinline__ Runs(int total, int n) : q(total / n), more(total - total / n * n) {}
    __device__ __forceinline__ int begin(int run) const { return run * q + min(run, more); }
    __device__ __forceinline__ int owner(int step) const {
        const int head = more * (q + 1);
        return step < head ? step / (q + 1) : more + (step - head) / q;
    }
};
// Of an item's steps, counted from its first, unit k is the run's that has step
// 2 k + 1; the last step is no unit's.  Runs have two steps at least, so that each
// run between an item's first and last has a unit of it.
__device__ __forceinline__ int units_before(int step) { return step >> 1; }
__device__ __forceinline__ int runs_of(int most, int total) { return min(most, total >> 1); }

// bit i: key `at` + i, i < 8, is in [from, to)
__device__ __forceinline__ uint32_t seen8(int at, int from, int to) {
    const uint32_t below = (1u << min(max(to - at, 0), 8)) - 1, before = (1u << min(max(from - at, 0), 8)) - 1;
    return below & ~before;
}
// ones where bits i and i + 1 are set, for a pair of 16-bit values
__device__ __forceinline__ uint32_t pair_mask(uint32_t bits, int i) {
    const uint32_t a = (uint32_t)((int)(bits << (31 - i)) >> 31), b = (uint32_t)((int)(bits << (30 - i)) >> 31);
    return (a & 0xFFFFu) | (b & 0xFFFF0000u);
}

// A CU serves its oldest workgroup first: of three that share a CU for a whole long
// call the first ended at 84 us, the last at 106, when it had the CU to itself.  With a
// unit each at every priority in turn they go on together (TB/s of long caches: head
// size 64 5.34 -> 5.46, 128 5.53 -> 5.61, 256 5.33 -> 5.44; q8_0, still without
// V's second part, 5.0 -> 5.2, 5.1 -> 5.35; two or one to a CU: no difference).
__device__ __forceinline__ void priority_in_turn(int turn) {
    switch (turn & 3) {
        case 0: __builtin_amdgcn_s_setprio(0); break;
        case 1: __builtin_amdgcn_s_setprio(1); break;
        case 2: __builtin_amdgcn_s_setprio(2); break;
        default: __builtin_amdgcn_s_setprio(3);
    }
}

constexpr float KV_LN2 = 0.69314718055994530942f, KV_LOG2E = 1.44269504088896340736f;

// WIDE: fp32 queries and results
template <int CT, bool WIDE, int HD, int NT>
struct KvShape {
    static constexpr bool HALF = CT != KV_BF16;
    static constexpr int PQ = HALF ? (WIDE ? 2 : 1) : (WIDE ? 3 : 2);
    static constexpr int PP = HALF ? 2 : (WIDE ? 3 : 2);
    static constexpr int WAVES = kv_waves(HD), UNIT = kv_unit(HD), KT = UNIT / (16 * WAVES), NB = UNIT / KV_BLOCK;
    static constexpr int NC = HD / 32, NV = HD / 16, NVW = (NV + WAVES - 1) / WAVES;
    static constexpr int Q_BYTES = PQ * NT * NC * 1024;
    static constexpr int P_BYTES = NB * NT * PP * 1024;
    static constexpr int LDS = Q_BYTES + P_BYTES;
};

template <int CT, bool WIDE, int HD, int NT>
__global__ __launch_bounds__(64 * kv_waves(HD), kv_wgs(HD, NT) * kv_waves(HD) / 4) void k_kv_attn(const KvAttn p) {
    using Sh = KvShape<CT, WIDE, HD, NT>;
    constexpr bool HALF = Sh::HALF, Q8 = CT == KV_Q8;
    constexpr int PQ = Sh::PQ, PP = Sh::PP, NC = Sh::NC, NV = Sh::NV, NVW = Sh::NVW, KT = Sh::KT, NB = Sh::NB;
    constexpr int UNIT = Sh::UNIT, ROWS = 16 * NT, WAVES = Sh::WAVES, WGT = 64 * WAVES;
    constexpr int EL = Q8 ? 1 : 2;                                // bytes of a cached value
    constexpr float P_SHIFT = HALF ? 15.0f : 0.0f;                // log2 of p's scale
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ struct { int seq, step; SeqUnits su; } s_first;
    __shared__ int s_part[WAVES];
    __shared__ int s_exp[ROWS];
    __shared__ float s_top[WAVES][ROWS];
    uint8_t * const lds_p = lds + Sh::Q_BYTES;

    const int tid = threadIdx.x, lane = tid & 63, wave = same(tid >> 6);
    const int lm = lane & 15, lg = lane >> 4;
    const int page = 1 << p.page_shift, page_mask = page - 1;
    const int type = WIDE ? (int)T_F32 : p.type;
    // run and tile: a run's tiles are eight workgroups apart, on one XCD
    const int octet = blockIdx.x >> 3, tile = octet % p.tiles, run = octet / p.tiles * 8 + (blockIdx.x & 7);
    auto units_at = [&](int s) { return seq_units(p.b, s, p.page_shift, p.window, UNIT); };

    // ---- the line: thread t counts sequences [t per, (t + 1) per)
    const int per = (p.b.n_seq + WGT - 1) / WGT;
    int sum = 0;
    for (int i = 0; i < per; ++i) {
        const int s = tid * per + i;
        if (s < p.b.n_seq) sum += item_steps(units_at(s).units) * p.n_kv;
    }
    const int own = sum;
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(sum, o, 64);
        if (lane >= o) sum += v;
    }
    if (lane == 63) s_part[wave] = sum;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) sum += s_part[w];
        total += s_part[w];
    }
    total = same(total);
    const int n_runs = runs_of(p.runs, total);
    if (blockIdx.x == 0) {
        // for the join
        int at = sum - own;
        for (int i = 0; i < per; ++i) {
            const int s = tid * per + i;
            if (s < p.b.n_seq) {
                p.base[s] = at;
                at += item_steps(units_at(s).units) * p.n_kv;
            }
        }
        if (tid == 0) p.base[p.b.n_seq] = total;
    }
    if (run >= n_runs) return;
    const Runs runs(total, n_runs);
    const int lo = runs.begin(run), hi = runs.begin(run + 1);

    // ---- the sequence of the first step, which one thread has counted, and from
    // there on piece by piece
    if (sum - own <= lo && lo < sum) {
        int s = tid * per, at = sum - own;
        SeqUnits v = units_at(s);
        for (int n; lo - at >= (n = item_steps(v.units) * p.n_kv) && s + 1 < p.b.n_seq; v = units_at(++s)) at += n;
        s_first.seq = s;
        s_first.step = at;
        s_first.su = v;
    }
    __syncthreads();
    int at_seq = same(s_first.seq), at_step = same(s_first.step);      // a sequence and its first step
    SeqUnits at_su = uniform_units(s_first.su);
    struct Piece {
        SeqUnits su;
        int head, u0, n_u, key_begin, key_end;
        const int32_t * row;                          // of the page table
        uint64_t part;                                // a head's part of a page, which its scales follow
    };
    int step = lo;
    // the next piece with rows of this tile; false at the run's end (and where
    // another stream has changed the lengths meanwhile)
    auto next_piece = [&](Piece & c) {
        while (step < hi) {
            int n_here;
            while (step - at_step >= (n_here = item_steps(at_su.units) * p.n_kv)) {
                if (at_seq + 1 >= p.b.n_seq) return false;
                at_step += n_here;
                ++at_seq;
                at_su = uniform_units(units_at(at_seq));
            }
            if (tile * ROWS >= at_su.r.n * p.group) {
                step = at_step + n_here;              // this sequence has fewer rows
                continue;
            }
            const int steps = item_steps(at_su.units), head = (step - at_step) / steps, first = at_step + head * steps;
            const int u0 = units_before(step - first), u1 = units_before(min(hi - first, steps));
            step = min(hi, first + steps);
            if (u1 <= u0) continue;
            c.su = at_su;
            c.head = head;
            c.u0 = u0;
            c.n_u = u1 - u0;
            c.key_begin = at_su.k0 + u0 * UNIT;
            c.key_end = min(c.key_begin + c.n_u * UNIT, at_su.kend);
            c.row = p.b.table + at_seq * p.b.table_stride;
            c.part = (uint64_t)head * page * (Q8 ? HD + HD / 16 : 2 * HD);
            return true;
        }
        return false;
    };

    // ---- loads of a unit's K, ahead of its use
    // places of the wave's keys in a unit: those of its K rows, those of the lane's scores
    const int w_block = KT == 2 ? wave : wave >> 1, w_half = KT == 2 ? 0 : 4 * (wave & 1);
    const int k_oct = KV_BLOCK * w_block + 8 * (lm >> 2), s_oct = KV_BLOCK * w_block + 8 * lg;
    constexpr int NP = Q8 ? NC / 2 : 0, ODD = Q8 ? NC % 2 : 0;    // q8_0: pairs of 32 values, a last one
    constexpr int NKF = Q8 ? NP + ODD : NC;                       // K's loads of a row
    constexpr int NVL = Q8 ? UNIT / 64 : NB;                      // V's loads of a column
    constexpr int NVD = (NVW + 1) / 2;                            // 32-column blocks of a wave's V tiles
    u4 kf[KT][NKF], vf[NVL][NVW];
    uint32_t kd[KT][Q8 ? NKF : 1];                    // fp16 scales of the lane's K row
    int k_pg = 0, s_pg = 0, v_pg[NVL];
    auto has_page = [&](int pg) { return (uint32_t)pg < (uint32_t)p.n_pages; };
    auto page_at = [&](const int32_t * row, int key) {
        const int i = key >> p.page_shift;
        const int pg = row[min(i, p.b.max_pages - 1)];
        return i < p.b.max_pages ? pg : -1;
    };
    // places of a lane's V keys in a unit: 8 of each block, q8_0: 16 of each load, whose halves are blocks
    auto v_place = [&](int b) { return Q8 ? 64 * (b >> 1) + 16 * lg + 8 * (b & 1) : KV_BLOCK * b + 8 * lg; };
    auto load_pages = [&](const int32_t * row, int at) {
        k_pg = page_at(row, at + k_oct);
        s_pg = Q8 ? page_at(row, at + s_oct) : 0;
#pragma unroll
        for (int i = 0; i < NVL; ++i) v_pg[i] = page_at(row, at + v_place(Q8 ? 2 * i : i));
    };
    auto load_k = [&](uint64_t part, int at) {
        const uint8_t * pg = p.k + part + (uint64_t)(has_page(k_pg) ? k_pg : 0) * p.k_stride;
        const int slot = (at + k_oct + w_half + (lm & 3)) & page_mask;
        const uint8_t * a = pg + (slot * HD + (Q8 ? 16 : 8) * lg) * EL;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            if constexpr (Q8) {
#pragma unroll
                for (int c = 0; c < NP; ++c) kf[t][c] = *(const u4 *)(a + 4 * t * HD + 64 * c);
                if constexpr (ODD != 0) {
                    const u2 w = *(const u2 *)(a - 8 * lg + 4 * t * HD + 64 * NP);
                    kf[t][NP] = u4{w[0], w[1], 0, 0};
                }
                const uint16_t * d = (const uint16_t *)(pg + page * HD) + slot + 4 * t;
#pragma unroll
                for (int c = 0; c < NP; ++c) kd[t][c] = d[(2 * c + (lg >> 1)) * page];
                if constexpr (ODD != 0) kd[t][NP] = d[2 * NP * page];
            } else {
#pragma unroll
                for (int c = 0; c < NC; ++c) kf[t][c] = *(const u4 *)(a + (4 * t * HD + 32 * c) * EL);
            }
        }
    };
    // the wave's columns of V, from 16 v_tile on (a tile past the last one reads it again)
    const int v_tile = wave * NVW;

    Piece cur, then;
    if (!next_piece(cur)) return;
    if (cur.key_begin < cur.key_end) {
        load_pages(cur.row, cur.key_begin);
        load_k(cur.part, cur.key_begin);
    }
    for (;;) {
        const SeqUnits & su = cur.su;
        const int head = cur.head, key_end = cur.key_end;
        const int n_rows = min(su.r.n * p.group - tile * ROWS, ROWS);
        const bool whole = cur.n_u == su.units;
        const int64_t slot = ((int64_t)run * p.tiles + tile) * 2 + (cur.u0 == 0);

        // ---- Q into LDS as B operands, (part, 32 values) x lane: 16 threads a row
        __syncthreads();                                           // the last piece's LDS has been read
        constexpr int QE = (HD / 8 + 15) / 16;
#pragma unroll 1
        for (int r = tid >> 4; r < ROWS; r += WGT / 16) {
            const int rr = tile * ROWS + r, tok = rr / p.group;
            const int64_t from = (su.r.row0 + tok) * p.q_stride + (int64_t)(head * p.group + rr - tok * p.group) * HD;
            float qx[QE][8];
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < QE; ++e) {
                const int o = (tid & 15) + 16 * e;
#pragma unroll
                for (int j = 0; j < 8; ++j) qx[e][j] = 0.0f;
                if (r < n_rows && o < HD / 8) load8(p.q, type, from + 8 * o, qx[e]);
                if (HALF)
#pragma unroll
                    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(qx[e][j]));
            }
            int ex = 0;
            if (HALF) {
                // the row's largest to [2^13, 2^14): exact, and undone with the scale (0 and non-finite: left)
#pragma unroll
                for (int o = 8; o; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
                ex = amax > 0.0f && amax < __builtin_inff() ? 14 - __builtin_amdgcn_frexp_expf(amax) : 0;
                if ((tid & 15) == 0) s_exp[r] = ex;
            }
#pragma unroll
            for (int e = 0; e < QE; ++e) {
                const int o = (tid & 15) + 16 * e;
                if (o < HD / 8) {
                    if (HALF)
#pragma unroll
                        for (int j = 0; j < 8; ++j) qx[e][j] = __builtin_ldexpf(qx[e][j], ex);
                    u4 part[PQ];
                    split8<HALF, PQ>(qx[e], part);
                    // the product and lane group that eight values go to
                    const int c = o < 8 * NP ? 2 * (o >> 3) + (o & 1) : o >> 2, g = o < 8 * NP ? (o >> 1) & 3 : o & 3;
#pragma unroll
                    for (int q = 0; q < PQ; ++q) *(u4 *)(lds + ((q * NT + (r >> 4)) * NC + c) * 1024 + (g * 16 + (r & 15)) * 16) = part[q];
                }
            }
        }
        // the next piece, whose first K is loaded during this one's last unit
        const bool more = next_piece(then);
        __syncthreads();
        // the lane's query rows: token, position, score scale in log2
        int t_pos[NT], tok_of[NT];
        float q_scale[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            tok_of[nt] = min((tile * ROWS + 16 * nt + lm) / p.group, su.r.n - 1);
            t_pos[nt] = su.r.len - su.r.n + tok_of[nt];
            q_scale[nt] = p.scale * KV_LOG2E;
            if (HALF) q_scale[nt] = __builtin_ldexpf(q_scale[nt], -s_exp[16 * nt + lm]);
        }

        // ---- the units
        f4v acc[NT][NVW];
        float m[NT], l[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = -__builtin_inff();
            l[nt] = 0.0f;
#pragma unroll
            for (int t = 0; t < NVW; ++t) acc[nt][t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
        }
        // keys that every row of the sequence sees
        const int all_to = su.r.len - su.r.n + 1;                            // one past the first new token
        const int all_from = p.window > 0 ? su.r.len - p.window : 0;         // the last one's first key
        const uint8_t * vbase = p.v + cur.part;
        const bool then_keys = more && then.key_begin < then.key_end;
        if (cur.key_begin >= key_end && then_keys) {
            load_pages(then.row, then.key_begin);
            load_k(then.part, then.key_begin);
        }
        int lv = lm;
        for (int key = cur.key_begin; key < key_end; key += UNIT) {
            asm volatile("" : "+v"(lv));              // V's offsets are formed anew, not held
            if constexpr (kv_wgs(HD, NT) > 2) priority_in_turn(key / UNIT + (int)(blockIdx.x >> 8));
            bool full = key + UNIT <= min(all_to, key_end) && key >= all_from;
            uint32_t ok = 0;                          // bit i: the keys of the lane's load i have a page
            const uint8_t * va[NVL];
#pragma unroll
            for (int i = 0; i < NVL; ++i) {
                va[i] = vbase + (uint64_t)(has_page(v_pg[i]) ? v_pg[i] : 0) * p.v_stride;
                ok |= (uint32_t)has_page(v_pg[i]) << i;
            }
            full = full && __all(ok == (1u << NVL) - 1);
            const bool s_ok = Q8 ? has_page(s_pg) : (ok >> w_block) & 1;      // the lane's scores have a page
            const bool last = key + UNIT >= key_end, ahead = !last || then_keys;
            const int next = last ? then.key_begin : key + UNIT;
            if (ahead) load_pages(last ? then.row : cur.row, next);
            // the scales of a block's 32 columns, which two tiles share where v_tile is even
            u4 vd[Q8 ? NB : 1][Q8 ? NVD : 1];
            auto load_v = [&](int i) {
                const int slot = (key + v_place(Q8 ? 2 * i : i)) & page_mask;
#pragma unroll
                for (int t = 0; t < NVW; ++t) {
                    const int vt = NV % WAVES ? min(v_tile + t, NV - 1) : v_tile + t;
                    vf[i][t] = *(const u4 *)(va[i] + ((16 * vt + lv) * page + slot) * EL);
                }
                if constexpr (Q8)
#pragma unroll
                    for (int c = 0; c < NVD; ++c) {
                        const u4 * d = (const u4 *)(va[i] + page * HD + (min((v_tile >> 1) + c, NC - 1) * page + slot) * 2);
                        vd[2 * i][c] = d[0];
                        vd[2 * i + 1][c] = d[1];
                    }
            };
#pragma unroll
            for (int i = 0; i < NVL; ++i) load_v(i);
            // ---- S^T of the wave's keys
            __builtin_amdgcn_sched_barrier(0);
            f4v sc[NT][KT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int t = 0; t < KT; ++t) sc[nt][t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                u4 a[KT], a_lo[KT];
#pragma unroll
                for (int t = 0; t < KT; ++t)
                    if constexpr (Q8) {
                        const int f = c < 2 * NP ? c >> 1 : NP, h = c < 2 * NP ? c & 1 : 0;
                        // no part of the conversion moves up to the load, to wait for it there
                        if (h == 0) asm volatile("" : "+v"(kf[t][f]), "+v"(kd[t][f]));
                        const uint32_t d = kd[t][f] | kd[t][f] << 16;
                        times_scale(i8_to_half(u2{kf[t][f][2 * h], kf[t][f][2 * h + 1]}), u4{d, d, d, d}, a[t], a_lo[t]);
                    } else {
                        a[t] = kf[t][c];
                    }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int q = 0; q < PQ; ++q) {
                        const u4 b = *(const u4 *)(lds + ((q * NT + nt) * NC + c) * 1024 + lane * 16);
#pragma unroll
                        for (int t = 0; t < KT; ++t) {
                            sc[nt][t] = mfma16<HALF>(a[t], b, sc[nt][t]);
                            if (Q8 && q == 0) sc[nt][t] = mfma16<HALF>(a_lo[t], b, sc[nt][t]);
                        }
                    }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (ahead) load_k(last ? then.part : cur.part, next);
            __builtin_amdgcn_sched_barrier(0);
            // ---- softmax: the lane's keys are key + s_oct + w_half + (0 .. 4 KT - 1)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int t = 0; t < KT; ++t) sc[nt][t] *= q_scale[nt];
                if (!full) {
                    const int from = p.window > 0 ? t_pos[nt] - p.window + 1 : 0, to = min(t_pos[nt] + 1, s_ok ? key_end : 0);
#pragma unroll
                    for (int t = 0; t < KT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int at = key + s_oct + w_half + 4 * t + i;
                            sc[nt][t][i] = ((at >= from) & (at < to)) ? sc[nt][t][i] : -__builtin_inff();
                        }
                }
                float top = -__builtin_inff();
#pragma unroll
                for (int t = 0; t < KT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[nt][t][i]);
                top = over_groups(top, [](float a, float b) { return fmaxf(a, b); });
                if (lg == 0) s_top[wave][16 * nt + lm] = top;
            }
            __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float now = m[nt];
#pragma unroll
                for (int w = 0; w < WAVES; ++w) now = fmaxf(now, s_top[w][16 * nt + lm]);
                const float ref = now == -__builtin_inff() ? 0.0f : now;
                if (__any(now != m[nt])) {
                    const float f = __builtin_amdgcn_exp2f(m[nt] - ref);
                    l[nt] *= f;
#pragma unroll
                    for (int t = 0; t < NVW; ++t) acc[nt][t] *= f;
                    m[nt] = now;
                }
                float x[8];
#pragma unroll
                for (int i = 0; i < 4 * KT; ++i) {
                    x[i] = __builtin_amdgcn_exp2f(sc[nt][i >> 2][i & 3] - (ref - P_SHIFT));
                    l[nt] += x[i];
                }
#pragma unroll
                for (int i = 4 * KT; i < 8; ++i) x[i] = 0.0f;
                u4 part[PP];
                split8<HALF, PP>(x, part);
                const int b = Q8 ? 2 * (w_block >> 1) + (lg & 1) : w_block;
                const int at = Q8 ? (2 * (w_block & 1) + (lg >> 1)) * 16 + lm : lane;
#pragma unroll
                for (int q = 0; q < PP; ++q) {
                    uint8_t * w = lds_p + ((b * NT + nt) * PP + q) * 1024 + at * 16;
                    if constexpr (KT == 2) *(u4 *)w = part[q];
                    else *(u2 *)(w + 2 * w_half) = u2{part[q][0], part[q][1]};
                }
            }
            __syncthreads();
            // ---- O^T of the wave's columns
            // 0 times a masked infinity is no zero: what is not seen by every row
            // becomes 0 in V, for q8_0 in its scales
            const int core_to = min(all_to, key_end);
            auto add_block = [&](int b) {
                if (!full) {
                    const uint32_t bits = (ok >> (Q8 ? b >> 1 : b)) & 1 ? seen8(key + v_place(b), all_from, core_to) : 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t keep = pair_mask(bits, 2 * i);
                        if constexpr (Q8) {
#pragma unroll
                            for (int c = 0; c < NVD; ++c) vd[b][c][i] &= keep;
                        } else {
#pragma unroll
                            for (int t = 0; t < NVW; ++t) vf[b][t][i] &= keep;
                        }
                    }
                }
                u4 bp[NT][PP];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int q = 0; q < PP; ++q)
                        bp[nt][q] = *(const u4 *)(lds_p + ((b * NT + nt) * PP + q) * 1024 + lane * 16);
#pragma unroll
                for (int t = 0; t < NVW; ++t) {
                    u4 hi, lo;
                    if constexpr (Q8) {
                        if (b % 2 == 0) asm volatile("" : "+v"(vf[b / 2][t]));      // not converted where it is loaded
                        const u4 d = vd[b][NVW % 2 == 0 ? t / 2 : 0], d1 = vd[b][NVD - 1];
                        const bool next_block = NVW % 2 && ((v_tile + t) >> 1) != v_tile >> 1;
                        times_scale(i8_to_half(u2{vf[b / 2][t][2 * (b % 2)], vf[b / 2][t][2 * (b % 2) + 1]}),
                                    next_block ? d1 : d, hi, lo);
                    } else {
                        hi = vf[b][t];
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int q = 0; q < PP; ++q) acc[nt][t] = mfma16<HALF>(hi, bp[nt][q], acc[nt][t]);
                        if (Q8) acc[nt][t] = mfma16<HALF>(lo, bp[nt][0], acc[nt][t]);
                    }
                }
            };
#pragma unroll
            for (int b = 0; b < NB; ++b) add_block(b);
            // keys that only some of a sequence's tokens see (at its end, at the
            // window's begin) are added token by token
            if (!full && su.r.n > 1) {
#pragma unroll 1
                for (int b = 0; b < NB; ++b) {
                    // the block's keys lie in [kb, kb + span)
                    constexpr int span = Q8 ? 64 : KV_BLOCK;
                    const int kb = key + span * (Q8 ? b >> 1 : b);
                    const int first = p.window > 0 ? su.r.len - su.r.n - p.window + 1 : 0;
                    if (!((kb + span > core_to && kb < key_end) || (kb < all_from && kb + span > first))) continue;
                    const int at = key + v_place(b), pg = page_at(cur.row, at), slot = at & page_mask;
                    const uint8_t * a = vbase + (uint64_t)(has_page(pg) ? pg : 0) * p.v_stride;
                    typedef typename std::conditional<Q8, u2, u4>::type frag;
                    frag vz[NVW];
                    u4 dz[Q8 ? NVW : 1];
#pragma unroll
                    for (int t = 0; t < NVW; ++t) {
                        const int vt = NV % WAVES ? min(v_tile + t, NV - 1) : v_tile + t;
                        vz[t] = *(const frag *)(a + ((16 * vt + lv) * page + slot) * EL);
                        if constexpr (Q8) dz[t] = *(const u4 *)(a + page * HD + ((vt >> 1) * page + slot) * 2);
                    }
#pragma unroll 1
                    for (int tok = 0; tok < su.r.n; ++tok) {
                        asm volatile("" ::: "memory");        // P stays in LDS
                        const int pos = su.r.len - su.r.n + tok;
                        uint32_t bits = seen8(at, p.window > 0 ? pos - p.window + 1 : 0, min(pos + 1, key_end));
                        bits = has_page(pg) ? bits & ~seen8(at, all_from, core_to) : 0;
                        u4 keep;
#pragma unroll
                        for (int i = 0; i < 4; ++i) keep[i] = pair_mask(bits, 2 * i);
#pragma unroll
                        for (int t = 0; t < NVW; ++t) {
                            u4 hi, lo;
                            if constexpr (Q8) times_scale(i8_to_half(vz[t]), dz[t] & keep, hi, lo);
                            else hi = vz[t] & keep;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                f4v d = f4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                                for (int q = 0; q < PP; ++q) {
                                    const u4 bp = *(const u4 *)(lds_p + ((b * NT + nt) * PP + q) * 1024 + lane * 16);
                                    d = mfma16<HALF>(hi, bp, d);
                                    if (Q8 && q == 0) d = mfma16<HALF>(lo, bp, d);
                                }
#pragma unroll
                                for (int i = 0; i < 4; ++i) acc[nt][t][i] += tok_of[nt] == tok ? d[i] : 0.0f;
                            }
                        }
                    }
                }
            }
        }

        // ---- the sums of the waves, in their order; maxima are the same in all
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) l[nt] = over_groups(l[nt], [](float a, float b) { return a + b; });
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            if (lg == 0) s_top[wave][16 * nt + lm] = l[nt];
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = 16 * nt + lm;
            if (r >= n_rows) continue;
            float sum = s_top[0][r];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum += s_top[w][r];
            if (whole) {
                const int rr = tile * ROWS + r, tok = rr / p.group, hq = head * p.group + rr - tok * p.group;
                const int64_t out_row = su.r.row0 + tok;
                const float norm = p.row_ml ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int t = 0; t < NVW; ++t)
                    if (v_tile + t < NV)
                        store4(p.out, p.row_ml ? (int)T_F32 : type, out_row * p.out_stride + (int64_t)hq * HD + 16 * (v_tile + t) + 4 * lg, acc[nt][t] * norm);
                const int64_t at = out_row * (p.group * p.n_kv) + hq;
                if (p.row_ml && wave == 0 && lg == 0) {
                    p.row_ml[2 * at] = m[nt];
                    p.row_ml[2 * at + 1] = sum;
                } else if (p.lse && wave == 0 && lg == 0) {
                    p.lse[at] = sum == 0.0f ? -__builtin_inff() : (m[nt] + (__builtin_amdgcn_logf(sum) - P_SHIFT)) * KV_LN2;
                }
            } else {
                float * a = p.acc + (slot * ROWS + r) * HD;
#pragma unroll
                for (int t = 0; t < NVW; ++t)
                    if (v_tile + t < NV) *(f4v *)(a + 16 * (v_tile + t) + 4 * lg) = acc[nt][t];
                if (wave == 0 && lg == 0) {
                    p.ml[(slot * ROWS + r) * 2] = m[nt];
                    p.ml[(slot * ROWS + r) * 2 + 1] = sum;
                }
            }
        }
        if (!more) return;
        cur = then;
    }
}

template <int CT, bool WIDE, int HD, int NT>
hipError_t launch_kv_attn_one(const KvAttn & p, hipStream_t s) {
    hipLaunchKernelGGL((k_kv_attn<CT, WIDE, HD, NT>), dim3(p.runs * p.tiles), dim3(64 * kv_waves(HD)),
                       (KvShape<CT, WIDE, HD, NT>::LDS), s, p);
    return hipGetLastError();
}

template <int CT, bool WIDE, int NT>
hipError_t launch_kv_attn_hd(const KvAttn & p, int head_dim, hipStream_t s) {
    switch (head_dim) {
        case 64: return launch_kv_attn_one<CT, WIDE, 64, NT>(p, s);
        case 96: return launch_kv_attn_one<CT, WIDE, 96, NT>(p, s);
        case 128: return launch_kv_attn_one<CT, WIDE, 128, NT>(p, s);
        case 192: return launch_kv_attn_one<CT, WIDE, 192, NT>(p, s);
        case 256: return launch_kv_attn_one<CT, WIDE, 256, NT>(p, s);
        case 512: return launch_kv_attn_one<CT, WIDE, 512, NT>(p, s);
    }
    return hipErrorInvalidValue;
}

template <int CT>
hipError_t launch_kv_attn_type(const KvAttn & p, int head_dim, hipStream_t s) {
    if (p.type == T_F32)
        return p.nt == 1 ? launch_kv_attn_hd<CT, true, 1>(p, head_dim, s) : launch_kv_attn_hd<CT, true, 2>(p, head_dim, s);
    return p.nt == 1 ? launch_kv_attn_hd<CT, false, 1>(p, head_dim, s) : launch_kv_attn_hd<CT, false, 2>(p, head_dim, s);
}

}  // namespace dev
}  // namespace llapis
