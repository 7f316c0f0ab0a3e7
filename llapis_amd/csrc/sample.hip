// sample.hip -- the next token of each sequence from its logits (llapis_step.h).
//
// With M the largest logit a value's weight is w = e^((x - M) / T), and every
// filter keeps an upper part of the values in the order (value descending, index
// ascending).  Four kernels find where that part ends and draw from it, without
// sorting the row:
//   k_sample_scan   a workgroup's values: the largest, and where a top_k or top_p is to be
//                   found a histogram over SMP_BINS bins, 16 to a factor of 2 of the weight
//   k_sample_find   a workgroup a sequence adds the histograms and finds the few bins in
//                   which top_k and top_p may end, and the values that these begin with
//   k_sample_split  a workgroup's values again: those above are surely kept (summed), those
//                   between only count towards top_p's whole (summed), the candidates are listed
//   k_sample_pick   a workgroup a sequence ends both filters among the candidates exactly
//                   and finds the token: its segment by the segments' sums, then the value
// and k_sample_probs writes probabilities if they are wanted.  A histogram's word holds the
// sum of a bin's weights, in 2^-18 of the bin's least: all of it to 2^-15, and the number of its values
// to 4 % (for top_k alone it holds their number).  They only say which bins are looked at: mostly one for
// each filter.  (Words of numbers and of coarse weights, to 0.3 %, had ten times the candidates at a top_p of 0.99, where they
// did not fit: 8 rows of 65536 230 us.)  What decides is fp64 (and fixed point, where sums are made by atomics: 49 bits
// of the candidates' largest weight and more, and where the border may lie too far below that, twice as many): weights,
// their sums and products, in a fixed order, so that a draw next to a border falls as the definition says.
//
// Bound, for few rows, by the four launches and a workgroup's barriers (1 row of 32003 fp32 values: 4.0, 6.9, 3.9 and
// 8.9 us); for many by two passes over the logits (32 rows of 262144, 33.5 MB: 12.4 and 13.9 us, the sequences' kernels
// 10.0 and 12.8), the second of which forms every kept value's weight in fp64: with top_p alone that is
// most of them (64 rows of 128001 bf16: 11.7, 9.0, 18.5 and 13.0 us, probabilities 20.1; the VALU is busy for 68 % of the
// split's time and 63 % of the probabilities').  All values kept, and the largest alone: 32 rows of 262144 34 and 14 us.
// Where the end's bins hold more candidates than SMP_HOLD a thread, or a bucket of them more than there are threads,
// k_sample_pick finds it digit by digit (8 rows of 262144 at top_p 0.9999999: 113 us a call; 32 rows all of whose values are
// equal: 1.3 ms).  Hundreds of equal values there are compared each with each (32 rows of 262144 bf16 at 0.9, 480 ties:
// 79 us, k_sample_pick 41 of them; at 0.99 with 90 56 and 19).
#include <algorithm>
#include <cstdio>

#include "kv.h"

namespace llapis {
namespace dev {

constexpr int SMP_WG = 256, SMP_WAVES = SMP_WG / 64;      // of the kernels that read rows
constexpr int SMP_SEQ_WG = 1024, SMP_SEQ_WAVES = SMP_SEQ_WG / 64;     // of those with a workgroup a sequence
// Values of a lane: 32, and 8 where rows are few and short, which then go to four times the
// workgroups.  A wave's values are a segment, a workgroup's a chunk
constexpr int smp_seg(int lane_values) { return 64 * lane_values; }
constexpr int smp_chunk(int lane_values) { return SMP_WG * lane_values; }
constexpr int SMP_BINS = 1024, SMP_OUT = SMP_BINS + 1;    // a value below all bins is in SMP_OUT
constexpr float SMP_PER_OCTAVE = 16.0f;
constexpr int SMP_HOLD = 8;                               // candidates of a thread, held at once
// a weight in a histogram's word, the least and the most of a bin: 2^18 to 2^(18 + 1 / 16)
constexpr uint32_t SMP_LEAST = 1 << 18, SMP_MOST = 273750;
static_assert((uint64_t)smp_chunk(32) * SMP_MOST < 1ull << 32, "a chunk's values fit in a word");

struct SmpChunk { float top; int32_t at; };               // a chunk's largest value and its lowest index
struct SmpSeg { double sure, draw, mid; int32_t n_sure, n_mid, n_cand, pad; };
// A sequence's cut.  In the order of values: from x_sure on surely kept, from x_cand on
// candidates, from x_mid on not kept by top_p, from x_end on candidates again (top_k's end); the rest is out
struct SmpCut {
    float top;                     // M
    float x_sure, x_cand, x_mid, x_end;
    int32_t token;                 // the first value's index, -1 without one
    uint64_t key;                  // the last candidate that is kept, ~0 without one
    double total;                  // the kept weights' sum
};

struct SmpAbove { int32_t n; int64_t hi, lo; };            // number and weight of the candidates above a digit

struct SmpWs {
    SmpCut * cuts;                 // [n_seq]
    SmpChunk * chunks;             // [n_seq][n_chunks]
    SmpSeg * segs;                 // [n_seq][n_chunks * SMP_WAVES]
    uint32_t * hist;               // [n_seq][n_chunks][SMP_BINS]
    uint64_t * keys;               // [n_seq][n_chunks * chunk] candidates, by segment
    int n_chunks;
};

// a sequence's settings
struct SmpSet {
    bool greedy, by_k, by_p;       // the largest value alone; a number of values; a part of their weight
    int k;
    double p, min_p;
    double octaves;                // log2 of the weight a unit of x
    float bins;                    // bins a unit of x; 0: one bin for all values
};

__device__ __forceinline__ SmpSet smp_settings(const llapis_sample_args & a, int seq) {
    SmpSet s;
    const float t = a.temperature ? a.temperature[seq] : 1.0f, p = a.top_p ? a.top_p[seq] : 1.0f;
    const float m = a.min_p ? a.min_p[seq] : 0.0f;
    s.k = a.top_k ? a.top_k[seq] : 0;
    s.by_k = s.k > 0 && s.k < a.vocab;
    s.by_p = p < 1.0f;
    s.greedy = !(t > 0.0f) || s.k == 1 || p <= 0.0f || m > 1.0f;
    s.p = (double)p;
    s.min_p = m > 0.0f ? (double)m : 0.0;
    s.octaves = 1.44269504088896340736 / (double)t;
    s.bins = (float)s.octaves * SMP_PER_OCTAVE;
    if (!(s.bins < 0x1p60f)) s.bins = 0.0f;
    return s;
}

// ordered as the values are; of equal ones the lowest index is the largest key
__device__ __forceinline__ uint64_t smp_key(float x, int i) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float smp_value(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ int smp_index(uint64_t key) { return (int)~(uint32_t)key; }

constexpr float SMP_NONE = -__builtin_inff();             // no value: it has no weight

// 2^t for t <= 0: the whole part in the exponent, the rest r by the polynomial that agrees with 2^r at
// the 11 Chebyshev nodes of |r| <= 1/2, to 2^-51 of it.  Its coefficients are kept in scalar
// registers, where a multiply-add reads them: in vector registers each is first copied
__device__ __forceinline__ double smp_exp2(double t) {
    constexpr double c[11] = {1.0, 0.69314718055995, 0.24022650695910097, 0.05550410866444772, 0.009618129107606888,
                              0.0013333558230164974, 0.0001540353044173605, 1.5252657260200837e-05, 1.321544258792169e-06,
                              1.0208690299958306e-07, 7.072585949269223e-09};
    const double in = __builtin_fmax(t, -1100.0), n = __builtin_rint(in), r = in - n;
    double y = c[10];
#pragma unroll
    for (int k = 9; k >= 0; --k) {
        double ck = c[k];
        asm("" : "+s"(ck));
        y = __builtin_fma(y, r, ck);
    }
    return __builtin_ldexp(y, (int)n);
}
// (a difference with an infinite value, or times an infinite 1 / T, is -inf or NaN: weight 0 unless x is M)
__device__ __forceinline__ double smp_weight(float x, float top, double octaves) {
    const double w = smp_exp2(((double)x - (double)top) * octaves);
    return x == top ? 1.0 : w;
}
// A value's bin below the largest's, the same wherever it is asked for, and never less for a
// smaller value.  What lies below all bins, or too far for fp32, is in SMP_OUT
__device__ __forceinline__ int smp_bin(float x, float top, float top_bin, float bins) {
    return x == top ? 0 : (int)fminf(top_bin - floorf(x * bins), (float)SMP_OUT);
}

// a NaN counts as no value, -0 as 0
__device__ __forceinline__ float smp_clean(float x) { return x != x ? SMP_NONE : x + 0.0f; }

template <class T> struct SmpVec { typedef T v __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T)))); };

// a lane's values of the segment at `base`: value j is row[smp_at<T>(base, j)]
template <class T>
__device__ __forceinline__ int smp_at(int base, int j) {
    constexpr int W = 16 / sizeof(T);
    return base + (j / W * 64 + (threadIdx.x & 63)) * W + j % W;
}
template <class T, int N>
__device__ __forceinline__ void smp_read(const T * row, int base, int n, float (&x)[N]) {
    constexpr int W = 16 / sizeof(T);
    if (base + smp_seg(N) <= n) {
        typename SmpVec<T>::v w[N / W];
#pragma unroll
        for (int c = 0; c < N / W; ++c) w[c] = *(const typename SmpVec<T>::v *)(row + smp_at<T>(base, c * W));
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = smp_clean((float)w[j / W][j % W]);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = smp_at<T>(base, j);
            x[j] = i < n ? smp_clean((float)row[i]) : SMP_NONE;
        }
    }
}

// f(first value's index, values) of the segment's vectors one after the other, two of them under way.
// (All of them at once, a loop over them unrolled: its code takes longer to fetch than to run.  Through
// LDS: work waits for the last.)
template <class T, int N, class F>
__device__ __forceinline__ void smp_stream(const T * row, int base, int n, F f) {
    constexpr int W = 16 / sizeof(T), C = N / W;
    typedef typename SmpVec<T>::v V;
    const bool whole = base + smp_seg(N) <= n;
    auto fetch = [&](int c) {
        const int i = smp_at<T>(base, min(c, C - 1) * W);
        V w;
        if (whole) {
            w = *(const V *)(row + i);
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j) w[j] = i + j < n ? row[i + j] : (T)SMP_NONE;
        }
        return w;
    };
    auto give = [&](int c, const V & w) {
        float x[W];
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] = smp_clean((float)w[j]);
        f(smp_at<T>(base, c * W), x);
    };
    V a = fetch(0);
    if constexpr (C == 1) {
        give(0, a);
    } else {
        V b = fetch(1);
#pragma unroll 1
        for (int c = 0; c < C; c += 2) {
            give(c, a);
            a = fetch(c + 2);
            give(c + 1, b);
            b = fetch(c + 3);
        }
    }
}

// ---- over a wave's lanes, by lane moves within rows of 16 and from row to row (a tenth of
// the time of permutes through LDS).  What a lane has none of is 0
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t smp_move(uint32_t x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false); }
template <int CTRL, int ROWS, class V>
__device__ __forceinline__ V smp_moved(V x) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, smp_move<CTRL, ROWS>(__builtin_bit_cast(uint32_t, x)));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        return __builtin_bit_cast(V, (uint64_t)smp_move<CTRL, ROWS>((uint32_t)(u >> 32)) << 32 | smp_move<CTRL, ROWS>((uint32_t)u));
    }
}
// f over this lane and those before it in their row of 16
template <class V, class F>
__device__ __forceinline__ V smp_row(V x, F f) {
    x = f(x, smp_moved<0x111, 0xF>(x));
    x = f(x, smp_moved<0x112, 0xF>(x));
    x = f(x, smp_moved<0x114, 0xF>(x));
    return f(x, smp_moved<0x118, 0xF>(x));
}
// ... and in the wave
template <class V, class F>
__device__ __forceinline__ V smp_wave(V x, F f) {
    x = smp_row(x, f);
    x = f(x, smp_moved<0x142, 0xA>(x));
    return f(x, smp_moved<0x143, 0xC>(x));
}
template <class V>
__device__ __forceinline__ V smp_lane(V x, int lane) {
    if constexpr (sizeof(V) == 4) {
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(uint32_t, x), lane));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, x);
        return __builtin_bit_cast(V, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(u >> 32), lane) << 32 |
                                         (uint32_t)__builtin_amdgcn_readlane((uint32_t)u, lane));
    }
}
struct SmpAdd { template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; } };
struct SmpMax { template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; } };

// ---- over a workgroup of WAVES <= 16 waves: a wave's last lane leaves its wave's, and
// after a barrier every wave has those of all.  A `part` is used once between two barriers
template <class V> __device__ __forceinline__ void smp_leave(V wave_value, V * part) {
    if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = wave_value;
}
template <int WAVES, class V, class F>
__device__ __forceinline__ V smp_all(const V * part, F f) {
    const int lane = threadIdx.x & 63;
    return smp_lane(smp_row(lane < WAVES ? part[lane] : V(0), f), WAVES - 1);
}
// what the waves before this one left, added
template <int WAVES, class V>
__device__ __forceinline__ V smp_before(const V * part, V & all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const V x = smp_row(lane < WAVES ? part[lane] : V(0), SmpAdd());
    all = smp_lane(x, WAVES - 1);
    return wave ? smp_lane(x, __builtin_amdgcn_readfirstlane(wave - 1)) : V(0);
}
// exclusive sums over the threads in order, and the whole
template <int WAVES, class V>
__device__ __forceinline__ V smp_scan(V x, V * part, V & all) {
    const V v = smp_wave(x, SmpAdd());
    smp_leave(v, part);
    __syncthreads();
    return smp_before<WAVES>(part, all) + smp_moved<0x138, 0xF>(v);
}

// the first of the lowest wave's first lanes with `yes`, by a minimum in LDS that begins above
__device__ __forceinline__ void smp_first(bool yes, int * at) {
    const uint64_t votes = __ballot(yes);
    if (votes && (threadIdx.x & 63) == 0) atomicMin(at, (int)threadIdx.x + (int)__builtin_ctzll(votes));
}

// ---------------------------------------------------------------- scan

template <class T, int N>
__global__ __launch_bounds__(SMP_WG) void k_sample_scan(const llapis_sample_args a, const SmpWs ws) {
    __shared__ uint32_t s_hist[SMP_BINS];
    __shared__ uint64_t s_part[SMP_WAVES];
    const int seq = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
    const int64_t chunk = (int64_t)seq * ws.n_chunks + blockIdx.x;
    const int base = blockIdx.x * smp_chunk(N) + wave * smp_seg(N);
    float x[N];
    smp_read((const T *)a.logits + seq * a.logits_stride, base, a.vocab, x);
    const SmpSet s = smp_settings(a, seq);
#pragma unroll
    for (int i = 0; i < SMP_BINS / SMP_WG; ++i) s_hist[i * SMP_WG + tid] = 0;
    // the largest, then the lowest index that has it
    float most = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) most = fmaxf(most, x[j]);
    int where = 0;
#pragma unroll
    for (int j = N - 1; j >= 0; --j) where = x[j] == most ? j : where;
    smp_leave(smp_wave(smp_key(most, smp_at<T>(base, where)), SmpMax()), s_part);
    __syncthreads();
    const uint64_t best = smp_all<SMP_WAVES>(s_part, SmpMax());
    const float top = smp_value(best);
    if (tid == 0) ws.chunks[chunk] = {top, smp_index(best)};
    if (s.greedy || !(s.by_k || s.by_p)) return;
    const float top_bin = floorf(top * s.bins);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float at = x[j] * s.bins;
        const int b = smp_bin(x[j], top, top_bin, s.bins);
        // (its place in the bin says nothing for what is out of fp32's range, as its bin does)
        const float w = __builtin_amdgcn_exp2f((at - floorf(at)) / SMP_PER_OCTAVE) * (float)SMP_LEAST;
        const uint32_t v = s.by_p ? (uint32_t)fminf(fmaxf(w + 0.5f, (float)SMP_LEAST), (float)SMP_MOST) : 1;
        if (x[j] != SMP_NONE && b < SMP_BINS) atomicAdd(&s_hist[b], v);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SMP_BINS / SMP_WG; ++i) ws.hist[chunk * SMP_BINS + i * SMP_WG + tid] = s_hist[i * SMP_WG + tid];
}

// ---------------------------------------------------------------- find

__global__ __launch_bounds__(SMP_SEQ_WG) void k_sample_find(const llapis_sample_args a, const SmpWs ws) {
    __shared__ uint64_t s_best[SMP_SEQ_WAVES];
    __shared__ int s_few[SMP_SEQ_WAVES], s_many[SMP_SEQ_WAVES], s_at[4];
    __shared__ float s_sum[SMP_SEQ_WAVES], s_mass[2];
    const int seq = blockIdx.x, tid = threadIdx.x;
    const SmpSet s = smp_settings(a, seq);
    const SmpChunk * chunks = ws.chunks + (int64_t)seq * ws.n_chunks;
    uint64_t best = 0;
    for (int c = tid; c < ws.n_chunks; c += SMP_SEQ_WG) {
        const uint64_t key = smp_key(chunks[c].top, chunks[c].at);
        best = key > best ? key : best;
    }
    smp_leave(smp_wave(best, SmpMax()), s_best);
    if (tid < 4) s_at[tid] = SMP_BINS - 1;
    __syncthreads();
    best = smp_all<SMP_SEQ_WAVES>(s_best, SmpMax());
    const float top = smp_value(best), none = __builtin_nanf(""), least = -3.40282347e38f;
    // without filters every value is surely kept
    SmpCut cut = {top, least, none, none, none, top == SMP_NONE ? -1 : smp_index(best), ~0ull, 0.0};
    if (s.greedy || top == SMP_NONE || !(s.by_k || s.by_p)) {
        if (tid == 0) ws.cuts[seq] = cut;
        return;
    }
    // ---- a thread's bin over all chunks
    const float top_bin = floorf(top * s.bins);
    uint64_t held_all = 0;
    const uint32_t * hist = ws.hist + (int64_t)seq * ws.n_chunks * SMP_BINS;
    constexpr int MANY = 16;                               // loads under way, then their use: in the compiler's own order each is waited for
    for (int c0 = 0; c0 < ws.n_chunks; c0 += MANY) {
        int b[MANY];
        uint32_t held[MANY];
#pragma unroll
        for (int i = 0; i < MANY; ++i) {
            const int c = min(c0 + i, ws.n_chunks - 1);
            b[i] = tid - smp_bin(chunks[c].top, top, top_bin, s.bins);
            held[i] = hist[(int64_t)c * SMP_BINS + max(b[i], 0)];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < MANY; ++i) {
            held_all += b[i] < 0 || c0 + i >= ws.n_chunks ? 0 : held[i];
        }
    }
    // the number of values, between two, and the sum of their weights.  fp32 has a value's place to 2^-23 of its
    // distance from 0; the words' rounding and the sums' are less than the last factor
    const int many = s.by_p ? (int)(held_all / SMP_LEAST) : (int)held_all;
    const int few = s.by_p ? (int)((double)held_all * ((1.0 - 0x1p-40) / SMP_MOST)) : many;
    const float off = exp2f((fabsf(top * s.bins) + 2 * SMP_BINS) * 0x1p-22f / SMP_PER_OCTAVE) * (1.0f + 0x1p-16f);
    const float mass = exp2f((top_bin - top * s.bins - (float)tid) / SMP_PER_OCTAVE) * ((float)held_all / (float)SMP_LEAST);
    const int few_w = smp_wave(few, SmpAdd()), many_w = smp_wave(many, SmpAdd());
    const float mass_w = smp_wave(mass, SmpAdd());
    smp_leave(few_w, s_few);
    smp_leave(many_w, s_many);
    smp_leave(mass_w, s_sum);
    __syncthreads();
    int few_all, many_all;
    float mass_all;
    const int few_upto = smp_before<SMP_SEQ_WAVES>(s_few, few_all) + few_w;
    const int many_upto = smp_before<SMP_SEQ_WAVES>(s_many, many_all) + many_w;
    const float mass_upto = smp_before<SMP_SEQ_WAVES>(s_sum, mass_all) + mass_w;
    const bool spread = s.bins > 0.0f && fabsf(top * s.bins) < __builtin_inff();      // else the bins say nothing
    // top_k ends in bins k_lo .. k_hi (in the last without one)
    int k_lo = SMP_BINS - 1, k_hi = SMP_BINS - 1;
    if (s.by_k) {
        smp_first(many_upto >= s.k, &s_at[2]);
        smp_first(few_upto >= s.k, &s_at[3]);
        __syncthreads();
        k_lo = spread ? s_at[2] : 0;
        k_hi = spread ? s_at[3] : k_hi;
    }
    int lo = k_lo, hi = k_hi;
    if (s.by_p) {
        // the first bin in which the sum may, and in which it must have reached top_p's part of what top_k leaves
        if (tid == k_lo) s_mass[0] = s.by_k ? mass_upto - mass : mass_all;
        if (tid == k_hi) s_mass[1] = s.by_k ? mass_upto : mass_all;
        __syncthreads();
        const float p = (float)s.p;
        smp_first(mass_upto * off >= p * s_mass[0] / off, &s_at[0]);
        smp_first(mass_upto / off >= p * s_mass[1] * off, &s_at[1]);
        __syncthreads();
        lo = spread ? min(s_at[0], k_lo) : 0;
        hi = spread ? min(s_at[1], k_hi) : k_hi;
        if (hi >= k_lo) hi = k_hi;                         // one window for both
    }
    // ---- the least value of bins lo - 1, hi, k_lo - 1 (without a top_k: k_hi) and k_hi, by bisection of the
    // values' order; a lane each
    const int of = tid == 0 ? lo - 1 : tid == 1 ? hi : tid == 2 ? (s.by_k ? k_lo - 1 : k_hi) : k_hi;
    uint32_t below = (uint32_t)(smp_key(least, 0) >> 32) - 1, from = (uint32_t)(smp_key(top, 0) >> 32);
    if (tid < 4) {
        auto try_at = [&](uint32_t at) {
            if (smp_bin(smp_value((uint64_t)at << 32), top, top_bin, s.bins) <= of) from = at;
            else below = at;
        };
        // the quotient is next to it: where it is, 5 steps remain of 32
        const float near = (top_bin - (float)of) / s.bins;
        const uint32_t at = (uint32_t)(smp_key(near, 0) >> 32);
        if (near == near && at - 8 > below && at - 8 < from) try_at(at - 8);
        if (near == near && at + 8 > below && at + 8 < from) try_at(at + 8);
        while (from - below > 1) try_at(below + (from - below) / 2);
    }
    if (tid < 64) {
        const float x = of < 0 ? none : smp_value((uint64_t)from << 32);
        cut.x_sure = smp_lane(x, 0);
        cut.x_cand = smp_lane(x, 1);
        // (in one window there are no values between)
        cut.x_mid = hi == k_hi ? cut.x_cand : smp_lane(x, 2);
        cut.x_end = hi == k_hi ? cut.x_cand : smp_lane(x, 3);
        if (tid == 0) ws.cuts[seq] = cut;
    }
}

// --------------------------------------------------------------- split

template <class T, int N>
__global__ __launch_bounds__(SMP_WG) void k_sample_split(const llapis_sample_args a, const SmpWs ws) {
    const int seq = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const SmpSet s = smp_settings(a, seq);
    if (s.greedy) return;
    const int base = blockIdx.x * smp_chunk(N) + wave * smp_seg(N);
    const SmpCut cut = ws.cuts[seq];
    if (cut.token < 0) return;
    SmpSeg g = {0.0, 0.0, 0.0, 0, 0, 0, 0};
    const int64_t seg = ((int64_t)seq * ws.n_chunks + blockIdx.x) * SMP_WAVES + wave;
    uint64_t * list = ws.keys + seg * smp_seg(N);
    smp_stream<T, N>((const T *)a.logits + seq * a.logits_stride, base, a.vocab, [&](int at, const auto & x) {
        constexpr int W = 16 / sizeof(T);
#pragma unroll
        for (int j0 = 0; j0 < W; j0 += 2) {                // (the two chains of multiply-adds overlap)
            bool sure[2], mid[2], cand[2];
            uint64_t any = 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float y = x[j0 + j];
                sure[j] = y >= cut.x_sure;
                mid[j] = !sure[j] && y >= cut.x_mid && y < cut.x_cand;
                cand[j] = !sure[j] && y >= cut.x_end && !mid[j];
                const uint64_t n_sure = __ballot(sure[j]), n_mid = __ballot(mid[j]);
                g.n_sure += __popcll(n_sure);
                g.n_mid += __popcll(n_mid);
                any |= n_sure | n_mid;
            }
            if (any) {
                double w[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) w[j] = smp_weight(x[j0 + j], cut.top, s.octaves);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    g.sure += sure[j] ? w[j] : 0.0;
                    g.draw += sure[j] && w[j] >= s.min_p ? w[j] : 0.0;
                    g.mid += mid[j] ? w[j] : 0.0;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint64_t votes = __ballot(cand[j]);
                if (cand[j]) list[g.n_cand + __popcll(votes & ((1ull << lane) - 1))] = smp_key(x[j0 + j], at + j0 + j);
                g.n_cand += __popcll(votes);
            }
        }
    });
    g.sure = smp_wave(g.sure, SmpAdd());
    g.draw = smp_wave(g.draw, SmpAdd());
    g.mid = smp_wave(g.mid, SmpAdd());
    if (lane == 63) ws.segs[seg] = g;
}

// ---------------------------------------------------------------- pick

// short rows, whose barriers are what it costs, take fewer waves
constexpr int smp_pick_wg(int lane_values) { return lane_values < 32 ? 256 : 1024; }

template <class T, int N>
__global__ __launch_bounds__(smp_pick_wg(N)) void k_sample_pick(const llapis_sample_args a, const SmpWs ws) {
    constexpr int WG = smp_pick_wg(N), WAVES = WG / 64, SEG = smp_seg(N), HOLD = SMP_HOLD, FEW = HOLD * WG, LIST = WG;
    __shared__ double s_sure[WAVES], s_mid[WAVES], s_sum[2][WAVES];
    __shared__ int s_n[3][WAVES], s_count[WAVES], s_digit[256];
    __shared__ uint64_t s_mass[WAVES];
    __shared__ int64_t s_parts[2][WAVES];
    __shared__ SmpAbove s_above;
    __shared__ int s_first[WG + 1], s_bucket_n[WG], s_list_n, s_found, s_last;
    __shared__ unsigned long long s_bucket[WG], s_kept[WG], s_weigh[2][256], s_all_k;
    __shared__ uint64_t s_list[LIST], s_list_w[LIST], s_key;
    __shared__ unsigned long long s_upto[LIST];
    __shared__ struct { int bucket, before, n; uint64_t mass; } s_sel;
    __shared__ double s_before;
    const int seq = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const SmpSet s = smp_settings(a, seq);
    const SmpCut cut = ws.cuts[seq];
    if (s.greedy || cut.token < 0) {
        if (tid == 0) a.tokens[seq] = cut.token;
        return;
    }
    const int n_segs = (a.vocab + SEG - 1) / SEG, per = (n_segs + WG - 1) / WG;
    const int64_t seg0 = (int64_t)seq * ws.n_chunks * SMP_WAVES;
    SmpSeg * segs = ws.segs + seg0;
    const uint64_t * keys = ws.keys + seg0 * SEG;
    auto weight = [&](uint64_t key) { return smp_weight(smp_value(key), cut.top, s.octaves); };
    // ---- a thread's segments are consecutive
    double sure = 0.0, mid = 0.0, draw = 0.0;
    int n_sure = 0, n_mid = 0, n_mine = 0;
    for (int i = tid * per; i < min((tid + 1) * per, n_segs); ++i) {
        const SmpSeg g = segs[i];
        sure += g.sure;
        mid += g.mid;
        draw += g.draw;
        n_sure += g.n_sure;
        n_mid += g.n_mid;
        n_mine += g.n_cand;
    }
    const int cand_w = smp_wave(n_mine, SmpAdd());
    smp_leave(cand_w, s_n[0]);
    smp_leave(smp_wave(n_sure, SmpAdd()), s_n[1]);
    smp_leave(smp_wave(n_mid, SmpAdd()), s_n[2]);
    smp_leave(smp_wave(sure, SmpAdd()), s_sure);
    smp_leave(smp_wave(mid, SmpAdd()), s_mid);
    s_bucket_n[tid] = 0;
    s_bucket[tid] = 0;
    s_kept[tid] = 0;
    if (tid == 0) {
        s_list_n = 0;
        s_all_k = 0;
        s_found = 0x7FFFFFFF;
        s_last = -1;
    }
    __syncthreads();
    int n_cand;
    const int first = smp_before<WAVES>(s_n[0], n_cand) + cand_w - n_mine;
    uint64_t key = ~0ull;                                  // the last that is kept
    if (n_cand > 0) {
        n_sure = smp_all<WAVES>(s_n[1], SmpAdd());
        n_mid = smp_all<WAVES>(s_n[2], SmpAdd());
        sure = smp_all<WAVES>(s_sure, SmpAdd());
        mid = smp_all<WAVES>(s_mid, SmpAdd());
        // candidates within top_k, the first of them in order
        const int n_k = s.by_k ? max(min(s.k - n_sure - n_mid, n_cand), 0) : n_cand;
        // the largest weight that a candidate may have
        const float upper = cut.x_sure == cut.x_sure ? cut.x_sure : cut.top;
        const double upper_w = smp_weight(upper, cut.top, s.octaves);
        const int sum_bits = n_cand > 1 ? 32 - __builtin_clz(n_cand - 1) : 0;      // 2^sum_bits candidates at most
        // Held at once, weights are one word, cut off at 2^(sum_bits - 62) of the largest, which moves the border by at
        // most n_cand^2 of that / (1 - top_p) of its values: 2^-5 here.  (All 8192 up to a top_p of 1 - 2^-17; 1 row of 131072
        // at 0.999999 47 us, digit by digit 76)
        bool few = n_cand <= FEW && per == 1 && (!s.by_p || (double)n_cand * n_cand * n_cand <= 0x1p56 * (1.0 - s.p));
        if (few) {
            // ---- the candidates in registers, and in buckets by value, thread b's the b-th from above.
            // Weights are whole numbers, of 2^-49 of the largest that a candidate may have, or less
            const double scale = __builtin_ldexp(1.0, 62 - sum_bits) / upper_w;
            if (tid < n_segs) s_first[tid] = first;
            if (tid == 0) s_first[n_segs] = n_cand;
            __syncthreads();
            const bool two = cut.x_end < cut.x_mid;         // candidates of top_k's end apart
            const int n_upper = two ? WG / 2 : WG;
            const double per_upper = n_upper / fmax((double)upper - (double)cut.x_cand, 1e-300);
            const double per_lower = (WG / 2) / fmax((double)cut.x_mid - (double)cut.x_end, 1e-300);
            uint64_t k[HOLD];
            unsigned long long w[HOLD];
            int bucket[HOLD], seg_of[HOLD];
#pragma unroll
            for (int e = 0; e < HOLD; ++e) {
                const int r = tid + e * WG;
                k[e] = 0;
                w[e] = 0;
                bucket[e] = -1;
                seg_of[e] = 0;
                if (r < n_cand) {
                    int l = 0;
                    for (int h = n_segs; h - l > 1;) {
                        const int mid_seg = (l + h) >> 1;
                        if (s_first[mid_seg] <= r) l = mid_seg;
                        else h = mid_seg;
                    }
                    seg_of[e] = l;
                    k[e] = keys[(int64_t)l * SEG + r - s_first[l]];
                }
            }
#pragma unroll 1
            for (int e = 0; e < HOLD && e * WG < n_cand; ++e) {
                uint64_t u = 0;
#pragma unroll
                for (int i = 0; i < HOLD; ++i) u = i == e ? k[i] : u;
                if (u) {
                    const float x = smp_value(u);
                    const unsigned long long y = (unsigned long long)(weight(u) * scale);
                    const bool above = !two || x >= cut.x_cand;
                    const double at = ((double)(above ? upper : cut.x_mid) - (double)x) * (above ? per_upper : per_lower);
                    const int most = above ? n_upper - 1 : WG / 2 - 1;
                    // (the largest of all may be infinite: it is first)
                    const int b = x == upper ? 0 : (above ? 0 : n_upper) + (int)fmin(fmax(at, 0.0), (double)most);
#pragma unroll
                    for (int i = 0; i < HOLD; ++i)
                        if (i == e) {
                            bucket[i] = b;
                            w[i] = y;
                        }
                    atomicAdd(&s_bucket_n[b], 1);
                    atomicAdd(&s_bucket[b], y);
                }
            }
            __syncthreads();
            const int b_n = s_bucket_n[tid];
            const uint64_t b_mass = s_bucket[tid];
            const int b_n_w = smp_wave(b_n, SmpAdd());
            const uint64_t b_mass_w = smp_wave(b_mass, SmpAdd());
            smp_leave(b_n_w, s_count);
            smp_leave(b_mass_w, s_mass);
            __syncthreads();
            int all_n;
            uint64_t all_mass;
            const int n_upto = smp_before<WAVES>(s_count, all_n) + b_n_w;
            const uint64_t mass_upto = smp_before<WAVES>(s_mass, all_mass) + b_mass_w;
            // ---- the bucket that a filter ends in, then the key: top_k's by number, top_p's by weight
            uint64_t all_k = all_mass;
            key = n_k > 0 ? 0 : ~0ull;
            for (int pass = n_k < n_cand ? 0 : 1; pass < (s.by_p ? 2 : 1) && n_k > 0 && few; ++pass) {
                const double whole = sure + mid + (double)all_k / scale;
                const uint64_t goal = (uint64_t)ceil(fmax(s.p * whole - sure, 0.0) * scale);
                const bool mine = b_n > 0 && (pass == 0 ? n_upto >= n_k && n_upto - b_n < n_k : mass_upto >= goal && (mass_upto - b_mass < goal || n_upto == b_n));
                if (tid == 0) s_sel.bucket = -1;
                __syncthreads();
                if (mine) s_sel = {tid, n_upto - b_n, b_n, mass_upto - b_mass};
                __syncthreads();
                if (s_sel.bucket < 0) break;               // the weight of all is not top_p's part by a rounding: all are kept
                const int n = s_sel.n;
                if (n > LIST) {
                    few = false;
                    break;
                }
#pragma unroll
                for (int e = 0; e < HOLD; ++e) {
                    if (bucket[e] == s_sel.bucket) {
                        const int i = atomicAdd(&s_list_n, 1);
                        s_list[i] = k[e];
                        s_list_w[i] = w[e];
                        s_upto[i] = 0;
                    }
                }
                __syncthreads();
                // a key's rank in the list, or the mass of it and those above it: the list in parts, as many as there are threads for
                const int slots = (n + 63) & ~63, parts = WG / slots, part = tid / slots, at = tid - part * slots;
                if (at < n && part < parts) {
                    const uint64_t u = s_list[at];
                    uint64_t upto = 0;
                    if (pass == 0) {
#pragma unroll 4
                        for (int i = part; i < n; i += parts) upto += s_list[i] >= u;
                    } else {
#pragma unroll 4
                        for (int i = part; i < n; i += parts) upto += s_list[i] >= u ? s_list_w[i] : 0;
                    }
                    atomicAdd(&s_upto[at], (unsigned long long)upto);
                }
                __syncthreads();
                if (tid < n) {
                    const uint64_t mass = s_list_w[tid], upto = s_upto[tid];
                    if (pass == 0) {
                        const int rank = s_sel.before + (int)upto;
                        if (rank <= n_k) atomicAdd(&s_all_k, (unsigned long long)mass);
                        if (rank == n_k) s_key = s_list[tid];
                    } else {
                        const uint64_t g = goal > s_sel.mass ? goal - s_sel.mass : 0;
                        if (upto >= g && (upto - mass < g || upto == mass)) s_key = s_list[tid];
                    }
                }
                __syncthreads();
                if (pass == 0) all_k = s_sel.mass + s_all_k;
                key = s_key > key ? s_key : key;
                if (tid == 0) s_list_n = 0;
                __syncthreads();
            }
            // ---- the segments' kept weights
            if (few) {
#pragma unroll 1
                for (int e = 0; e < HOLD && e * WG < n_cand; ++e) {
                    uint64_t u = 0;
                    unsigned long long y = 0;
                    int at = 0;
#pragma unroll
                    for (int i = 0; i < HOLD; ++i)
                        if (i == e) {
                            u = k[i];
                            y = w[i];
                            at = seg_of[i];
                        }
                    if (u && u >= key && (s.min_p == 0.0 || weight(u) >= s.min_p)) atomicAdd(&s_kept[at], y);
                }
                __syncthreads();
                draw += (double)s_kept[tid] / scale;
            }
        }
        if (!few) {
            // ---- too many at once: eight bits of the key at a time, the candidates counted (and
            // weighed) by them: the first key at which the number or the weight of what is not below
            // it reaches the goal.  A weight is two whole numbers, of 2^-bits of the largest that a candidate may have and
            // of 2^-2bits, as many bits as leave room for the sums (43 for 2^19 candidates): the border may
            // lie far below the largest, and what one weight is cut by all of them are
            const int bits = min(50, 62 - sum_bits);
            const double one = __builtin_ldexp(1.0, bits), scale = one / upper_w;
            // to nearest, the second of either sign (a number below 2^51 is in the low bits of its sum with 1.5 2^52)
            auto parts = [&](double v, int64_t & hi, int64_t & lo) {
#pragma clang fp contract(off)                             // (a weight is the same wherever it is added)
                const double near = v + 0x1.8p52, rest = (v - (near - 0x1.8p52)) * one + 0x1.8p52;
                hi = __builtin_bit_cast(int64_t, near) - __builtin_bit_cast(int64_t, 0x1.8p52);
                lo = __builtin_bit_cast(int64_t, rest) - __builtin_bit_cast(int64_t, 0x1.8p52);
            };
            // f(key) of each candidate, a wave a segment; lane l knows the number of the wave's l-th segment from here
            auto each = [&](auto f) {
                for (int i0 = wave; i0 < n_segs; i0 += 64 * WAVES) {
                    const int there = min((n_segs - i0 + WAVES - 1) / WAVES, 64);
                    const int n_mine = lane < there ? segs[i0 + lane * WAVES].n_cand : 0;
                    for (int l = 0; l < there; ++l) {
                        const int n = smp_lane(n_mine, __builtin_amdgcn_readfirstlane(l));
                        const uint64_t * list = keys + (int64_t)(i0 + l * WAVES) * SEG;
                        for (int c = lane; c < n; c += 64) f(list[c]);
                    }
                }
            };
            int64_t want_hi = 0, want_lo = 0;
            key = n_k > 0 ? 0 : ~0ull;
            for (int pass = n_k < n_cand ? 0 : 1; pass < (s.by_p ? 2 : 1) && n_k > 0; ++pass) {
                const bool by_mass = pass == 1;
                if (by_mass) {
                    int64_t hi = 0, lo = 0, all_hi, all_lo;
                    each([&](uint64_t u) {
                        int64_t y, y_lo;
                        parts(u >= key ? weight(u) * scale : 0.0, y, y_lo);
                        hi += y;
                        lo += y_lo;
                    });
                    __syncthreads();
                    smp_scan<WAVES>(hi, s_parts[0], all_hi);
                    smp_scan<WAVES>(lo, s_parts[1], all_lo);
                    const double all_k = ((double)all_hi + (double)all_lo / one) / scale;
                    const double goal = fmax(s.p * (sure + mid + all_k) - sure, 0.0) * scale;
                    want_hi = (int64_t)goal;
                    want_lo = (int64_t)ceil((goal - (double)want_hi) * one);
                }
                uint64_t prefix = 0;
                SmpAbove above = {0, 0, 0};
                for (int shift = 56; shift >= 0; shift -= 8) {
                    __syncthreads();
                    if (tid < 256) {
                        s_digit[tid] = 0;
                        s_weigh[0][tid] = 0;
                        s_weigh[1][tid] = 0;
                    }
                    if (tid == 0) {
                        s_found = 0x7FFFFFFF;
                        s_last = -1;
                    }
                    __syncthreads();
                    // (equal values have equal digits: a thread adds them up before it adds them to the others')
                    int at = 0, n_at = 0;
                    int64_t at_hi = 0, at_lo = 0;
                    auto add = [&]() {
                        if (n_at) atomicAdd(&s_digit[at], n_at);
                        if (n_at && by_mass) {
                            atomicAdd(&s_weigh[0][at], (unsigned long long)at_hi);
                            atomicAdd(&s_weigh[1][at], (unsigned long long)at_lo);
                        }
                        n_at = 0;
                        at_hi = at_lo = 0;
                    };
                    each([&](uint64_t u) {
                        if (shift < 56 && (u >> (shift + 8)) != (prefix >> (shift + 8))) return;
                        const int d = (int)(u >> shift) & 255;
                        if (d != at) add();
                        at = d;
                        ++n_at;
                        if (by_mass) {
                            int64_t y, y_lo;
                            parts(weight(u) * scale, y, y_lo);
                            at_hi += y;
                            at_lo += y_lo;
                        }
                    });
                    add();
                    __syncthreads();
                    // thread t's digit is the t-th from above; the first that there is whose sum reaches the goal, else the last
                    const int n_d = tid < 256 ? s_digit[255 - tid] : 0;
                    const int64_t hi_d = tid < 256 ? (int64_t)s_weigh[0][255 - tid] : 0, lo_d = tid < 256 ? (int64_t)s_weigh[1][255 - tid] : 0;
                    const int n_w = smp_wave(n_d, SmpAdd());
                    const int64_t hi_w = smp_wave(hi_d, SmpAdd()), lo_w = smp_wave(lo_d, SmpAdd());
                    smp_leave(n_w, s_n[0]);
                    smp_leave(hi_w, s_parts[0]);
                    smp_leave(lo_w, s_parts[1]);
                    __syncthreads();
                    int n_all;
                    int64_t hi_all, lo_all;
                    const int n_upto = above.n + smp_before<WAVES>(s_n[0], n_all) + n_w;
                    const int64_t hi_upto = above.hi + smp_before<WAVES>(s_parts[0], hi_all) + hi_w;
                    const int64_t lo_upto = above.lo + smp_before<WAVES>(s_parts[1], lo_all) + lo_w;
                    const int64_t whole = hi_upto + (lo_upto >> bits), rest = lo_upto & ((1ll << bits) - 1);
                    const bool reached = by_mass ? whole > want_hi || (whole == want_hi && rest >= want_lo) : n_upto >= n_k;
                    smp_first(n_d > 0 && reached, &s_found);
                    const uint64_t any = __ballot(n_d > 0);
                    if (any && lane == 0) atomicMax(&s_last, tid + 63 - (int)__builtin_clzll(any));
                    __syncthreads();
                    const int who = s_found != 0x7FFFFFFF ? s_found : s_last;
                    if (tid == who) s_above = {n_upto - n_d, hi_upto - hi_d, lo_upto - lo_d};
                    __syncthreads();
                    above = s_above;
                    prefix |= (uint64_t)(255 - who) << shift;
                }
                key = prefix > key ? prefix : key;
            }
            for (int i = wave; i < n_segs; i += WAVES) {
                const int n = segs[i].n_cand;
                double sum = 0.0;
                for (int c = lane; c < n; c += 64) {
                    const uint64_t u = keys[(int64_t)i * SEG + c];
                    const double y = u >= key ? weight(u) : 0.0;
                    sum += y >= s.min_p ? y : 0.0;
                }
                sum = smp_lane(smp_wave(sum, SmpAdd()), 63);
                if (lane == 0) segs[i].draw += sum;
            }
            if (tid == 0) {
                s_found = 0x7FFFFFFF;
                s_last = -1;
            }
            __syncthreads();
            draw = 0.0;
            for (int i = tid * per; i < min((tid + 1) * per, n_segs); ++i) draw += segs[i].draw;
        }
    }
    // ---- the first thread in whose segments the sum passes the goal; without one
    // (rounding, u of 1 and more) the last that has anything
    double total;
    double cum = smp_scan<WAVES>(draw, s_sum[1], total);
    const double goal = (double)a.u[seq] * total;
    const uint64_t any = __ballot(draw > 0.0);
    if (any && lane == 0) atomicMax(&s_last, tid + 63 - (int)__builtin_clzll(any));
    smp_first(draw > 0.0 && cum + draw > goal, &s_found);
    __syncthreads();
    const bool found = s_found != 0x7FFFFFFF;
    const int who = found ? s_found : s_last;
    __syncthreads();
    if (tid == who) {
        int seg = tid;
        if (per > 1) {
            seg = -1;
            for (int i = tid * per; i < min((tid + 1) * per, n_segs); ++i) {
                const double y = segs[i].draw;
                if (!(y > 0.0)) continue;
                seg = i;
                s_before = cum;
                cum += y;
                if (found && cum > goal) break;
            }
        } else {
            s_before = cum;
        }
        s_found = seg;
    }
    if (tid == 0) {
        s_last = -1;
        s_list_n = 0x7FFFFFFF;
    }
    __syncthreads();
    // ---- the token: consecutive values a thread
    constexpr int E = (SEG + WG - 1) / WG;
    const int at = s_found * SEG + tid * E, end = min(s_found * SEG + SEG, a.vocab);
    const T * row = (const T *)a.logits + seq * a.logits_stride;
    double w[E], sum = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float x = at + i < end ? smp_clean((float)row[at + i]) : SMP_NONE;
        const bool keep = x >= cut.x_sure || (x >= cut.x_end && !(x >= cut.x_mid && x < cut.x_cand) && smp_key(x, at + i) >= key);
        w[i] = keep ? smp_weight(x, cut.top, s.octaves) : 0.0;
        if (w[i] < s.min_p) w[i] = 0.0;
        sum += w[i];
    }
    double part;
    cum = s_before + smp_scan<WAVES>(sum, s_sum[0], part);
    int token = -1, last = -1;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        cum += w[i];
        if (w[i] > 0.0) {
            last = at + i;
            if (token < 0 && found && cum > goal) token = at + i;
        }
    }
    // the lowest that passes, else the last that has a weight
    const uint64_t passes = __ballot(token >= 0), has = __ballot(last >= 0);
    if (passes) {
        token = __builtin_amdgcn_readlane(token, __builtin_ctzll(passes));
        if (lane == 0) atomicMin(&s_list_n, token);
    }
    if (has) {
        last = __builtin_amdgcn_readlane(last, 63 - __builtin_clzll(has));
        if (lane == 0) atomicMax(&s_last, last);
    }
    __syncthreads();
    if (tid == 0) {
        a.tokens[seq] = s_list_n != 0x7FFFFFFF ? s_list_n : s_last;
        ws.cuts[seq].key = key;
        ws.cuts[seq].total = total;
    }
}

// --------------------------------------------------------------- probs

template <class T, int N>
__global__ __launch_bounds__(SMP_WG) void k_sample_probs(const llapis_sample_args a, const SmpWs ws) {
    const int seq = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
    const SmpSet s = smp_settings(a, seq);
    const int base = blockIdx.x * smp_chunk(N) + wave * smp_seg(N);
    if (base >= a.vocab) return;
    const SmpCut cut = ws.cuts[seq];
    const double inv = 1.0 / cut.total;
    T * out = (T *)a.probs + seq * a.probs_stride;
    smp_stream<T, N>((const T *)a.logits + seq * a.logits_stride, base, a.vocab, [&](int at, const auto & x) {
        constexpr int W = 16 / sizeof(T);
        typename SmpVec<T>::v p;
#pragma unroll
        for (int j0 = 0; j0 < W; j0 += 2) {
            bool keep[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float y = x[j0 + j];
                keep[j] = !s.greedy && (y >= cut.x_sure || (y >= cut.x_end && !(y >= cut.x_mid && y < cut.x_cand) && smp_key(y, at + j0 + j) >= cut.key));
                p[j0 + j] = (T)(s.greedy && at + j0 + j == cut.token ? 1.0f : 0.0f);
            }
            if (__ballot(keep[0] || keep[1])) {
                double w[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) w[j] = smp_weight(x[j0 + j], cut.top, s.octaves);
#pragma unroll
                for (int j = 0; j < 2; ++j) p[j0 + j] = keep[j] && w[j] >= s.min_p ? (T)(w[j] * inv) : p[j0 + j];
            }
        }
        if (at + W <= a.vocab) {
            *(typename SmpVec<T>::v *)(out + at) = p;
        } else {
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (at + j < a.vocab) out[at + j] = p[j];
        }
    });
}

}  // namespace dev

using namespace dev;

namespace {

constexpr int SMP_MAX_SEQ = 65535, SMP_MAX_VOCAB = 1 << 30;

int32_t refuse_sample(const char * why) noexcept {
    char msg[256];
    snprintf(msg, sizeof msg, "llapis_sample: %s", why);
    return refuse(msg);
}

uint64_t round_up(uint64_t n) { return (n + 255) / 256 * 256; }

// Values of a lane: 8 where a call's rows leave most of the card without work at 32 (1 row of 32003: 23 us, at 32
// values 32; 64 rows: 31 and 36), but k_sample_find adds four times the histograms then (16 rows of 128001: 37 us and
// 34; 8 of 262144: 51 and 39)
constexpr int SMP_SHORT = 1 << 16;
constexpr int64_t SMP_SHORT_ALL = 1 << 21;
bool short_rows(int n_seq, int vocab) { return vocab <= SMP_SHORT && (int64_t)n_seq * vocab <= SMP_SHORT_ALL; }

// the workspace's parts for `chunks` chunks of n_seq sequences; its size
uint64_t sample_parts(uint64_t n_seq, uint64_t chunks, int lane_values, uint8_t * at, SmpWs & ws) {
    uint64_t n = 0;
    auto part = [&](uint64_t bytes) {
        uint8_t * p = at ? at + n : nullptr;
        n += round_up(bytes);
        return p;
    };
    ws.cuts = (SmpCut *)part(n_seq * sizeof(SmpCut));
    ws.chunks = (SmpChunk *)part(chunks * sizeof(SmpChunk));
    ws.segs = (SmpSeg *)part(chunks * SMP_WAVES * sizeof(SmpSeg));
    ws.hist = (uint32_t *)part(chunks * SMP_BINS * 4);
    ws.keys = (uint64_t *)part(chunks * smp_chunk(lane_values) * 8);
    return n;
}

int chunks_of(int vocab, int lane_values) { return (vocab + smp_chunk(lane_values) - 1) / smp_chunk(lane_values); }

// ... of the long chunks, and of the most short ones that a call of no more sequences and values has
uint64_t sample_bytes(int n_seq, int vocab) {
    SmpWs ws;
    const uint64_t few = std::min<uint64_t>((uint64_t)n_seq * chunks_of(std::min(vocab, SMP_SHORT), 8), SMP_SHORT_ALL / smp_chunk(8) + n_seq);
    return std::max(sample_parts(n_seq, (uint64_t)n_seq * chunks_of(vocab, 32), 32, nullptr, ws), sample_parts(n_seq, few, 8, nullptr, ws));
}

template <class T, int N>
hipError_t launch_sample(const llapis_sample_args & a, void * workspace, hipStream_t s) {
    SmpWs ws;
    ws.n_chunks = chunks_of(a.vocab, N);
    sample_parts(a.n_seq, (uint64_t)a.n_seq * ws.n_chunks, N, (uint8_t *)workspace, ws);
    const dim3 grid(ws.n_chunks, a.n_seq), wg(SMP_WG), each(a.n_seq), seq_wg(SMP_SEQ_WG), pick_wg(smp_pick_wg(N));
    hipError_t e;
    hipLaunchKernelGGL((k_sample_scan<T, N>), grid, wg, 0, s, a, ws);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL(k_sample_find, each, seq_wg, 0, s, a, ws);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((k_sample_split<T, N>), grid, wg, 0, s, a, ws);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((k_sample_pick<T, N>), each, pick_wg, 0, s, a, ws);
    if ((e = hipGetLastError()) != hipSuccess || !a.probs) return e;
    hipLaunchKernelGGL((k_sample_probs<T, N>), grid, wg, 0, s, a, ws);
    return hipGetLastError();
}

template <class T>
hipError_t launch_sample(const llapis_sample_args & a, void * workspace, hipStream_t s) {
    return short_rows(a.n_seq, a.vocab) ? launch_sample<T, 8>(a, workspace, s) : launch_sample<T, 32>(a, workspace, s);
}

}  // namespace
}  // namespace llapis

using namespace llapis;

extern "C" {

uint64_t llapis_sample_workspace_size(int32_t n_seq, int32_t vocab) {
    return n_seq <= 0 || n_seq > SMP_MAX_SEQ || vocab <= 0 || vocab > SMP_MAX_VOCAB ? 0 : sample_bytes(n_seq, vocab);
}

int32_t llapis_sample(const llapis_sample_args * a, void * workspace, uint64_t ws_bytes, void * stream) {
    if (!a) return refuse_sample("null arguments");
    if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) return refuse_sample("need type F32, F16 or BF16");
    if (a->n_seq < 0 || a->n_seq > SMP_MAX_SEQ || a->vocab <= 0 || a->vocab > SMP_MAX_VOCAB)
        return refuse_sample("need 0 <= n_seq <= 65535, 0 < vocab <= 2^30");
    if (a->n_seq == 0) return 0;
    if (!a->logits || !a->u || !a->tokens) return refuse_sample("null logits, u or tokens");
    if (a->probs == a->logits) return refuse_sample("probs may not be the logits");
    if (a->n_seq > 1 && (a->logits_stride < a->vocab || (a->probs && a->probs_stride < a->vocab)))
        return refuse_sample("rows shorter than vocab");
    if (!workspace || ((uintptr_t)workspace & 15) || ws_bytes < llapis_sample_workspace_size(a->n_seq, a->vocab))
        return refuse_sample("workspace too small or not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a->type == T_F32 ? launch_sample<float>(*a, workspace, s)
                         : a->type == T_F16 ? launch_sample<_Float16>(*a, workspace, s) : launch_sample<__bf16>(*a, workspace, s);
    return e == hipSuccess ? 0 : refuse_sample(hipGetErrorString(e));
}

}  // extern "C"
