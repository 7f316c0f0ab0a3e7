// sample.hip -- the next token of each sequence from its logits (llapis_step.h).
//
// With M the largest logit a value's weight is w = e^((x - M) / T), and every
// filter keeps an upper part of the values in the order (value descending, index
// ascending).  Three kernels find where that part ends and draw from it, without
// sorting the row:
//   k_sample_scan   a chunk's largest value, and where a top_k or top_p is to be found
//                   a histogram of its values over SMP_BINS bins, 16 to a factor of 2
//                   of the weight: their numbers and (roughly) their weights
//   k_sample_cut    every workgroup adds the chunks' histograms, finds the few bins in
//                   which top_k and top_p may end, and sorts its values into those
//                   that are surely kept (summed), those that only count towards
//                   top_k's weight (summed), and the candidates of those bins (listed)
//   k_sample_pick   a workgroup a sequence orders the candidates, ends both filters
//                   among them exactly, and finds the token: its segment of 2048
//                   values by the segments' sums, then the value
// and k_sample_probs writes probabilities if they are wanted.  The histogram's weights
// are fp32 in fixed point: they only bound which bins are looked at, with a margin far
// above their error.  What decides is fp64: weights, their sums and products, in a
// fixed order, so that a draw next to a border falls as the definition says.
#include <algorithm>
#include <cstdio>

#include "kv.h"

namespace llapis {
namespace dev {

constexpr int SMP_WG = 1024, SMP_WAVES = SMP_WG / 64;
constexpr int SMP_LANE = 32;                              // values of a lane
constexpr int SMP_SEG = 64 * SMP_LANE;                    // ... of a wave: a segment
constexpr int SMP_CHUNK = SMP_WAVES * SMP_SEG;            // ... of a workgroup
constexpr int SMP_BINS = 1024, SMP_OUT = SMP_BINS + 1;     // a value below all bins is in SMP_OUT
constexpr double SMP_PER_OCTAVE = 16.0;
constexpr int SMP_SORT = 4096;                            // candidates that are sorted in LDS
// a histogram's word: the number of values (a chunk's at most) above 48 bits of their
// weights' sum, 32 of them its fraction, each weight rounded down
constexpr int SMP_COUNT_AT = 48;
constexpr float SMP_ONE = 4294967296.0f;
constexpr double SMP_LEAST = 1.0 / (1ull << 32);
constexpr double SMP_MARGIN = 1.0 / 4096;                 // of a weight, whose error in fp32 is below 2^-16

struct SmpChunk { float top; int32_t at; };               // a chunk's largest value and its lowest index
struct SmpSeg { double sure, draw, mid; int32_t n_sure, n_mid, n_cand, pad; };
// a sequence's cut; bins are counted from the largest value's
struct SmpCut {
    float top;                     // M
    int32_t lo, hi, last;          // candidates: bins lo .. hi and `last`, top_k's (SMP_BINS without one); those before lo are sure
    uint64_t key;                  // the last candidate that is kept, ~0 without one
    double total;                  // the kept weights' sum; 0: nothing to draw from
    int32_t token, pad;
};

struct SmpWs {
    SmpChunk * chunks;             // [n_seq][n_chunks]
    SmpSeg * segs;                 // [n_seq][n_chunks * SMP_WAVES]
    SmpCut * cuts;                 // [n_seq]
    uint64_t * hist;               // [n_seq][n_chunks][SMP_BINS]
    uint64_t * keys;               // [n_seq][n_chunks * SMP_CHUNK] candidates, by segment
    int n_chunks;
};

// a sequence's settings
struct SmpSet {
    bool greedy, by_k, by_p;       // the largest value alone; a number of values; a part of their weight
    int k;
    double inv_t, p, min_p;
    double per_bin;                // bins a unit of x
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
    s.inv_t = 1.0 / (double)t;
    s.per_bin = s.inv_t * (1.44269504088896340736 * SMP_PER_OCTAVE);
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

__device__ __forceinline__ double smp_weight(float x, float top, double inv_t) {
    // (the difference with an infinite M, or times an infinite 1 / T, says nothing)
    return x == top ? 1.0 : x == SMP_NONE || top == __builtin_inff() ? 0.0 : exp(((double)x - (double)top) * inv_t);
}
// bins below the largest value's
__device__ __forceinline__ int smp_bin(float x, float top, double per_bin) {
    return x == top ? 0 : (int)fmin(floor((double)top * per_bin) - floor((double)x * per_bin), (double)SMP_OUT);
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
template <class T>
__device__ __forceinline__ void smp_read(const T * row, int base, int n, float (&x)[SMP_LANE]) {
    constexpr int W = 16 / sizeof(T);
    if (base + SMP_SEG <= n) {
        typename SmpVec<T>::v w[SMP_LANE / W];
#pragma unroll
        for (int c = 0; c < SMP_LANE / W; ++c) w[c] = *(const typename SmpVec<T>::v *)(row + smp_at<T>(base, c * W));
#pragma unroll
        for (int j = 0; j < SMP_LANE; ++j) x[j] = smp_clean((float)w[j / W][j % W]);
    } else {
#pragma unroll
        for (int j = 0; j < SMP_LANE; ++j) {
            const int i = smp_at<T>(base, j);
            x[j] = i < n ? smp_clean((float)row[i]) : SMP_NONE;
        }
    }
}

__device__ __forceinline__ uint64_t smp_max(uint64_t x) {
    for (int o = 32; o; o >>= 1) {
        const uint64_t y = __shfl_xor(x, o, 64);
        x = y > x ? y : x;
    }
    return x;
}

// the largest over a workgroup; s_part is read before the next barrier
__device__ __forceinline__ uint64_t smp_max_wg(uint64_t x, uint64_t * s_part) {
    x = smp_max(x);
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < SMP_WAVES; ++w) x = s_part[w] > x ? s_part[w] : x;
    return x;
}

// exclusive sums over the workgroup's threads in order, and the whole
template <class V>
__device__ __forceinline__ V smp_scan(V x, V * s_part, V & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    V v = x;
    for (int o = 1; o < 64; o <<= 1) {
        const V y = __shfl_up(v, o, 64);
        if (lane >= o) v += y;
    }
    __syncthreads();                                     // the last use of s_part is over
    if (lane == 63) s_part[wave] = v;
    __syncthreads();
    V before = 0;
    total = 0;
    for (int w = 0; w < SMP_WAVES; ++w) {
        const V y = s_part[w];
        if (w < wave) before += y;
        total += y;
    }
    const V up = __shfl_up(v, 1, 64);
    return before + (lane ? up : (V)0);
}

template <class T>
__global__ __launch_bounds__(SMP_WG) void k_sample_scan(const llapis_sample_args a, const SmpWs ws) {
    __shared__ uint64_t s_hist[SMP_BINS];
    __shared__ uint64_t s_part[SMP_WAVES];
    const int seq = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
    const int64_t chunk = (int64_t)seq * ws.n_chunks + blockIdx.x;
    const int base = blockIdx.x * SMP_CHUNK + wave * SMP_SEG;
    float x[SMP_LANE];
    smp_read((const T *)a.logits + seq * a.logits_stride, base, a.vocab, x);
    const SmpSet s = smp_settings(a, seq);
    s_hist[tid] = 0;
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < SMP_LANE; ++j) {
        const uint64_t key = smp_key(x[j], smp_at<T>(base, j));
        best = key > best ? key : best;
    }
    best = smp_max_wg(best, s_part);
    const float top = smp_value(best);
    if (tid == 0) ws.chunks[chunk] = {top, smp_index(best)};
    if (s.greedy || !(s.by_k || s.by_p)) return;
    const float per = (float)(s.inv_t * 1.44269504088896340736);
    const double top_bin = floor((double)top * s.per_bin);
#pragma unroll
    for (int j = 0; j < SMP_LANE; ++j) {
        if (x[j] == SMP_NONE) continue;
        const int b = x[j] == top ? 0 : (int)fmin(top_bin - floor((double)x[j] * s.per_bin), (double)SMP_OUT);
        const float w = x[j] == top ? 1.0f : fmaxf(__builtin_amdgcn_exp2f((x[j] - top) * per), 0.0f);
        if (b < SMP_BINS) atomicAdd((unsigned long long *)&s_hist[b], 1ull << SMP_COUNT_AT | (unsigned long long)(w * SMP_ONE));
    }
    __syncthreads();
    ws.hist[chunk * SMP_BINS + tid] = s_hist[tid];
}

template <class T>
__global__ __launch_bounds__(SMP_WG) void k_sample_cut(const llapis_sample_args a, const SmpWs ws) {
    __shared__ uint64_t s_part[SMP_WAVES];
    __shared__ double s_sum[SMP_WAVES];
    __shared__ int s_count[SMP_WAVES], s_at[3];
    __shared__ double s_mass[2];
    const int seq = blockIdx.y, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const SmpSet s = smp_settings(a, seq);
    const SmpChunk * chunks = ws.chunks + (int64_t)seq * ws.n_chunks;
    const int base = blockIdx.x * SMP_CHUNK + wave * SMP_SEG;
    float x[SMP_LANE];
    if (!s.greedy) smp_read((const T *)a.logits + seq * a.logits_stride, base, a.vocab, x);
    uint64_t best = 0;
    for (int c = tid; c < ws.n_chunks; c += SMP_WG) {
        const uint64_t key = smp_key(chunks[c].top, chunks[c].at);
        best = key > best ? key : best;
    }
    best = smp_max_wg(best, s_part);
    const float top = smp_value(best);
    SmpCut cut = {top, SMP_OUT, SMP_OUT, SMP_OUT, ~0ull, 0.0, top == SMP_NONE ? -1 : smp_index(best), 0};
    if (s.greedy || top == SMP_NONE) {
        if (blockIdx.x == 0 && tid == 0) ws.cuts[seq] = cut;
        return;
    }
    if (s.by_k || s.by_p) {
        // ---- a thread's bin over all chunks
        int count = 0;
        double mass = 0.0;
        const uint64_t * hist = ws.hist + (int64_t)seq * ws.n_chunks * SMP_BINS;
        for (int c = 0; c < ws.n_chunks; ++c) {
            const float its = chunks[c].top;
            if (its == SMP_NONE) continue;
            const int b = tid - smp_bin(its, top, s.per_bin);
            if (b < 0) continue;
            const uint64_t v = hist[(int64_t)c * SMP_BINS + b];
            count += (int)(v >> SMP_COUNT_AT);
            mass += (double)(v & ((1ull << SMP_COUNT_AT) - 1)) * SMP_LEAST * smp_weight(its, top, s.inv_t);
        }
        int n_all;
        double all;
        const int n_before = smp_scan(count, s_count, n_all);
        const double before = smp_scan(mass, s_sum, all), upto = before + mass;
        const int k = s.by_k ? min(s.k, n_all) : n_all;
        if (tid == 0) s_at[0] = s_at[1] = s_at[2] = SMP_BINS - 1;
        __syncthreads();
        const int n_upto = n_before + count;
        if (n_before < k && k <= n_upto) {                 // one bin: top_k ends here
            s_at[2] = tid;
            s_mass[0] = s.by_k ? before : all;
            s_mass[1] = s.by_k ? upto + n_upto * SMP_LEAST : all + n_all * SMP_LEAST;
        }
        __syncthreads();
        const int last = s_at[2];
        if (s.by_p) {
            // the first bin in which the sum may, and in which it must have reached top_p's part
            const uint64_t may = __ballot((upto + n_upto * SMP_LEAST) * (1.0 + SMP_MARGIN) >= s.p * s_mass[0] * (1.0 - SMP_MARGIN));
            const uint64_t must = __ballot(upto * (1.0 - SMP_MARGIN) >= s.p * s_mass[1] * (1.0 + SMP_MARGIN));
            if (lane == 0) {
                if (may) atomicMin(&s_at[0], tid + (int)__builtin_ctzll(may));
                if (must) atomicMin(&s_at[1], tid + (int)__builtin_ctzll(must));
            }
            __syncthreads();
            cut.lo = min(s_at[0], last);
            cut.hi = min(s_at[1], last);
        } else {
            cut.lo = cut.hi = last;
        }
        cut.last = s.by_k ? last : SMP_BINS;
    }
    if (blockIdx.x == 0 && tid == 0) ws.cuts[seq] = cut;
    // ---- the wave's segment
    SmpSeg g = {0.0, 0.0, 0.0, 0, 0, 0, 0};
    const int64_t seg = ((int64_t)seq * ws.n_chunks + blockIdx.x) * SMP_WAVES + wave;
    uint64_t * list = ws.keys + seg * SMP_SEG;
    const double top_bin = floor((double)top * s.per_bin);
    const bool bins = s.by_k || s.by_p;
#pragma unroll
    for (int j = 0; j < SMP_LANE; ++j) {
        const int b = !bins || x[j] == top ? 0 : (int)fmin(top_bin - floor((double)x[j] * s.per_bin), (double)SMP_OUT);
        const bool there = x[j] != SMP_NONE, cand = there && ((b >= cut.lo && b <= cut.hi) || b == cut.last);
        const bool sure = there && b < cut.lo, mid = there && b > cut.hi && b < cut.last;
        if (sure || mid) {
            const double w = smp_weight(x[j], top, s.inv_t);
            if (sure) {
                g.sure += w;
                g.draw += w >= s.min_p ? w : 0.0;
                ++g.n_sure;
            } else {
                g.mid += w;
                ++g.n_mid;
            }
        }
        const uint64_t votes = __ballot(cand);
        if (cand) list[g.n_cand + __popcll(votes & ((1ull << lane) - 1))] = smp_key(x[j], smp_at<T>(base, j));
        g.n_cand += __popcll(votes);
    }
    for (int o = 32; o; o >>= 1) {
        g.sure += __shfl_xor(g.sure, o, 64);
        g.draw += __shfl_xor(g.draw, o, 64);
        g.mid += __shfl_xor(g.mid, o, 64);
        g.n_sure += __shfl_xor(g.n_sure, o, 64);
        g.n_mid += __shfl_xor(g.n_mid, o, 64);
    }
    if (lane == 0) ws.segs[seg] = g;
}

template <class T>
__global__ __launch_bounds__(SMP_WG) void k_sample_pick(const llapis_sample_args a, const SmpWs ws) {
    __shared__ uint64_t s_key[SMP_SORT];
    __shared__ double s_sum[SMP_WAVES];
    __shared__ int s_count[SMP_WAVES];
    __shared__ unsigned long long s_mass[256];
    __shared__ int s_n[256];
    __shared__ int s_seg, s_last;
    __shared__ double s_before;
    const int seq = blockIdx.x, tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const SmpSet s = smp_settings(a, seq);
    const SmpCut cut = ws.cuts[seq];
    if (s.greedy || cut.token < 0) {
        if (tid == 0) a.tokens[seq] = cut.token;
        return;
    }
    const int n_segs = (a.vocab + SMP_SEG - 1) / SMP_SEG, per = (n_segs + SMP_WG - 1) / SMP_WG;
    const int64_t seg0 = (int64_t)seq * ws.n_chunks * SMP_WAVES;
    const SmpSeg * segs = ws.segs + seg0;
    const uint64_t * keys = ws.keys + seg0 * SMP_SEG;
    auto weight = [&](uint64_t key) { return smp_weight(smp_value(key), cut.top, s.inv_t); };
    // ---- a thread's segments are consecutive
    SmpSeg mine = {0.0, 0.0, 0.0, 0, 0, 0, 0};
    for (int i = tid * per; i < min((tid + 1) * per, n_segs); ++i) {
        const SmpSeg g = segs[i];
        mine.sure += g.sure;
        mine.mid += g.mid;
        mine.n_sure += g.n_sure;
        mine.n_mid += g.n_mid;
        mine.n_cand += g.n_cand;
    }
    double sure, mid;
    int n_sure, n_mid, n_cand;
    smp_scan(mine.sure, s_sum, sure);
    smp_scan(mine.mid, s_sum, mid);
    smp_scan(mine.n_sure, s_count, n_sure);
    smp_scan(mine.n_mid, s_count, n_mid);
    const int at = smp_scan(mine.n_cand, s_count, n_cand);
    // f(key) of each candidate, a wave a segment
    auto each = [&](auto f) {
        for (int i = wave; i < n_segs; i += SMP_WAVES) {
            const int n = segs[i].n_cand;
            for (int c = lane; c < n; c += 64) f(keys[(int64_t)i * SMP_SEG + c]);
        }
    };
    uint64_t key = ~0ull;                                  // the last that is kept
    if (n_cand > 0) {
        // candidates within top_k, the first of them in order
        const int n_k = s.by_k ? max(min(s.k - n_sure - n_mid, n_cand), 0) : n_cand;
        if (n_cand <= SMP_SORT) {
            int n2 = 64;
            while (n2 < n_cand) n2 *= 2;
            // each segment's list to its place
            int to = at;
            for (int i = tid * per; i < min((tid + 1) * per, n_segs); ++i) {
                const int n = segs[i].n_cand;
                for (int c = 0; c < n; ++c) s_key[to++] = keys[(int64_t)i * SMP_SEG + c];
            }
            for (int i = n_cand + tid; i < n2; i += SMP_WG) s_key[i] = 0;
            __syncthreads();
            for (int size = 2; size <= n2; size *= 2)
                for (int step = size / 2; step; step /= 2) {
                    for (int i = tid; i < n2 / 2; i += SMP_WG) {
                        const int l = (i / step) * 2 * step + i % step, r = l + step;
                        const uint64_t u = s_key[l], v = s_key[r];
                        if ((u < v) == ((l & size) == 0)) {
                            s_key[l] = v;
                            s_key[r] = u;
                        }
                    }
                    __syncthreads();
                }
            // a thread's keys are consecutive
            const int each_n = (n2 + SMP_WG - 1) / SMP_WG;
            double w[SMP_SORT / SMP_WG], sum = 0.0, within = 0.0;
#pragma unroll
            for (int i = 0; i < SMP_SORT / SMP_WG; ++i) {
                const int r = tid * each_n + i;
                w[i] = i < each_n && r < n_cand ? weight(s_key[r]) : 0.0;
                sum += w[i];
                within += r < n_k ? w[i] : 0.0;
            }
            double all_k, all;
            smp_scan(within, s_sum, all_k);
            double before = sure + smp_scan(sum, s_sum, all);
            const double goal = s.p * (sure + mid + all_k);
            int kept = 0;
#pragma unroll
            for (int i = 0; i < SMP_SORT / SMP_WG; ++i) {
                const int r = tid * each_n + i;
                if (i < each_n && r < n_k && (!s.by_p || before < goal)) ++kept;
                before += w[i];
            }
            int n_kept;
            smp_scan(kept, s_count, n_kept);
            if (n_kept > 0) key = s_key[n_kept - 1];
        } else {
            // too many: eight bits of the key at a time, the candidates counted (and
            // weighed in fixed point) by them: the first key at which the number or the
            // weight of what is not below it reaches the goal
            int bits = 1;
            while (bits < 31 && (1 << bits) < n_cand) ++bits;
            const double scale = __builtin_ldexp(1.0, 61 - bits);
            auto descend = [&](bool by_mass, int n_goal, double goal) {
                uint64_t prefix = 0;
                int n_above = 0;
                unsigned long long above = 0;
                const unsigned long long want = by_mass ? (unsigned long long)ceil(fmax(goal, 0.0) * scale) : 0;
                for (int shift = 56; shift >= 0; shift -= 8) {
                    if (tid < 256) {
                        s_n[tid] = 0;
                        s_mass[tid] = 0;
                    }
                    __syncthreads();
                    each([&](uint64_t u) {
                        if (shift < 56 && (u >> (shift + 8)) != (prefix >> (shift + 8))) return;
                        const int d = (int)(u >> shift) & 255;
                        atomicAdd(&s_n[d], 1);
                        if (by_mass) atomicAdd(&s_mass[d], (unsigned long long)(weight(u) * scale));
                    });
                    __syncthreads();
                    int d = 255, found = -1;
                    for (; d >= 0; --d) {
                        if (s_n[d] == 0) continue;
                        found = d;
                        if (by_mass ? above + s_mass[d] >= want : n_above + s_n[d] >= n_goal) break;
                        n_above += s_n[d];
                        above += s_mass[d];
                    }
                    if (d < 0) {                          // all of them: the last
                        n_above -= s_n[found];
                        above -= s_mass[found];
                    }
                    prefix |= (uint64_t)found << shift;
                    __syncthreads();
                }
                return prefix;
            };
            if (n_k > 0) {
                key = n_k < n_cand ? descend(false, n_k, 0.0) : 0;
                if (s.by_p) {
                    double within = 0.0, all_k;
                    each([&](uint64_t u) { within += u >= key ? weight(u) : 0.0; });
                    smp_scan(within, s_sum, all_k);
                    const uint64_t by_p = descend(true, 0, s.p * (sure + mid + all_k) - sure);
                    key = by_p > key ? by_p : key;
                }
            }
        }
    }
    // ---- the segments' kept weights, in their order
    auto kept = [&](uint64_t u) {
        const double w = u >= key ? weight(u) : 0.0;
        return w >= s.min_p ? w : 0.0;
    };
    for (int i = wave; i < n_segs; i += SMP_WAVES) {
        const int n = segs[i].n_cand;
        double w = 0.0;
        for (int c = lane; c < n; c += 64) w += kept(keys[(int64_t)i * SMP_SEG + c]);
        if (n > 0) {
            for (int o = 32; o; o >>= 1) w += __shfl_xor(w, o, 64);
            if (lane == 0) ws.segs[seg0 + i].draw = segs[i].draw + w;
        }
    }
    if (tid == 0) {
        s_seg = 0x7FFFFFFF;
        s_last = -1;
    }
    __syncthreads();
    double sum = 0.0, total;
    for (int i = tid * per; i < min((tid + 1) * per, n_segs); ++i) sum += ws.segs[seg0 + i].draw;
    double cum = smp_scan(sum, s_sum, total);
    const double goal = (double)a.u[seq] * total;
    // the first thread in whose segments the sum passes the goal; without one
    // (rounding, u of 1 and more) the last that has anything
    const uint64_t any = __ballot(sum > 0.0), over = __ballot(sum > 0.0 && cum + sum > goal);
    if (lane == 0) {
        if (any) atomicMax(&s_last, tid + 63 - (int)__builtin_clzll(any));
        if (over) atomicMin(&s_seg, tid + (int)__builtin_ctzll(over));
    }
    __syncthreads();
    const bool found = s_seg != 0x7FFFFFFF;
    const int who = found ? s_seg : s_last;
    __syncthreads();
    if (tid == who) {
        int seg = -1;
        for (int i = tid * per; i < min((tid + 1) * per, n_segs); ++i) {
            const double y = ws.segs[seg0 + i].draw;
            if (!(y > 0.0)) continue;
            s_before = cum;
            seg = i;
            cum += y;
            if (found && cum > goal) break;
        }
        s_seg = seg;
        s_last = -1;
    }
    __syncthreads();
    // ---- the token: two consecutive values a thread
    const int first = s_seg * SMP_SEG + tid * (SMP_SEG / SMP_WG);
    const T * row = (const T *)a.logits + seq * a.logits_stride;
    double w[SMP_SEG / SMP_WG];
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < SMP_SEG / SMP_WG; ++i) {
        const float x = first + i < a.vocab ? smp_clean((float)row[first + i]) : SMP_NONE;
        const int b = !(s.by_k || s.by_p) ? 0 : smp_bin(x, cut.top, s.per_bin);
        const bool keep = x != SMP_NONE && (b < cut.lo || ((b <= cut.hi || b == cut.last) && smp_key(x, first + i) >= key));
        w[i] = keep ? smp_weight(x, cut.top, s.inv_t) : 0.0;
        if (w[i] < s.min_p) w[i] = 0.0;
        sum += w[i];
    }
    double part;
    cum = s_before + smp_scan(sum, s_sum, part);
    int token = -1, last = -1;
#pragma unroll
    for (int i = 0; i < SMP_SEG / SMP_WG; ++i) {
        cum += w[i];
        if (w[i] > 0.0) {
            last = first + i;
            if (token < 0 && found && cum > goal) token = first + i;
        }
    }
    // the lowest that passes, else the last that has a weight
    if (tid == 0) s_count[0] = 0x7FFFFFFF;
    __syncthreads();
    if (token >= 0) atomicMin(&s_count[0], token);
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    if (tid == 0) {
        a.tokens[seq] = s_count[0] != 0x7FFFFFFF ? s_count[0] : s_last;
        ws.cuts[seq].key = key;
        ws.cuts[seq].total = total;
    }
}

template <class T>
__global__ __launch_bounds__(SMP_WG) void k_sample_probs(const llapis_sample_args a, const SmpWs ws) {
    const int seq = blockIdx.y, wave = threadIdx.x >> 6;
    const SmpSet s = smp_settings(a, seq);
    const SmpCut cut = ws.cuts[seq];
    const int base = blockIdx.x * SMP_CHUNK + wave * SMP_SEG;
    if (base >= a.vocab) return;
    float x[SMP_LANE];
    smp_read((const T *)a.logits + seq * a.logits_stride, base, a.vocab, x);
    T * out = (T *)a.probs + seq * a.probs_stride;
    const double inv = 1.0 / cut.total;
    const bool bins = s.by_k || s.by_p;
#pragma unroll
    for (int j = 0; j < SMP_LANE; ++j) {
        const int i = smp_at<T>(base, j);
        float p = 0.0f;
        if (s.greedy) {
            p = i == cut.token ? 1.0f : 0.0f;
        } else if (x[j] != SMP_NONE && cut.token >= 0) {
            const int b = bins ? smp_bin(x[j], cut.top, s.per_bin) : 0;
            if (b < cut.lo || ((b <= cut.hi || b == cut.last) && smp_key(x[j], i) >= cut.key)) {
                const double w = smp_weight(x[j], cut.top, s.inv_t);
                p = w >= s.min_p ? (float)(w * inv) : 0.0f;
            }
        }
        if (i < a.vocab) out[i] = (T)p;
    }
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

// the workspace's parts; its size
uint64_t sample_parts(int n_seq, int vocab, uint8_t * at, SmpWs & ws) {
    ws.n_chunks = (vocab + SMP_CHUNK - 1) / SMP_CHUNK;
    const uint64_t chunks = (uint64_t)n_seq * ws.n_chunks;
    uint64_t n = 0;
    auto part = [&](uint64_t bytes) {
        uint8_t * p = at ? at + n : nullptr;
        n += round_up(bytes);
        return p;
    };
    ws.cuts = (SmpCut *)part((uint64_t)n_seq * sizeof(SmpCut));
    ws.chunks = (SmpChunk *)part(chunks * sizeof(SmpChunk));
    ws.segs = (SmpSeg *)part(chunks * SMP_WAVES * sizeof(SmpSeg));
    ws.hist = (uint64_t *)part(chunks * SMP_BINS * 8);
    ws.keys = (uint64_t *)part(chunks * SMP_CHUNK * 8);
    return n;
}

template <class T>
hipError_t launch_sample(const llapis_sample_args & a, const SmpWs & ws, hipStream_t s) {
    const dim3 grid(ws.n_chunks, a.n_seq), wg(SMP_WG);
    hipLaunchKernelGGL((k_sample_scan<T>), grid, wg, 0, s, a, ws);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_sample_cut<T>), grid, wg, 0, s, a, ws);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((k_sample_pick<T>), dim3(a.n_seq), wg, 0, s, a, ws);
    if ((e = hipGetLastError()) != hipSuccess || !a.probs) return e;
    hipLaunchKernelGGL((k_sample_probs<T>), grid, wg, 0, s, a, ws);
    return hipGetLastError();
}

}  // namespace
}  // namespace llapis

using namespace llapis;

extern "C" {

uint64_t llapis_sample_workspace_size(int32_t n_seq, int32_t vocab) {
    SmpWs ws;
    return n_seq <= 0 || n_seq > SMP_MAX_SEQ || vocab <= 0 || vocab > SMP_MAX_VOCAB ? 0 : sample_parts(n_seq, vocab, nullptr, ws);
}

int32_t llapis_sample(const llapis_sample_args * a, void * workspace, uint64_t ws_bytes, void * stream) {
    if (!a) return refuse_sample("null arguments");
    if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) return refuse_sample("need type F32, F16 or BF16");
    if (a->n_seq < 0 || a->n_seq > SMP_MAX_SEQ || a->vocab <= 0 || a->vocab > SMP_MAX_VOCAB)
        return refuse_sample("need 0 <= n_seq <= 65535, 0 < vocab <= 2^30");
    if (a->n_seq == 0) return 0;
    if (!a->logits || !a->u || !a->tokens) return refuse_sample("null logits, u or tokens");
    if (a->n_seq > 1 && (a->logits_stride < a->vocab || (a->probs && a->probs_stride < a->vocab)))
        return refuse_sample("rows shorter than vocab");
    if (!workspace || ((uintptr_t)workspace & 15) || ws_bytes < llapis_sample_workspace_size(a->n_seq, a->vocab))
        return refuse_sample("workspace too small or not 16-byte aligned");
    SmpWs ws;
    sample_parts(a->n_seq, a->vocab, (uint8_t *)workspace, ws);
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a->type == T_F32 ? launch_sample<float>(*a, ws, s) : a->type == T_F16 ? launch_sample<_Float16>(*a, ws, s)
                                                                                           : launch_sample<__bf16>(*a, ws, s);
    return e == hipSuccess ? 0 : refuse_sample(hipGetErrorString(e));
}

}  // extern "C"
