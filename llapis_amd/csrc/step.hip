// step.hip -- the norms between two blocks of a residual stream and the
// verification of drafted tokens (llapis_step.h).
#include <algorithm>
#include <cstdio>

#include "kv.h"

namespace llapis {
namespace dev {

// four values as they lie, aligned to one value: rows may start anywhere
typedef float f4 __attribute__((ext_vector_type(4)));
template <class T> struct Four { typedef T v __attribute__((ext_vector_type(4), aligned(sizeof(T)))); };

// values i .. i + 3 of a row of n, zeros past its end.  WHOLE: n is a multiple of
// 4 (and not 0); no branch then parts one load from the next
template <bool WHOLE, class T>
__device__ __forceinline__ typename Four<T>::v raw4(const T * p, int i, int n) {
    typename Four<T>::v r = {(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
    if constexpr (WHOLE) {
        const typename Four<T>::v w = *(const typename Four<T>::v *)(p + min(i, n - 4));
        r = i < n ? w : r;
    } else if (i + 4 <= n) {
        r = *(const typename Four<T>::v *)(p + i);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) r[j] = p[i + j];
    }
    return r;
}

template <class T>
__device__ __forceinline__ f4 wide4(typename Four<T>::v w) { return f4{(float)w[0], (float)w[1], (float)w[2], (float)w[3]}; }

template <bool WHOLE, class T>
__device__ __forceinline__ f4 get4(const T * p, int i, int n) { return wide4<T>(raw4<WHOLE>(p, i, n)); }

template <class T>
__device__ __forceinline__ void put4(T * p, int i, int n, f4 x) {
    if (i + 4 <= n) {
        typename Four<T>::v w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (T)x[j];
        *(typename Four<T>::v *)(p + i) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) p[i + j] = (T)x[j];
    }
}

// --------------------------------------------------------------- norms
//
// A workgroup takes tokens blockIdx, blockIdx + grid, ...; a thread holds 4 NCH
// values of a token, which are read and written once, and its share of the
// weights, which it reads once for all its tokens.  The next token's values are
// asked for before this one's sums.  The squares are summed per thread in order,
// then over the wave, then over the waves in order.
//
// Bound by memory: 11200 tokens of 2816 bf16 values, a gate and two outputs, 69 us
// (4.6 TB/s; a copy reaches 5.0), 88 with a workgroup a token, which reads the
// weights each time.  4 tokens of F32: 4.7 us, a launch and the chain of one load,
// two sums over the workgroup and a store.

__device__ __forceinline__ float block_sum(float x, float * s_part) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, 64);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    if (lane == 0) s_part[wave] = x;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += s_part[w];
    return s;
}

template <int NCH>
__device__ __forceinline__ float squares(const f4 (&x)[NCH]) {
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(x[c][j], x[c][j], ss);
    return ss;
}

// a token's values, as they lie until they are used
template <class T, int NCH>
struct NormRow {
    typename Four<T>::v h[NCH], y[NCH], g[NCH];
    float g1;
    template <bool WHOLE>
    __device__ __forceinline__ void read(const llapis_block_norm_args & a, int64_t t) {
        const int n = blockDim.x;
#pragma unroll
        for (int c = 0; c < NCH; ++c) h[c] = raw4<WHOLE>((const T *)a.h + t * a.h_stride, 4 * (threadIdx.x + c * n), a.d);
        if (!a.y) return;
#pragma unroll
        for (int c = 0; c < NCH; ++c) y[c] = raw4<WHOLE>((const T *)a.y + t * a.y_stride, 4 * (threadIdx.x + c * n), a.d);
        if (!a.gate) return;
        const T * gp = (const T *)a.gate + t * a.gate_token_stride;
        if (a.gate_value_stride) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) g[c] = raw4<WHOLE>(gp, 4 * (threadIdx.x + c * n), a.d);
        } else {
            g1 = (float)gp[0];
        }
    }
    __device__ __forceinline__ void load(const llapis_block_norm_args & a, int64_t t) {
        if (a.d % 4 == 0) read<true>(a, t);
        else read<false>(a, t);
    }
};

// NO: outputs that weights are held for, n_out at most
template <class T, int NCH, int NO, int THREADS>
__global__ __launch_bounds__(THREADS) void k_block_norm(const llapis_block_norm_args a) {
    __shared__ float s_part[2][2][16];
    const int d = a.d, n = blockDim.x;
    NormRow<T, NCH> row, next;
    row.load(a, blockIdx.x);
    // (4096 threads' worth of values and weights is more than the registers
    // hold: the weights are then read where they are used)
    constexpr bool HOLD = THREADS * NCH <= 2048;
    const float * wp = a.y && a.post_norm ? a.post_weight : nullptr;
    auto weight = [&](const float * w, int c) {
        const int i = 4 * (threadIdx.x + c * n);
        return !w ? f4{1.0f, 1.0f, 1.0f, 1.0f} : d % 4 == 0 ? get4<true>(w, i, d) : get4<false>(w, i, d);
    };
    f4 w_post[HOLD ? NCH : 1], w_pre[NO][HOLD ? NCH : 1];
    if constexpr (HOLD) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) w_post[c] = weight(wp, c);
#pragma unroll
        for (int o = 0; o < NO; ++o)
#pragma unroll
            for (int c = 0; c < NCH; ++c) w_pre[o][c] = weight(o < a.n_out ? a.weight[o] : nullptr, c);
    }
    int turn = 0;                                       // the sums' places are used in turn: one barrier a sum
    for (int64_t t = blockIdx.x; t < a.n_tokens; t += gridDim.x, turn ^= 1) {
        const bool more = t + gridDim.x < a.n_tokens;
        if (HOLD && more) next.load(a, t + gridDim.x);
        f4 h[NCH];
#pragma unroll
        for (int c = 0; c < NCH; ++c) h[c] = a.alpha * wide4<T>(row.h[c]);
        if (a.y) {
            f4 u[NCH];
#pragma unroll
            for (int c = 0; c < NCH; ++c) u[c] = wide4<T>(row.y[c]);
            if (a.post_norm) {
                const float inv = 1.0f / __fsqrt_rn(block_sum(squares<NCH>(u), s_part[turn][0]) / (float)d + a.eps);
#pragma unroll
                for (int c = 0; c < NCH; ++c) u[c] = u[c] * inv * (HOLD ? w_post[HOLD ? c : 0] : weight(wp, c));
            }
            if (a.gate)
#pragma unroll
                for (int c = 0; c < NCH; ++c) u[c] *= a.gate_value_stride ? wide4<T>(row.g[c]) : f4{row.g1, row.g1, row.g1, row.g1};
#pragma unroll
            for (int c = 0; c < NCH; ++c) h[c] += a.beta * u[c];
        }
        if (a.h_out)
#pragma unroll
            for (int c = 0; c < NCH; ++c) put4((T *)a.h_out + t * a.h_out_stride, 4 * (threadIdx.x + c * n), d, h[c]);
        if (a.n_out > 0) {
            const float inv = 1.0f / __fsqrt_rn(block_sum(squares<NCH>(h), s_part[turn][1]) / (float)d + a.eps);
#pragma unroll
            for (int o = 0; o < NO; ++o)
                if (o < a.n_out)
#pragma unroll
                    for (int c = 0; c < NCH; ++c)
                        put4((T *)a.x[o] + t * a.x_stride[o], 4 * (threadIdx.x + c * n), d, h[c] * inv * (HOLD ? w_pre[o][HOLD ? c : 0] : weight(a.weight[o], c)));
        }
        if (HOLD && more) row = next;
        if (!HOLD && more) row.load(a, t + gridDim.x);
    }
}

// -------------------------------------------------------- verification
//
// k_verify_sum: every workgroup finds the number of taken drafts anew (a few
// loads) and sums 4 segments of 1024 values of the row the next token comes from,
// r, and p for the case that r is 0 everywhere.  (16 loads of 16 bytes a lane in two
// batches, or in one at three waves a SIMD, took twice the time of one batch of 8.)
// k_verify_pick: one workgroup a sequence adds the segments in order, finds the one
// where the sum passes u_next of the whole, and in it the token.
//
// Only the rows that the verdict names are read, about 50 MB for 32 sequences of
// 262144 values: 11.5 and 4.5 us, 27 together with more batches of loads and with
// LDS atomics for the pick's votes.  What bounds them is the chain: a sequence's
// verdict (two dependent loads), its rows, its sums, the segment's values again.  One
// sequence of 32003: 7.4 us together; one kernel of one workgroup, which saves a
// launch, took 9.9, its rows coming through one CU.

constexpr int VER_SEG = 1024;                   // values of a segment: 16 a lane, four a thread of the pick
constexpr int VER_RUN = 4 * VER_SEG;            // values of a workgroup, a segment a wave

template <class T>
__device__ __forceinline__ double prob(const T * p, int64_t i) {
    const float x = (float)p[i];
    return x > 0.0f && x < __builtin_inff() ? (double)x : 0.0;
}

// taken, whether one was refused, and it; from the first kernel to the second
struct Verdict { int a, refused, draft, pad; };

template <class T>
__device__ __forceinline__ Verdict verdict(const llapis_verify_args & v, int seq) {
    const int lane = threadIdx.x & 63;
    const int n = v.n_draft ? min(max(v.n_draft[seq], 0), v.max_draft) : v.max_draft;
    bool ok = false;
    int x = -1;
    if (lane < v.max_draft) {
        const int64_t i = (int64_t)seq * v.max_draft + lane;
        x = v.drafts[i];
        const float u = v.u[i];
        if (lane < n && x >= 0 && x < v.vocab) {
            const double p = prob((const T *)v.target + ((int64_t)seq * (v.max_draft + 1) + lane) * v.target_stride, x);
            const double q = v.draft ? prob((const T *)v.draft + i * v.draft_stride, x) : 1.0;
            ok = (double)u * q < p;
        }
    }
    const uint64_t no = ~__ballot(ok);
    const int a = min(no ? (int)__builtin_ctzll(no) : 64, n);
    return {a, a < n, a < n ? __shfl(x, a, 64) : -1, 0};
}

// the row the next token comes from, and what is taken off it: the draft's row
// (less), without one 1 at the place `draft`
template <class T>
struct Row {
    const T * p;
    const T * q;
    bool less;
    int draft;
    __device__ __forceinline__ Row(const llapis_verify_args & v, int seq, const Verdict & w) {
        p = (const T *)v.target + ((int64_t)seq * (v.max_draft + 1) + w.a) * v.target_stride;
        q = (const T *)v.draft + ((int64_t)seq * v.max_draft + w.a) * v.draft_stride;
        less = w.refused && v.draft;
        draft = w.refused && !v.draft ? w.draft : -1;
    }
    // N times four values, from i + 0, i + step, ...
    template <int N>
    __device__ __forceinline__ void read(const T * row, int i, int step, int n, f4 (&x)[N]) const {
        if (n % 4 == 0) {
#pragma unroll
            for (int c = 0; c < N; ++c) x[c] = get4<true>(row, i + c * step, n);
        } else {
#pragma unroll
            for (int c = 0; c < N; ++c) x[c] = get4<false>(row, i + c * step, n);
        }
    }
    // f(c, j, r, p) of each value j of each four c
    template <int N, class F>
    __device__ __forceinline__ void values(int i, int step, int n, F f) const {
        f4 x[N], y[N];
        read<N>(p, i, step, n, x);
        if (less) {
            read<N>(q, i, step, n, y);
#pragma unroll
            for (int c = 0; c < N; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const double w = (double)some(x[c][j]);
                    f(c, j, fmax(w - (double)some(y[c][j]), 0.0), w);
                }
        } else {
#pragma unroll
            for (int c = 0; c < N; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const double w = (double)some(x[c][j]);
                    f(c, j, i + c * step + j == draft ? fmax(w - 1.0, 0.0) : w, w);
                }
        }
    }
    // what is not positive and finite counts as 0
    static __device__ __forceinline__ float some(float x) { return x > 0.0f && x < __builtin_inff() ? x : 0.0f; }
};

struct Sums { double r, p; };

// segments of a sequence, a whole number of workgroups
__host__ __device__ __forceinline__ int verify_segments(int vocab) { return (vocab + VER_RUN - 1) / VER_RUN * 4; }

template <class T>
__global__ __launch_bounds__(256, 4) void k_verify_sum(const llapis_verify_args v, Sums * sums, Verdict * verdicts) {
    const int seq = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Verdict w = verdict<T>(v, seq);
    const Row<T> row(v, seq, w);
    if (blockIdx.x == 0 && threadIdx.x == 0) verdicts[seq] = w;
    Sums s = {0.0, 0.0};
    row.template values<4>(blockIdx.x * VER_RUN + wave * VER_SEG + 4 * lane, 256, v.vocab, [&](int, int, double r, double p) {
        s.r += r;
        s.p += p;
    });
    for (int o = 32; o; o >>= 1) {
        s.r += __shfl_xor(s.r, o, 64);
        s.p += __shfl_xor(s.p, o, 64);
    }
    if (lane == 0) sums[((int64_t)seq * gridDim.x + blockIdx.x) * 4 + wave] = s;
}

// exclusive sums over the workgroup's 256 threads in order, and the whole
__device__ __forceinline__ Sums scan256(Sums x, Sums * s_part, Sums & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums v = x;
    for (int o = 1; o < 64; o <<= 1) {
        const double r = __shfl_up(v.r, o, 64), p = __shfl_up(v.p, o, 64);
        if (lane >= o) {
            v.r += r;
            v.p += p;
        }
    }
    if (lane == 63) s_part[wave] = v;
    __syncthreads();
    Sums before = {0.0, 0.0};
    total = {0.0, 0.0};
    for (int w = 0; w < 4; ++w) {
        const Sums y = s_part[w];
        if (w < wave) {
            before.r += y.r;
            before.p += y.p;
        }
        total.r += y.r;
        total.p += y.p;
    }
    const double r = __shfl_up(v.r, 1, 64), p = __shfl_up(v.p, 1, 64);
    return {before.r + (lane ? r : 0.0), before.p + (lane ? p : 0.0)};
}

template <class T>
__global__ __launch_bounds__(256) void k_verify_pick(const llapis_verify_args v, const Sums * sums, const Verdict * verdicts) {
    __shared__ Sums s_part[2][4];
    // of each wave: the first thread whose sum passes the goal, the last that has
    // anything; then the tokens
    __shared__ int s_first[2][4], s_last[2][4];
    __shared__ int s_seg;
    __shared__ double s_before;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n_seg = verify_segments(v.vocab), per = (n_seg + 255) / 256;
    const Verdict w = verdicts[seq];
    const float u = v.u_next[seq];
    const Sums * mine = sums + (int64_t)seq * n_seg;
    const int drafted = tid < w.a ? v.drafts[(int64_t)seq * v.max_draft + tid] : -1;
    if (tid == 0) s_seg = -1;
    auto vote = [&](int k, bool any, bool passes, int mark) {
        const uint64_t a = __ballot(any), p = __ballot(passes);
        const int first = __shfl(mark, p ? __builtin_ctzll(p) : 0, 64);
        const int last = __shfl(mark, a ? 63 - __builtin_clzll(a) : 0, 64);
        if (lane == 0) {
            s_first[k][wave] = p ? first : 0x7FFFFFFF;
            s_last[k][wave] = a ? last : -1;
        }
    };
    auto first_of = [&](int k) { return min(min(s_first[k][0], s_first[k][1]), min(s_first[k][2], s_first[k][3])); };
    auto last_of = [&](int k) { return max(max(s_last[k][0], s_last[k][1]), max(s_last[k][2], s_last[k][3])); };
    // a thread's segments are consecutive
    Sums x = {0.0, 0.0}, total;
    for (int i = tid * per; i < min((tid + 1) * per, n_seg); ++i) {
        x.r += mine[i].r;
        x.p += mine[i].p;
    }
    const Sums before = scan256(x, s_part[0], total);
    const bool rest = w.refused && total.r > 0.0;
    const double goal = (double)u * (rest ? total.r : total.p), part = rest ? x.r : x.p;
    const double at = rest ? before.r : before.p;
    // the thread in whose segments the sum passes the goal; without one
    // (rounding, u_next of 1 and more) the last that has anything
    vote(0, part > 0.0, part > 0.0 && at + part > goal, tid);
    __syncthreads();
    const int first = first_of(0);
    const bool found = first != 0x7FFFFFFF;
    if (tid == (found ? first : last_of(0))) {
        // ... and the segment
        double cum = at;
        int seg = -1;
        for (int i = tid * per; i < min((tid + 1) * per, n_seg); ++i) {
            const double y = rest ? mine[i].r : mine[i].p;
            if (!(y > 0.0)) continue;
            s_before = cum;
            seg = i;
            cum += y;
            if (found && cum > goal) break;
        }
        s_seg = seg;
    }
    __syncthreads();
    int next = -1;
    const int seg = s_seg;
    if (seg >= 0) {
        const Row<T> row(v, seq, w);
        double r[4];
        const int i0 = seg * VER_SEG + 4 * tid;
        Sums y = {0.0, 0.0};
        row.template values<1>(i0, 0, v.vocab, [&](int, int j, double a, double p) {
            r[j] = rest ? a : p;
            y.r += r[j];
        });
        double cum = s_before + scan256(y, s_part[1], total).r;
        int tok = -1, last = -1;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            cum += r[j];
            if (r[j] > 0.0) {
                last = i0 + j;
                if (tok < 0 && found && cum > goal) tok = i0 + j;
            }
        }
        // a thread that passes marks its token, the others their last
        vote(1, last >= 0, tok >= 0, tok >= 0 ? tok : last);
        __syncthreads();
        const int f = first_of(1);
        next = f != 0x7FFFFFFF ? f : last_of(1);
    }
    if (tid <= v.max_draft)
        v.tokens[(int64_t)seq * (v.max_draft + 1) + tid] = tid < w.a ? drafted : tid == w.a ? next : -1;
    if (tid == 0) v.accepted[seq] = w.a;
}

}  // namespace dev

using namespace dev;

namespace {

#define ST_TRY(expr)                                                       \
    do {                                                                   \
        const hipError_t e_ = (expr);                                      \
        if (e_ != hipSuccess) return refuse(hipGetErrorString(e_));        \
    } while (0)

int32_t refuse_as(const char * who, const char * why) noexcept {
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", who, why);
    return refuse(msg);
}

template <class T, int NO>
void launch_norm_chunks(const llapis_block_norm_args & a, int nch, int threads, int grid, hipStream_t s) {
    const dim3 g(grid), wg(threads);
    if (nch == 1) {
        if (threads <= 256) hipLaunchKernelGGL((k_block_norm<T, 1, NO, 256>), g, wg, 0, s, a);
        else hipLaunchKernelGGL((k_block_norm<T, 1, NO, 1024>), g, wg, 0, s, a);
    } else if (nch == 2) {
        if (threads <= 256) hipLaunchKernelGGL((k_block_norm<T, 2, NO, 256>), g, wg, 0, s, a);
        else hipLaunchKernelGGL((k_block_norm<T, 2, NO, 1024>), g, wg, 0, s, a);
    } else if (threads <= 256) {
        if (nch == 3) hipLaunchKernelGGL((k_block_norm<T, 3, NO, 256>), g, wg, 0, s, a);
        else hipLaunchKernelGGL((k_block_norm<T, 4, NO, 256>), g, wg, 0, s, a);
    } else {
        hipLaunchKernelGGL((k_block_norm<T, 4, NO, 1024>), g, wg, 0, s, a);
    }
}

template <class T>
hipError_t launch_norm(const llapis_block_norm_args & a, hipStream_t s) {
    // few tokens: as many threads as a token has use for; many: fewer, with more
    // values each, and as many workgroups as the card holds, each for as many tokens
    const int quads = (a.d + 3) / 4;
    int threads = a.n_tokens > 512 ? 256 : 1024;
    while (threads > 64 && threads / 2 >= quads) threads /= 2;
    while (threads < 1024 && (quads + threads - 1) / threads > 4) threads *= 2;
    const int nch = (quads + threads - 1) / threads;
    const int held = 256 * 1024 / threads;
    const int each = (a.n_tokens - 1) / held + 1, grid = (a.n_tokens - 1) / each + 1;
    if (a.n_out <= 1) launch_norm_chunks<T, 1>(a, nch, threads, grid, s);
    else if (a.n_out == 2) launch_norm_chunks<T, 2>(a, nch, threads, grid, s);
    else launch_norm_chunks<T, 4>(a, nch, threads, grid, s);
    return hipGetLastError();
}

constexpr int VER_MAX_SEQ = 65535, VER_MAX_VOCAB = 1 << 30;

// a sequence's sums, then its verdict
uint64_t verify_sums_bytes(int n_seq, int vocab) { return (uint64_t)n_seq * verify_segments(vocab) * sizeof(Sums); }

template <class T>
hipError_t launch_verify(const llapis_verify_args & v, void * ws, hipStream_t s) {
    Sums * sums = (Sums *)ws;
    Verdict * verdicts = (Verdict *)((uint8_t *)ws + verify_sums_bytes(v.n_seq, v.vocab));
    hipLaunchKernelGGL((k_verify_sum<T>), dim3(verify_segments(v.vocab) / 4, v.n_seq), dim3(256), 0, s, v, sums, verdicts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_verify_pick<T>), dim3(v.n_seq), dim3(256), 0, s, v, sums, verdicts);
    return hipGetLastError();
}

}  // namespace
}  // namespace llapis

using namespace llapis;

extern "C" {

int32_t llapis_block_norm(const llapis_block_norm_args * a, void * stream) {
    const char * who = "llapis_block_norm";
    if (!a) return refuse_as(who, "null arguments");
    if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) return refuse_as(who, "need type F32, F16 or BF16");
    if (a->n_tokens < 0 || a->d <= 0 || a->d > 16384) return refuse_as(who, "need n_tokens >= 0 and 0 < d <= 16384");
    if (a->n_out < 0 || a->n_out > LLAPIS_NORM_MAX_OUT) return refuse_as(who, "need 0 <= n_out <= 4");
    if (a->n_tokens == 0) return 0;
    if (!a->h) return refuse_as(who, "null h");
    if (!a->h_out && a->n_out == 0) return refuse_as(who, "nothing to write");
    if (a->gate && a->gate_value_stride != 0 && a->gate_value_stride != 1) return refuse_as(who, "need gate_value_stride 0 or 1");
    for (int i = 0; i < a->n_out; ++i)
        if (!a->x[i]) return refuse_as(who, "null output");
    if (a->n_tokens > 1) {
        bool shorter = a->h_out && a->h_out_stride < a->d;
        for (int i = 0; i < a->n_out; ++i) shorter |= a->x_stride[i] < a->d;
        if (shorter) return refuse_as(who, "output rows overlap");
    }
    hipStream_t s = (hipStream_t)stream;
    if (a->type == T_F32) ST_TRY(launch_norm<float>(*a, s));
    else if (a->type == T_F16) ST_TRY(launch_norm<_Float16>(*a, s));
    else ST_TRY(launch_norm<__bf16>(*a, s));
    return 0;
}

uint64_t llapis_verify_drafts_workspace_size(int32_t n_seq, int32_t vocab) {
    return n_seq <= 0 || n_seq > VER_MAX_SEQ || vocab <= 0 || vocab > VER_MAX_VOCAB ? 0 : verify_sums_bytes(n_seq, vocab) + (uint64_t)n_seq * sizeof(Verdict);
}

int32_t llapis_verify_drafts(const llapis_verify_args * a, void * workspace, uint64_t ws_bytes, void * stream) {
    const char * who = "llapis_verify_drafts";
    if (!a) return refuse_as(who, "null arguments");
    if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) return refuse_as(who, "need type F32, F16 or BF16");
    if (a->n_seq < 0 || a->n_seq > VER_MAX_SEQ || a->max_draft < 0 || a->max_draft > 63 || a->vocab <= 0 || a->vocab > VER_MAX_VOCAB)
        return refuse_as(who, "need 0 <= n_seq <= 65535, 0 <= max_draft <= 63, 0 < vocab <= 2^30");
    if (a->n_seq == 0) return 0;
    if (!a->target || !a->u_next || !a->tokens || !a->accepted || (a->max_draft > 0 && (!a->drafts || !a->u)))
        return refuse_as(who, "null pointer");
    if (a->target_stride < a->vocab || (a->draft && a->draft_stride < a->vocab)) return refuse_as(who, "rows shorter than vocab");
    if (!workspace || ((uintptr_t)workspace & 7) || ws_bytes < llapis_verify_drafts_workspace_size(a->n_seq, a->vocab))
        return refuse_as(who, "workspace too small or not 8-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    if (a->type == T_F32) ST_TRY(launch_verify<float>(*a, workspace, s));
    else if (a->type == T_F16) ST_TRY(launch_verify<_Float16>(*a, workspace, s));
    else ST_TRY(launch_verify<__bf16>(*a, workspace, s));
    return 0;
}

}  // extern "C"
