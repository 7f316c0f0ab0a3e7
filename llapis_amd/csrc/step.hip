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

template <class T>
__device__ __forceinline__ f4 get4(const T * p, int i, int n) {
    f4 r = {0.0f, 0.0f, 0.0f, 0.0f};
    if (i + 4 <= n) {
        const typename Four<T>::v w = *(const typename Four<T>::v *)(p + i);
        r = f4{(float)w[0], (float)w[1], (float)w[2], (float)w[3]};
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) r[j] = (float)p[i + j];
    }
    return r;
}

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
// One workgroup a token.  Every load is issued before the first sum; a thread
// holds 4 NCH values, which are read and written once.  The squares are summed
// per thread in order, then over the wave, then over the waves in order.

__device__ __forceinline__ float block_sum(float x, float * s_part) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, 64);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    if (lane == 0) s_part[wave] = x;
    __syncthreads();
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) s += s_part[w];
    return s;
}

template <class T, int NCH>
__global__ __launch_bounds__(1024) void k_block_norm(const llapis_block_norm_args a) {
    __shared__ float s_part[2][16];
    const int d = a.d, n = blockDim.x;
    const int64_t t = blockIdx.x;
    const T * hp = (const T *)a.h + t * a.h_stride;
    f4 h[NCH], u[NCH];
#pragma unroll
    for (int c = 0; c < NCH; ++c) h[c] = get4(hp, 4 * (threadIdx.x + c * n), d);
    if (a.y) {
        const T * yp = (const T *)a.y + t * a.y_stride;
#pragma unroll
        for (int c = 0; c < NCH; ++c) u[c] = get4(yp, 4 * (threadIdx.x + c * n), d);
        if (a.post_norm) {
            float ss = 0.0f;
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(u[c][j], u[c][j], ss);
            const float inv = 1.0f / __fsqrt_rn(block_sum(ss, s_part[0]) / (float)d + a.eps);
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                u[c] *= inv;
                if (a.post_weight) u[c] *= get4(a.post_weight, 4 * (threadIdx.x + c * n), d);
            }
        }
        if (a.gate) {
            const T * gp = (const T *)a.gate + t * a.gate_token_stride;
            const float g = a.gate_value_stride ? 0.0f : (float)gp[0];
#pragma unroll
            for (int c = 0; c < NCH; ++c)
                u[c] *= a.gate_value_stride ? get4(gp, 4 * (threadIdx.x + c * n), d) : f4{g, g, g, g};
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c) h[c] = a.alpha * h[c] + a.beta * u[c];
    } else {
#pragma unroll
        for (int c = 0; c < NCH; ++c) h[c] = a.alpha * h[c];
    }
    if (a.h_out) {
        T * op = (T *)a.h_out + t * a.h_out_stride;
#pragma unroll
        for (int c = 0; c < NCH; ++c) put4(op, 4 * (threadIdx.x + c * n), d, h[c]);
    }
    if (a.n_out == 0) return;
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = __builtin_fmaf(h[c][j], h[c][j], ss);
    const float inv = 1.0f / __fsqrt_rn(block_sum(ss, s_part[1]) / (float)d + a.eps);
#pragma unroll
    for (int o = 0; o < LLAPIS_NORM_MAX_OUT; ++o)
        if (o < a.n_out) {
            T * xp = (T *)a.x[o] + t * a.x_stride[o];
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int i = 4 * (threadIdx.x + c * n);
                f4 x = h[c] * inv;
                if (a.weight[o]) x *= get4(a.weight[o], i, d);
                put4(xp, i, d, x);
            }
        }
}

// -------------------------------------------------------- verification
//
// k_verify_sum: every workgroup finds the number of taken drafts anew (a few
// loads) and sums a run of VER_RUN values of the row the next token comes from,
// r and, for drafts that all were refused to no rest, p.  k_verify_pick: one
// workgroup a sequence adds the runs in order, finds the run where the sum
// passes u_next of the whole, and in it the token.

constexpr int VER_PER = 32;                     // consecutive values of a thread
constexpr int VER_RUN = 256 * VER_PER;

template <class T>
__device__ __forceinline__ double prob(const T * p, int64_t i) {
    const float x = (float)p[i];
    return x > 0.0f && x < __builtin_inff() ? (double)x : 0.0;
}

struct Verdict { int a, n, draft; };            // taken, drafted, the refused draft (or -1)

template <class T>
__device__ __forceinline__ Verdict verdict(const llapis_verify_args & v, int seq) {
    const int lane = threadIdx.x & 63;
    const int n = v.n_draft ? min(max(v.n_draft[seq], 0), v.max_draft) : v.max_draft;
    bool ok = false;
    if (lane < n) {
        const int64_t i = (int64_t)seq * v.max_draft + lane;
        const int x = v.drafts[i];
        if (x >= 0 && x < v.vocab) {
            const double p = prob((const T *)v.target + ((int64_t)seq * (v.max_draft + 1) + lane) * v.target_stride, x);
            const double q = v.draft ? prob((const T *)v.draft + i * v.draft_stride, x) : 1.0;
            ok = (double)v.u[i] * q < p;
        }
    }
    const uint64_t no = ~__ballot(ok);
    const int a = min(no ? (int)__builtin_ctzll(no) : 64, n);
    return {a, n, a < n ? v.drafts[(int64_t)seq * v.max_draft + a] : -1};
}

// the row the next token comes from, and what is taken off it
template <class T>
struct Row {
    const T * p;
    const T * q;                                // or null
    int draft;                                  // without q: the place that 1 is taken off
    __device__ __forceinline__ Row(const llapis_verify_args & v, int seq, const Verdict & w) {
        p = (const T *)v.target + ((int64_t)seq * (v.max_draft + 1) + w.a) * v.target_stride;
        q = w.a < w.n && v.draft ? (const T *)v.draft + ((int64_t)seq * v.max_draft + w.a) * v.draft_stride : nullptr;
        draft = w.a < w.n && !v.draft ? w.draft : -1;
    }
    // VER_PER / 8 or fewer values from i on: r, and p
    __device__ __forceinline__ void four(int i, int n, double (&r)[4], double (&whole)[4]) const {
        const f4 x = get4(p, i, n);
        const f4 y = q ? get4(q, i, n) : f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            whole[j] = x[j] > 0.0f && x[j] < __builtin_inff() ? (double)x[j] : 0.0;
            double off = y[j] > 0.0f && y[j] < __builtin_inff() ? (double)y[j] : 0.0;
            if (i + j == draft) off = 1.0;
            r[j] = whole[j] > off ? whole[j] - off : 0.0;
        }
    }
};

__device__ __forceinline__ double wave_sum(double x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}

template <class T>
__global__ __launch_bounds__(256) void k_verify_sum(const llapis_verify_args v, double * sums) {
    __shared__ double s_part[4][2];
    const int seq = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Row<T> row(v, seq, verdict<T>(v, seq));
    const int at = blockIdx.x * VER_RUN;
    double s = 0.0, w = 0.0;
#pragma unroll
    for (int c = 0; c < VER_PER / 4; ++c) {
        double r[4], p[4];
        row.four(at + 4 * (threadIdx.x + 256 * c), v.vocab, r, p);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s += r[j];
            w += p[j];
        }
    }
    s = wave_sum(s);
    w = wave_sum(w);
    if (lane == 0) {
        s_part[wave][0] = s;
        s_part[wave][1] = w;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        const int k = threadIdx.x;
        sums[((int64_t)seq * gridDim.x + blockIdx.x) * 2 + k] =
            (s_part[0][k] + s_part[1][k]) + (s_part[2][k] + s_part[3][k]);
    }
}

// exclusive sum over the workgroup's 256 threads in order, and the whole
__device__ __forceinline__ double scan256(double x, double * s_part, double & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double v = x;
    for (int o = 1; o < 64; o <<= 1) {
        const double u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) s_part[wave] = v;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
    for (int w = 0; w < 4; ++w) {
        if (w < wave) before += s_part[w];
        total += s_part[w];
    }
    const double prev = __shfl_up(v, 1, 64);
    return before + (lane ? prev : 0.0);
}

template <class T>
__global__ __launch_bounds__(256) void k_verify_pick(const llapis_verify_args v, const double * sums, int n_runs) {
    __shared__ double s_part[4];
    __shared__ int s_run, s_tok, s_last;
    __shared__ double s_before;
    const int seq = blockIdx.x, tid = threadIdx.x;
    const Verdict w = verdict<T>(v, seq);
    const Row<T> row(v, seq, w);
    const double * mine = sums + (int64_t)seq * n_runs * 2;
    // the sum of r, or of p where r is 0
    double part[2] = {0.0, 0.0};
    for (int i = tid; i < n_runs; i += 256) {
        part[0] += mine[2 * i];
        part[1] += mine[2 * i + 1];
    }
    double rest, whole;
    (void)scan256(part[0], s_part, rest);
    (void)scan256(part[1], s_part, whole);
    const int k = rest > 0.0 && w.a < w.n ? 0 : 1;
    const double goal = (double)v.u_next[seq] * (k ? whole : rest);
    if (tid == 0) {
        s_run = -1;
        s_tok = s_last = -1;
        s_before = 0.0;
    }
    __syncthreads();
    // the run in which the sum passes the goal; without one (rounding, u_next
    // of 1 and more) the last run that has anything
    double before = 0.0;
    for (int i0 = 0; i0 < n_runs; i0 += 256) {
        const double x = i0 + tid < n_runs ? mine[2 * (i0 + tid) + k] : 0.0;
        double all;
        const double at = before + scan256(x, s_part, all);
        const bool passes = x > 0.0 && at + x > goal;
        const int here = passes ? i0 + tid : 0x7FFFFFFF;
        // first passing run of the workgroup, last one with a positive sum
        if (x > 0.0) atomicMax(&s_last, i0 + tid);
        __syncthreads();
        if (passes) atomicMin((unsigned int *)&s_run, (unsigned int)here);      // -1 is the largest unsigned
        __syncthreads();
        if (s_run == i0 + tid || (s_run < 0 && s_last == i0 + tid)) s_before = at;
        before += all;
        __syncthreads();
        if (s_run >= 0) break;
    }
    const bool found = s_run >= 0;
    const int run = found ? s_run : s_last;
    __syncthreads();
    if (run >= 0) {
        if (tid == 0) s_last = -1;
        const int at = run * VER_RUN + tid * VER_PER;
        double x[VER_PER], sum = 0.0;
#pragma unroll
        for (int c = 0; c < VER_PER / 4; ++c) {
            double r[4], p[4];
            row.four(at + 4 * c, v.vocab, r, p);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[4 * c + j] = k ? p[j] : r[j];
                sum += x[4 * c + j];
            }
        }
        double all;
        double cum = s_before + scan256(sum, s_part, all);
        int tok = 0x7FFFFFFF, last = -1;
#pragma unroll
        for (int j = 0; j < VER_PER; ++j) {
            cum += x[j];
            if (x[j] > 0.0) {
                last = at + j;
                if (found && cum > goal && tok == 0x7FFFFFFF) tok = at + j;
            }
        }
        if (last >= 0) atomicMax(&s_last, last);
        if (tok != 0x7FFFFFFF) atomicMin((unsigned int *)&s_tok, (unsigned int)tok);
    }
    __syncthreads();
    const int next = s_tok >= 0 ? s_tok : run >= 0 ? s_last : -1;
    for (int i = tid; i <= v.max_draft; i += 256)
        v.tokens[(int64_t)seq * (v.max_draft + 1) + i] =
            i < w.a ? v.drafts[(int64_t)seq * v.max_draft + i] : i == w.a ? next : -1;
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

template <class T>
hipError_t launch_norm(const llapis_block_norm_args & a, hipStream_t s) {
    // few tokens: as many threads as a token has use for; many: fewer, with
    // more values each
    const int quads = (a.d + 3) / 4;
    int threads = a.n_tokens <= 512 ? 1024 : 256;
    while (threads > 64 && threads / 2 >= quads) threads /= 2;
    while (threads < 1024 && (quads + threads - 1) / threads > 4) threads *= 2;
    const int nch = (quads + threads - 1) / threads;
    const dim3 grid(a.n_tokens), wg(threads);
    if (nch <= 1) hipLaunchKernelGGL((k_block_norm<T, 1>), grid, wg, 0, s, a);
    else if (nch <= 2) hipLaunchKernelGGL((k_block_norm<T, 2>), grid, wg, 0, s, a);
    else if (nch <= 3) hipLaunchKernelGGL((k_block_norm<T, 3>), grid, wg, 0, s, a);
    else hipLaunchKernelGGL((k_block_norm<T, 4>), grid, wg, 0, s, a);
    return hipGetLastError();
}

int verify_runs(int vocab) { return (vocab + VER_RUN - 1) / VER_RUN; }

template <class T>
hipError_t launch_verify(const llapis_verify_args & v, double * sums, hipStream_t s) {
    const int runs = verify_runs(v.vocab);
    hipLaunchKernelGGL((k_verify_sum<T>), dim3(runs, v.n_seq), dim3(256), 0, s, v, sums);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((k_verify_pick<T>), dim3(v.n_seq), dim3(256), 0, s, v, sums, runs);
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
        bool shorter = (a->y && a->y_stride < 0) || a->h_stride < 0 || (a->h_out && a->h_out_stride < a->d);
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
    return n_seq <= 0 || vocab <= 0 ? 0 : (uint64_t)n_seq * verify_runs(vocab) * 16;
}

int32_t llapis_verify_drafts(const llapis_verify_args * a, void * workspace, uint64_t ws_bytes, void * stream) {
    const char * who = "llapis_verify_drafts";
    if (!a) return refuse_as(who, "null arguments");
    if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) return refuse_as(who, "need type F32, F16 or BF16");
    if (a->n_seq < 0 || a->n_seq > 65535 || a->max_draft < 0 || a->max_draft > 63 || a->vocab <= 0 || a->vocab > 1 << 30)
        return refuse_as(who, "need 0 <= n_seq <= 65535, 0 <= max_draft <= 63, 0 < vocab <= 2^30");
    if (a->n_seq == 0) return 0;
    if (!a->target || !a->u_next || !a->tokens || !a->accepted || (a->max_draft > 0 && (!a->drafts || !a->u)))
        return refuse_as(who, "null pointer");
    if (a->target_stride < a->vocab || (a->draft && a->draft_stride < a->vocab)) return refuse_as(who, "rows shorter than vocab");
    if (!workspace || ((uintptr_t)workspace & 7) || ws_bytes < llapis_verify_drafts_workspace_size(a->n_seq, a->vocab))
        return refuse_as(who, "workspace too small or not 8-byte aligned");
    double * sums = (double *)workspace;
    hipStream_t s = (hipStream_t)stream;
    if (a->type == T_F32) ST_TRY(launch_verify<float>(*a, sums, s));
    else if (a->type == T_F16) ST_TRY(launch_verify<_Float16>(*a, sums, s));
    else ST_TRY(launch_verify<__bf16>(*a, sums, s));
    return 0;
}

}  // extern "C"
