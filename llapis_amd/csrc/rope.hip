// rope.hip -- the norms of queries and keys for each head with their rotary
// positions, and the frequencies of a rotation (llapis_step.h).
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "kv.h"

namespace llapis {
namespace dev {

// A workgroup takes `each` consecutive tokens and a part of their heads.  Its
// threads first form the tokens' cosines and sines in LDS: the angle in turns in 64
// bits, reduced to an eighth of a turn either way, so that the fp32 function sees a
// small argument whose rounding is 2^-27 of a turn at most, whatever the position.
// Then 64 / L heads a wave: a lane holds slots of 2 V values of a head, the two
// vectors whose values turn together (half: V values of each half; pairs: 2 V
// consecutive ones), reads them once, adds the squares over the head's L lanes and
// writes them.
//
// Bound by memory for prompts (8192 tokens of 40 heads of 128 bf16: 168 MB in 40 us, 4.2 TB/s
// where a large copy reaches 5.1), by the launch and one load's chain for a step (4 tokens of 24 heads of
// 256: 3.7 us).
constexpr int ROPE_WG = 256, ROPE_TABLE = 1024;      // pairs of a workgroup's tokens in LDS

struct Rope {
    llapis_qk_rope_args a;
    int slots, lanes_log2;             // of a head
    int each;                          // tokens of a workgroup
};

template <class T, int V> struct RopeVec { typedef T v __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };
template <class T> struct RopeVec<T, 1> { typedef T v; };

template <class T, int V>
__device__ __forceinline__ void rope_get(const T * p, float (&x)[V]) {
    const typename RopeVec<T, V>::v w = *(const typename RopeVec<T, V>::v *)p;
    if constexpr (V == 1) x[0] = (float)w;
    else
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (float)w[i];
}

template <class T, int V>
__device__ __forceinline__ void rope_put(T * p, const float (&x)[V]) {
    typename RopeVec<T, V>::v w;
    if constexpr (V == 1) w = (T)x[0];
    else
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = (T)x[i];
    *(typename RopeVec<T, V>::v *)p = w;
}

// E: slots of a lane
template <class T, int V, int E>
__global__ __launch_bounds__(ROPE_WG) void k_qk_rope(const Rope p) {
    __shared__ float2 s_turn[ROPE_TABLE];
    const llapis_qk_rope_args & a = p.a;
    const int tid = threadIdx.x, half = a.rot_dim / 2, D = a.head_dim;
    const int t0 = blockIdx.x * p.each, n = min(p.each, a.n_tokens - t0);
    for (int i = tid; i < n * half; i += ROPE_WG) {
        const int t = i / half;
        // turns, their quarter and what is left of it
        const double turns = (double)a.pos[t0 + t] * a.freq[i - t * half] * 0.15915494309189533577;
        const double quarters = 4.0 * (turns - rint(turns)), q = rint(quarters);
        float sn, cs;
        sincospif((float)(0.5 * (quarters - q)), &sn, &cs);
        const int k = (int)q & 3;
        const float c = k & 1 ? sn : cs, s = k & 1 ? cs : sn;
        s_turn[i] = make_float2((k == 1 || k == 2 ? -c : c) * a.magnitude, (k >= 2 ? -s : s) * a.magnitude);
    }
    __syncthreads();
    const int L = 1 << p.lanes_log2, l = tid & (L - 1), heads = a.n_head + a.n_kv;
    // (token, head) in turn over the heads' places of the workgroups of these tokens
    const int places = (ROPE_WG >> p.lanes_log2) * gridDim.y;
    for (int i = blockIdx.y * (ROPE_WG >> p.lanes_log2) + (tid >> p.lanes_log2); i < n * heads; i += places) {
        const int t = i / heads, h = i - t * heads;
        if (a.pos && a.pos[t0 + t] < 0) continue;
        const bool is_k = h >= a.n_head;
        const int64_t row = t0 + t;
        const T * x = is_k ? (const T *)a.k + row * a.k_stride + (int64_t)(h - a.n_head) * D : (const T *)a.q + row * a.q_stride + (int64_t)h * D;
        T * y = is_k ? (T *)a.k_out + row * a.k_out_stride + (int64_t)(h - a.n_head) * D : (T *)a.q_out + row * a.q_out_stride + (int64_t)h * D;
        const float * w = is_k ? a.k_weight : a.q_weight;
        float u[E][V], v[E][V];
        int iu[E], iv[E];              // the two vectors' places
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int s = l + e * L, turned = half / V;
            const bool turns = s < turned;
            iu[e] = turns && a.layout == LLAPIS_ROPE_HALF ? s * V : 2 * s * V;
            iv[e] = turns && a.layout == LLAPIS_ROPE_HALF ? half + s * V : iu[e] + V;
#pragma unroll
            for (int j = 0; j < V; ++j) u[e][j] = v[e][j] = 0.0f;
            if (s < p.slots) {
                rope_get<T, V>(x + iu[e], u[e]);
                if (V > 1 || iv[e] < D) rope_get<T, V>(x + iv[e], v[e]);     // an odd head size ends in half a slot
            }
        }
        if (a.norm) {
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int j = 0; j < V; ++j) ss = __builtin_fmaf(u[e][j], u[e][j], __builtin_fmaf(v[e][j], v[e][j], ss));
            for (int o = 1; o < L; o <<= 1) ss += __shfl_xor(ss, o, 64);
            const float inv = 1.0f / __fsqrt_rn(ss / (float)D + a.eps);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (l + e * L < p.slots) {
                    float wu[V], wv[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) wu[j] = wv[j] = 1.0f;
                    if (w) {
                        rope_get<float, V>(w + iu[e], wu);
                        if (V > 1 || iv[e] < D) rope_get<float, V>(w + iv[e], wv);
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        u[e][j] *= inv * wu[j];
                        v[e][j] *= inv * wv[j];
                    }
                }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int s = l + e * L;
            if (s >= p.slots) continue;
            if (s < half / V) {
                const float2 * turn = s_turn + t * half + s * V;
                if (a.layout == LLAPIS_ROPE_HALF || V == 1) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float2 z = turn[j];
                        const float b = u[e][j], c = v[e][j];
                        u[e][j] = b * z.x - c * z.y;
                        v[e][j] = c * z.x + b * z.y;
                    }
                } else {
                    // V values of either vector are V / 2 pairs
#pragma unroll
                    for (int j = 0; j + 1 < V; j += 2) {
                        const float2 z = turn[j / 2], z1 = turn[V / 2 + j / 2];
                        const float b = u[e][j], c = u[e][j + 1], b1 = v[e][j], c1 = v[e][j + 1];
                        u[e][j] = b * z.x - c * z.y;
                        u[e][j + 1] = c * z.x + b * z.y;
                        v[e][j] = b1 * z1.x - c1 * z1.y;
                        v[e][j + 1] = c1 * z1.x + b1 * z1.y;
                    }
                }
            }
            rope_put<T, V>(y + iu[e], u[e]);
            if (V > 1 || iv[e] < D) rope_put<T, V>(y + iv[e], v[e]);
        }
    }
}

}  // namespace dev

using namespace dev;

namespace {

int32_t refuse_rope(const char * who, const char * why) noexcept {
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", who, why);
    return refuse(msg);
}

template <class T, int V, int E>
hipError_t launch_rope_as(const llapis_qk_rope_args & a, hipStream_t s) {
    Rope p{a, 0, 0, 1};
    p.slots = (a.head_dim + 2 * V - 1) / (2 * V);
    while (p.lanes_log2 < 6 && (E << p.lanes_log2) < p.slots) ++p.lanes_log2;
    // Four tokens to a workgroup where their heads leave it places (8192 tokens of 5 heads of 64 f16: 5.9 us, one token each
    // 9.7), and for 16-bit values where that still fills the card with workgroups of 256, eight to a CU; else one token's heads,
    // over several.  One and four, in us, on data that no cache holds: 40 heads of 128 bf16, 2048 tokens 13.9 and 17.8, 4096 22.8
    // and 23.0, 8192 41.1 and 37.6; 72 heads 4096 tokens 36.1 and 38.7, 8192 67.6 and 66.5; fp32, 24 heads of 256, 4096 tokens
    // 41.8 and 50.9, 8192 79.4 and 86.0
    const int places = ROPE_WG >> p.lanes_log2, heads = a.n_head + a.n_kv, most = a.rot_dim ? ROPE_TABLE / (a.rot_dim / 2) : 4;
    const bool four = 4 * heads <= places || (sizeof(T) == 2 && a.n_tokens >= 4 * 8 * 256);
    if (four) p.each = std::min(4, most);
    const int parts = four ? 1 : std::min((heads + places - 1) / places, 65535);
    hipLaunchKernelGGL((k_qk_rope<T, V, E>), dim3((a.n_tokens - 1) / p.each + 1, parts), dim3(ROPE_WG), 0, s, p);
    return hipGetLastError();
}

// the widest vectors that neither a head nor its turning part cuts
template <class T>
hipError_t launch_rope(const llapis_qk_rope_args & a, hipStream_t s) {
    constexpr int W = 16 / sizeof(T);
    auto fits = [&](int v) { return a.head_dim % (2 * v) == 0 && a.rot_dim % (2 * v) == 0; };
    if (fits(W)) return launch_rope_as<T, W, 1>(a, s);
    if (W > 4 && fits(4)) return launch_rope_as<T, 4, 1>(a, s);
    return launch_rope_as<T, 1, 4>(a, s);
}

}  // namespace
}  // namespace llapis

using namespace llapis;

extern "C" {

int32_t llapis_rope_frequencies(const llapis_rope_rule * r, double * freq, float * magnitude) {
    const char * who = "llapis_rope_frequencies";
    if (!r || !freq || !magnitude) return refuse_rope(who, "null argument");
    if (r->rot_dim <= 0 || r->rot_dim % 2 || r->rot_dim > 512) return refuse_rope(who, "need an even rot_dim, 2 to 512");
    if (r->kind < LLAPIS_ROPE_PLAIN || r->kind > LLAPIS_ROPE_BANDS) return refuse_rope(who, "unknown kind");
    if (!(r->base > 1.0) || !std::isfinite(r->base)) return refuse_rope(who, "need a base above 1");
    const bool scaled = r->kind != LLAPIS_ROPE_PLAIN, banded = r->kind == LLAPIS_ROPE_YARN || r->kind == LLAPIS_ROPE_BANDS;
    if (scaled && (!(r->factor > 0.0) || !std::isfinite(r->factor))) return refuse_rope(who, "need a factor above 0");
    if (banded && (!(r->trained > 0.0) || !std::isfinite(r->trained) || !(r->low > 0.0) || !(r->high > r->low) || !std::isfinite(r->high)))
        return refuse_rope(who, "need trained > 0 and 0 < low < high");
    const int half = r->rot_dim / 2;
    const double two_pi = 6.283185307179586476925;
    if (r->divisors)
        for (int i = 0; i < half; ++i)
            if (!(r->divisors[i] > 0.0)) return refuse_rope(who, "need divisors above 0");
    double base = r->base;
    if (r->kind == LLAPIS_ROPE_NTK && r->rot_dim > 2) base *= std::pow(r->factor, (double)r->rot_dim / (r->rot_dim - 2));
    double lo = 0.0, hi = 1.0;
    if (r->kind == LLAPIS_ROPE_YARN) {
        auto dim = [&](double turns) { return r->rot_dim * std::log(r->trained / (turns * two_pi)) / (2.0 * std::log(base)); };
        lo = std::max(std::floor(dim(r->high)), 0.0);
        hi = std::max(std::min(std::ceil(dim(r->low)), r->rot_dim - 1.0), lo + 0.001);
    }
    for (int i = 0; i < half; ++i) {
        double f = std::pow(base, -2.0 * i / r->rot_dim);
        if (r->divisors) f /= r->divisors[i];
        if (r->kind == LLAPIS_ROPE_LINEAR) {
            f /= r->factor;
        } else if (banded) {
            const double at = r->kind == LLAPIS_ROPE_YARN ? 1.0 - (i - lo) / (hi - lo)
                                                          : (r->trained * f / two_pi - r->low) / (r->high - r->low);
            const double keep = std::min(std::max(at, 0.0), 1.0);
            f = f * keep + f / r->factor * (1.0 - keep);
        }
        freq[i] = f;
    }
    *magnitude = r->kind == LLAPIS_ROPE_YARN && r->factor > 1.0 ? (float)(0.1 * std::log(r->factor) + 1.0) : 1.0f;
    return 0;
}

int32_t llapis_qk_rope(const llapis_qk_rope_args * a, void * stream) {
    const char * who = "llapis_qk_rope";
    if (!a) return refuse_rope(who, "null arguments");
    if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) return refuse_rope(who, "need type F32, F16 or BF16");
    if (a->n_tokens < 0 || a->n_head < 0 || a->n_kv < 0 || a->n_head > 65536 || a->n_kv > 65536)
        return refuse_rope(who, "need n_tokens >= 0, 0 <= n_head, n_kv <= 65536");
    if (a->n_tokens >= 1 << 24) return refuse_rope(who, "need n_tokens < 2^24");
    if (a->head_dim <= 0 || a->head_dim > 512) return refuse_rope(who, "need 0 < head_dim <= 512");
    if (a->rot_dim < 0 || a->rot_dim % 2 || a->rot_dim > a->head_dim) return refuse_rope(who, "need an even rot_dim, 0 to head_dim");
    if (a->layout != LLAPIS_ROPE_HALF && a->layout != LLAPIS_ROPE_PAIRS) return refuse_rope(who, "unknown layout");
    if (a->n_tokens == 0 || a->n_head + a->n_kv == 0) return 0;
    if (a->rot_dim && (!a->pos || !a->freq)) return refuse_rope(who, "null positions or frequencies");
    if ((a->n_head && (!a->q || !a->q_out)) || (a->n_kv && (!a->k || !a->k_out))) return refuse_rope(who, "null q or k");
    const int64_t wq = (int64_t)a->n_head * a->head_dim, wk = (int64_t)a->n_kv * a->head_dim;
    if (a->n_tokens > 1 && ((a->n_head && a->q_out_stride < wq) || (a->n_kv && a->k_out_stride < wk)))
        return refuse_rope(who, "output rows overlap");
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = a->type == T_F32 ? launch_rope<float>(*a, s) : a->type == T_F16 ? launch_rope<_Float16>(*a, s) : launch_rope<__bf16>(*a, s);
    return e == hipSuccess ? 0 : refuse_rope(who, hipGetErrorString(e));
}

}  // extern "C"
