// kv_extend.hip -- pages and slots for the new tokens of a step (llapis_step.h).
#include <algorithm>
#include <cstdio>

#include "kv.h"

namespace llapis {
namespace dev {

// Which sequences grow is decided by one workgroup: three sums over the sequences
// in their order, the tokens asked for, the pages that those need whose tokens
// fit, and tokens and pages of those that get theirs.  A condition on a sum that
// only grows holds for the first sequences and fails from then on, but for a
// sequence that adds nothing to it.  Rows and table entries then find their
// sequence in the last sums by bisection, in LDS up to EXT_HELD sequences.
//
// Bound by latency: a launch, lengths, three sums over the workgroup, bisection,
// the page: 6.3 us for a decode step of 48 sequences, 4.3 and 3.6 (with the rows in a kernel of
// their own) for 24 prompt chunks of up to 2048 tokens.
constexpr int EXT_WG = 1024, EXT_HELD = 2048;

struct Extend {
    llapis_kv_extend_args a;
    int32_t * first;                   // [n_seq + 1] new pages of earlier sequences, then n_free as it was
};

// exclusive sums over the workgroup's threads in order, and the whole
__device__ __forceinline__ int64_t scan_wg(int64_t x, int64_t * s_part, int64_t & total) {
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
    for (int w = 0; w < EXT_WG / 64; ++w) {
        const int64_t y = s_part[w];
        if (w < wave) before += y;
        total += y;
    }
    return before + v - x;
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page_size) { return (tokens + page_size - 1) / page_size; }

// the last i < n with at[i] <= x, where at[0] <= x < at[n]
__device__ __forceinline__ int find(const int32_t * at, int n, int x) {
    int lo = 0;
    for (int hi = n; hi - lo > 1;) {
        const int mid = lo + (hi - lo) / 2;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// rows i0, i0 + step, ... and new table entries likewise
__device__ __forceinline__ void fill_rows(const Extend & e, const int32_t * start, const int32_t * first, int i0, int step) {
    const llapis_kv_extend_args & a = e.a;
    const int tokens = a.n_seq > 0 ? start[a.n_seq] : 0, pages = a.n_seq > 0 ? first[a.n_seq] : 0;
    const int n_free = e.first[a.n_seq + 1];
    auto fresh = [&](int j) { return a.free_pages[n_free - 1 - j]; };
    for (int r = i0; r < a.n_tokens; r += step) {
        int s = -1, pos = -1;
        int64_t slot = -1;
        if (r < tokens) {
            s = find(start, a.n_seq, r);
            const int n = a.lens_out[s], n_new = start[s + 1] - start[s];
            pos = n - (start[s + 1] - r);
            const int i = pos / a.page_size, held = (int)pages_of(n - n_new, a.page_size);
            const int pg = i < held ? a.page_table[s * a.table_stride + i] : fresh(first[s] + i - held);
            if ((uint32_t)pg < (uint32_t)a.n_pages) slot = (int64_t)pg * a.page_size + (pos - i * a.page_size);
        }
        if (a.pos) a.pos[r] = pos;
        if (a.seq) a.seq[r] = s;
        if (a.slots) a.slots[r] = slot;
    }
    for (int j = i0; j < pages; j += step) {
        const int s = find(first, a.n_seq, j);
        const int held = (int)pages_of(a.lens_out[s] - (start[s + 1] - start[s]), a.page_size);
        a.page_table[s * a.table_stride + held + j - first[s]] = fresh(j);
    }
}

// ALL: rows and table entries too
template <bool ALL>
__global__ __launch_bounds__(EXT_WG) void k_kv_extend(const Extend e) {
    __shared__ int64_t s_part[3][EXT_WG / 64];
    __shared__ int32_t s_start[ALL ? EXT_HELD + 1 : 1], s_first[ALL ? EXT_HELD + 1 : 1];
    const llapis_kv_extend_args & a = e.a;
    const int tid = threadIdx.x, per = (a.n_seq + EXT_WG - 1) / EXT_WG, s0 = tid * per;
    const int64_t room = (int64_t)a.max_pages * a.page_size;
    const int n_free = min(max(a.n_free[0], 0), a.n_pages);
    const bool held = ALL && a.n_seq <= EXT_HELD;
    // a thread's sequences are consecutive; the first stays in registers
    const int n0 = s0 < a.n_seq ? max(a.lens[s0], 0) : 0, w0 = s0 < a.n_seq ? max(a.n_new[s0], 0) : 0;
    auto each = [&](auto f) {
        for (int i = 0; i < per && s0 + i < a.n_seq; ++i) {
            const int n = i ? max(a.lens[s0 + i], 0) : n0, w = i ? max(a.n_new[s0 + i], 0) : w0;
            f(s0 + i, n, n + (int64_t)w <= room ? w : 0);
        }
    };
    int64_t total, asked = 0, need = 0, got = 0;
    each([&](int, int, int w) { asked += w; });
    const int64_t asked0 = scan_wg(asked, s_part[0], total);
    // f(sequence, its length, its tokens if its rows fit, the pages these need)
    auto fitting = [&](auto f) {
        int64_t at = asked0;
        each([&](int s, int n, int w) {
            at += w;
            const int fit = at <= a.n_tokens ? w : 0;
            f(s, n, fit, pages_of(n + (int64_t)fit, a.page_size) - pages_of(n, a.page_size));
        });
    };
    fitting([&](int, int, int, int64_t pages) { need += pages; });
    const int64_t need0 = scan_wg(need, s_part[1], total);
    // f(sequence, its length, the tokens it gets, their pages)
    auto granted = [&](auto f) {
        int64_t at = need0;
        fitting([&](int s, int n, int w, int64_t pages) {
            at += pages;
            const bool ok = pages == 0 || at <= n_free;
            f(s, n, ok ? w : 0, ok ? (int)pages : 0);
        });
    };
    // both below 2^31: the tokens by n_tokens, the pages by n_free
    granted([&](int, int, int w, int pages) { got += ((int64_t)w << 32) + pages; });
    int64_t at = scan_wg(got, s_part[2], total);
    granted([&](int s, int n, int w, int pages) {
        a.lens_out[s] = n + w;
        a.new_start[s] = (int)(at >> 32);
        e.first[s] = (int)at;
        if (held) {
            s_start[s] = (int)(at >> 32);
            s_first[s] = (int)at;
        }
        at += ((int64_t)w << 32) + pages;
    });
    if (tid == 0) {
        a.new_start[a.n_seq] = (int)(total >> 32);
        e.first[a.n_seq] = (int)total;
        e.first[a.n_seq + 1] = n_free;
        a.n_free_out[0] = n_free - (int)total;
        if (held) {
            s_start[a.n_seq] = (int)(total >> 32);
            s_first[a.n_seq] = (int)total;
        }
    }
    if constexpr (ALL) {
        __syncthreads();
        if (held) fill_rows(e, s_start, s_first, tid, EXT_WG);
        else fill_rows(e, a.new_start, e.first, tid, EXT_WG);
    }
}

__global__ __launch_bounds__(256) void k_kv_extend_rows(const Extend e) {
    __shared__ int32_t s_start[EXT_HELD + 1], s_first[EXT_HELD + 1];
    const int i0 = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
    if (e.a.n_seq > EXT_HELD) {
        fill_rows(e, e.a.new_start, e.first, i0, step);
        return;
    }
    for (int s = threadIdx.x; s <= e.a.n_seq; s += 256) {
        s_start[s] = e.a.new_start[s];
        s_first[s] = e.first[s];
    }
    __syncthreads();
    fill_rows(e, s_start, s_first, i0, step);
}

}  // namespace dev

using namespace dev;

namespace {

constexpr int EXT_MAX_SEQ = 1 << 24, EXT_MAX_COUNT = 1 << 30;
// Rows that one workgroup fills; more take a second kernel (16 sequences with 500 rows:
// 6.3 us, with two kernels 7.4; with 2000: 7.8 and 7.6; with 4000: 9.8 and 8.0)
constexpr int EXT_ROWS = 1024;

int32_t refuse_extend(const char * why) noexcept {
    char msg[256];
    snprintf(msg, sizeof msg, "llapis_kv_extend: %s", why);
    return refuse(msg);
}

}  // namespace
}  // namespace llapis

using namespace llapis;

extern "C" {

uint64_t llapis_kv_extend_workspace_size(int32_t n_seq) { return n_seq >= 0 && n_seq < EXT_MAX_SEQ ? ((uint64_t)n_seq + 2) * 4 : 0; }

int32_t llapis_kv_extend(const llapis_kv_extend_args * a, void * workspace, uint64_t ws_bytes, void * stream) {
    if (!a) return refuse_extend("null arguments");
    if (a->n_seq < 0 || a->n_seq >= EXT_MAX_SEQ) return refuse_extend("need 0 <= n_seq < 2^24");
    if (a->n_tokens < 0 || a->n_tokens > EXT_MAX_COUNT) return refuse_extend("need 0 <= n_tokens <= 2^30");
    if (a->page_size <= 0 || a->n_pages <= 0 || a->n_pages > EXT_MAX_COUNT) return refuse_extend("need page_size > 0 and 0 < n_pages <= 2^30");
    if (a->max_pages <= 0 || a->table_stride < a->max_pages) return refuse_extend("need 0 < max_pages <= table_stride");
    if ((int64_t)a->max_pages * a->page_size > EXT_MAX_COUNT) return refuse_extend("max_pages * page_size above 2^30");
    if (a->n_seq > 0 && (!a->page_table || !a->lens || !a->n_new || !a->lens_out)) return refuse_extend("null page table, lengths or n_new");
    if (!a->free_pages || !a->n_free || !a->n_free_out || !a->new_start) return refuse_extend("null free pages or new_start");
    if (!workspace || ((uintptr_t)workspace & 3) || ws_bytes < llapis_kv_extend_workspace_size(a->n_seq))
        return refuse_extend("workspace too small or not 4-byte aligned");
    const Extend e{*a, (int32_t *)workspace};
    hipStream_t s = (hipStream_t)stream;
    const bool one = a->n_tokens <= EXT_ROWS;
    if (one) hipLaunchKernelGGL((k_kv_extend<true>), dim3(1), dim3(EXT_WG), 0, s, e);
    else hipLaunchKernelGGL((k_kv_extend<false>), dim3(1), dim3(EXT_WG), 0, s, e);
    hipError_t err = hipGetLastError();
    if (err == hipSuccess && !one) {
        hipLaunchKernelGGL(k_kv_extend_rows, dim3(std::min((a->n_tokens + 255) / 256, 1024)), dim3(256), 0, s, e);
        err = hipGetLastError();
    }
    return err == hipSuccess ? 0 : refuse_extend(hipGetErrorString(err));
}

}  // extern "C"
