// kv.h -- the paged key-value cache on the device: parameter blocks of its
// kernels, a step's sequences, and the page geometry (llapis_step.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/llapis_step.h"

namespace llapis {

enum { T_F32 = LLAPIS_T_F32, T_F16 = LLAPIS_T_F16, T_BF16 = LLAPIS_T_BF16 };

// the sequences of a step, as llapis_kv_batch
struct KvSeqs {
    const int32_t * table;
    const int32_t * lens;
    const int32_t * start;      // or null: one row each
    int64_t table_stride;
    int n_seq, n_tokens, max_new, max_pages;
};

constexpr int KV_BLOCK = 32;         // keys of one P V matrix instruction
// waves of a workgroup, and keys of a unit, what the work is shared out in and a
// workgroup takes at a time: 32 a wave, 16 where a wave's part of K and V would
// not leave registers for more waves
constexpr int kv_waves(int head_dim) { return head_dim > 256 ? 8 : 4; }
constexpr int kv_unit(int head_dim) { return kv_waves(head_dim) * (head_dim > 128 ? 16 : 32); }
constexpr int KV_MAX_NEW = 16;

struct KvAttn {
    KvSeqs b;
    const uint8_t * k;
    const uint8_t * v;
    uint64_t k_stride, v_stride;
    int n_pages, page_shift;
    int n_kv, group;                 // query heads of a kv head
    int window, unit;
    float scale;
    int type;                        // of q and out
    const void * q;
    int64_t q_stride;
    void * out;
    int64_t out_stride;
    float * lse;
    float * row_ml;                  // or null.  Rows that one run has all of stay parts: out is fp32 and
                                     // unnormalised, here [n_tokens][heads][2] are their maxima and sums
    int32_t * base;                  // [n_seq + 1] first unit of each sequence, [n_seq] their number
    int nt;                          // 16-row tiles of a workgroup
    int runs, tiles;                 // runs (a multiple of 8) of `tiles` workgroups, one for each 16 nt query rows
    float * ml;                      // [runs][tiles][2 parts][16 nt rows][2] running maximum and sum of a partial result
    float * acc;                     // [runs][tiles][2 parts][16 nt rows][head_dim]
};

// tiles of 16 query rows a workgroup holds
inline int kv_tiles(int rows) { return rows <= 16 ? 1 : 2; }
// workgroups of the kernel that a CU's registers and LDS hold
constexpr int kv_wgs(int head_dim, int nt) { return head_dim > 256 ? 1 : nt == 2 ? 2 : head_dim == 64 ? 4 : 3; }

// llapis_last_error() gets the message; returns -1
int32_t refuse(const char * msg) noexcept;

hipError_t launch_kv_attn_f16(const KvAttn & p, int head_dim, hipStream_t s);
hipError_t launch_kv_attn_bf16(const KvAttn & p, int head_dim, hipStream_t s);
hipError_t launch_kv_attn_q8(const KvAttn & p, int head_dim, hipStream_t s);

#if defined(__HIPCC__)

namespace dev {

// rows of sequence s: its new tokens' first row and number, and its length
struct SeqRows { int row0, n, len; };

__device__ __forceinline__ SeqRows seq_rows(const KvSeqs & b, int s) {
    SeqRows r;
    r.len = max(b.lens[s], 0);
    if (b.start) {
        // rows cut at a bound are the last ones: the others keep their positions
        const int64_t want = max((int64_t)b.start[s + 1] - max(b.start[s], 0), (int64_t)0);
        r.row0 = min(max(b.start[s], 0), b.n_tokens);
        r.n = (int)min(want, (int64_t)min(b.n_tokens - r.row0, b.max_new));
        r.len = (int)max(r.len - (want - r.n), (int64_t)0);
    } else {
        r.row0 = s;
        r.n = s < b.n_tokens ? 1 : 0;
    }
    return r;
}

}  // namespace dev

#endif

}  // namespace llapis
