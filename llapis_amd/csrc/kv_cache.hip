// kv_cache.hip -- the paged key-value cache (llapis_step.h): attention's entry
// point and the join of its parts, the append, and the operations on pages.
#include <algorithm>
#include <cstdio>

#include "kv_attn.h"

namespace llapis {
namespace dev {

// ---------------------------------------------------------------- join
//
// The parts of an item that several workgroups of k_kv_attn shared: with M the
// largest maximum, out = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i.  A
// workgroup takes 1024 / PG values of an item's tile, four a thread; its PG
// groups of threads take every PG-th part, each under a running maximum of its
// own, and are added in their order.  A part is read once, its maximum and sum
// with its values, so that the loads of several parts are in flight (a first pass
// over the maxima, then the values: 4 tokens of 11203 keys with the attention
// kernel 71 us, so 38).  A launch and a chain of four loads: 4.7 us for 700 keys,
// 6.8 for the 88 parts a head of 11203, 8.5 for 48 sequences.  It is a kernel of its
// own: added by the workgroup that ends last, the parts would need counters that are 0
// before the call, and the workspace, which calls share, carries nothing over.
template <int PG>
__global__ __launch_bounds__(256) void k_kv_join(const KvAttn p, int head_dim, float p_shift) {
    constexpr int TPG = 256 / PG;
    __shared__ f4v s_acc[PG][TPG];
    __shared__ float s_m[PG][TPG], s_l[PG][TPG];
    const int tid = threadIdx.x, g = tid / TPG, e = tid - g * TPG, tile_rows = 16 * p.nt;
    const int seq = blockIdx.x / (p.n_kv * p.tiles), rest = blockIdx.x - seq * p.n_kv * p.tiles;
    const int total = p.base[p.b.n_seq], base = p.base[seq];
    const SeqUnits su = seq_units(p.b, seq, p.page_shift, p.window, p.unit);
    const int head = rest / p.tiles, tile = rest - head * p.tiles;
    const int n_rows = min(su.r.n * p.group - tile * tile_rows, tile_rows);
    const int at = (blockIdx.y * TPG + e) * 4, r = at / head_dim, d = at - r * head_dim;
    if ((int)(blockIdx.y * TPG * 4) >= n_rows * head_dim) return;      // also: no such item
    // the runs of the item's first and last unit
    const Runs runs(total, runs_of(p.runs, total));
    const int first = base + head * item_steps(su.units);
    const int w0 = runs.owner(first + 1), w1 = runs.owner(first + 2 * su.units - 1);
    if (w0 == w1) return;                                              // written by k_kv_attn
    const bool live = r < n_rows;
    f4v a = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -__builtin_inff(), l = 0.0f;
    constexpr int UN = 8;
    for (int i0 = g; i0 <= w1 - w0; i0 += PG * UN) {
        f4v x[UN];
        float xm[UN], xl[UN];
#pragma unroll
        for (int j = 0; j < UN; ++j) {
            const int i = i0 + PG * j;
            x[j] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
            xm[j] = -__builtin_inff();
            xl[j] = 0.0f;
            if (live && i <= w1 - w0) {
                const int64_t row = (((int64_t)(w0 + i) * p.tiles + tile) * 2 + (i == 0)) * tile_rows + r;
                x[j] = *(const f4v *)(p.acc + row * head_dim + d);
                xm[j] = p.ml[2 * row];
                xl[j] = p.ml[2 * row + 1];
            }
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < UN; ++j) top = fmaxf(top, xm[j]);
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f(m - ref);
        a *= f;
        l *= f;
        m = top;
#pragma unroll
        for (int j = 0; j < UN; ++j) {
            const float w = __builtin_amdgcn_exp2f(xm[j] - ref);
            a += w * x[j];
            l += w * xl[j];
        }
    }
    if (PG > 1) {
        s_acc[g][e] = a;
        s_m[g][e] = m;
        s_l[g][e] = l;
        __syncthreads();
        if (g > 0) return;
        float top = m;
        for (int i = 1; i < PG; ++i) top = fmaxf(top, s_m[i][e]);
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f(m - ref);
        a *= f;
        l *= f;
        m = top;
        for (int i = 1; i < PG; ++i) {
            const float w = __builtin_amdgcn_exp2f(s_m[i][e] - ref);
            a += w * s_acc[i][e];
            l += w * s_l[i][e];
        }
    }
    if (!live) return;
    const int rr = tile * tile_rows + r, tok = rr / p.group, hq = head * p.group + rr - tok * p.group;
    const int64_t row = su.r.row0 + tok;
    const float inv = 1.0f / l;
    store4(p.out, p.type, row * p.out_stride + (int64_t)hq * head_dim + d, l == 0.0f ? f4v{0.0f, 0.0f, 0.0f, 0.0f} : a * inv);
    if (p.lse && d == 0)
        p.lse[row * (p.n_kv * p.group) + hq] = l == 0.0f ? -__builtin_inff() : (m + (__builtin_amdgcn_logf(l) - p_shift)) * KV_LN2;
}

// -------------------------------------------------------------- append
//
// Two workgroups, K's and V's, for 32 consecutive positions (from a multiple of
// 32) of one sequence and kv head.  K: a thread converts eight values of a row,
// written as they lie.  V: a thread converts a column's eight consecutive
// positions, which are one 16-byte store in the transposed page; at the ends of a
// run the positions that the call brings are stored one by one.  A thread asks for
// all its values before it converts the first.  Bound by memory: 2048 prompt tokens
// of 8 heads of 256 from F32 into F16, 50 MB, 12.1 us (15 with K and V in one
// workgroup; a large copy's rate would be 10); 4 tokens of 48 sequences 4.4 us, a
// launch and three dependent loads.
constexpr int APP_POS = 32;

struct KvAppend {
    KvSeqs b;
    uint8_t * k;
    uint8_t * v;
    uint64_t k_stride, v_stride;
    int n_pages, page_shift, n_kv, head_dim, x_type;
    const void * xk;
    const void * xv;
    int64_t xk_stride, xv_stride;
};

__device__ __forceinline__ float load1(const void * p, int type, int64_t at) {
    if (type == T_F32) return ((const float *)p)[at];
    if (type == T_F16) return (float)((const _Float16 *)p)[at];
    return __builtin_bit_cast(float, (uint32_t)((const uint16_t *)p)[at] << 16);
}

// q8_0 of one value, given its block's largest magnitude
struct Q8Scale { float id; uint16_t d; };
__device__ __forceinline__ Q8Scale q8_scale(float amax) {
    const float d = __fdiv_rn(amax, 127.0f);
    return {d > 0.0f ? __fdiv_rn(1.0f, d) : 0.0f, __builtin_bit_cast(uint16_t, (_Float16)d)};
}
// the larger magnitude, NaN if one is: the block's scale then says so
__device__ __forceinline__ float larger(float a, float b) {
    b = fabsf(b);
    return a != a || b != b ? __builtin_nanf("") : fmaxf(a, b);
}
__device__ __forceinline__ int q8_value(float x, float id) { return (int)__builtin_rintf(x * id) & 0xFF; }

// HDT: the head size, 0 for one that is not a multiple of 64
template <int CT, int HDT>
__global__ __launch_bounds__(256) void k_kv_append(const KvAppend p) {
    constexpr int EL = CT == KV_Q8 ? 1 : 2;
    const int seq = blockIdx.x, head = blockIdx.z >> 1, tid = threadIdx.x;
    const SeqRows r = seq_rows(p.b, seq);
    const int p0 = r.len - r.n;                                   // may be negative: such tokens have no place
    const int cap = p.b.max_pages << p.page_shift;
    if (p0 >= cap) return;
    const int base = (max(p0, 0) & ~(APP_POS - 1)) + APP_POS * blockIdx.y;
    const int from = max(p0, base), to = min(min(r.len, base + APP_POS), cap);
    if (from >= to) return;
    const int HD = HDT ? HDT : p.head_dim, page = 1 << p.page_shift, mask = page - 1;
    const int32_t * row = p.b.table + seq * p.b.table_stride;
    const uint64_t part = (uint64_t)head * page * (CT == KV_Q8 ? HD + HD / 16 : 2 * HD);
    const int items = APP_POS / 8 * HD;                           // of eight values
    constexpr int UN = HDT ? (HDT / 64 < 4 ? HDT / 64 : 4) : 1;   // of a thread at a time
    if (blockIdx.z & 1) {
        // V: (eight positions, column)
        for (int i0 = tid; i0 < items; i0 += 256 * UN) {
            float x[UN][8];
            int pg[UN];
#pragma unroll
            for (int e = 0; e < UN; ++e) {
                const int i = i0 + 256 * e, oct = base + 8 * (i / HD), c = i % HD;
                const int lo = max(from, oct), hi = min(to, oct + 8);
                pg[e] = lo < hi ? row[oct >> p.page_shift] : -1;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[e][j] = oct + j >= lo && oct + j < hi
                                  ? load1(p.xv, p.x_type, (int64_t)(r.row0 + oct + j - p0) * p.xv_stride + head * HD + c) : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < UN; ++e) {
                const int i = i0 + 256 * e, oct = base + 8 * (i / HD), c = i % HD;
                const int lo = max(from, oct), hi = min(to, oct + 8);
                if ((uint32_t)pg[e] >= (uint32_t)p.n_pages) continue;         // the same in the 32 threads of a block of columns
                uint8_t * dst = p.v + (uint64_t)pg[e] * p.v_stride + part;
                uint8_t * at = dst + (c * page + (oct & mask)) * EL;
                if constexpr (CT == KV_Q8) {
                    u2 w = {0, 0};
                    uint16_t d[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float amax = fabsf(x[e][j]);
#pragma unroll
                        for (int o = 16; o; o >>= 1) amax = larger(amax, __shfl_xor(amax, o, 64));
                        const Q8Scale s = q8_scale(amax);
                        w[j >> 2] |= (uint32_t)q8_value(x[e][j], s.id) << (8 * (j & 3));
                        d[j] = s.d;
                    }
                    uint16_t * sc = (uint16_t *)(dst + page * HD) + (c / 32) * page + (oct & mask);
                    if (hi - lo == 8) {
                        *(u2 *)at = w;
                        if (c % 32 == 0)
#pragma unroll
                            for (int j = 0; j < 8; ++j) sc[j] = d[j];
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (oct + j >= lo && oct + j < hi) {
                                at[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
                                if (c % 32 == 0) sc[j] = d[j];
                            }
                    }
                } else {
                    u4 w[1];
                    split8<CT == KV_F16, 1>(x[e], w);
                    if (hi - lo == 8) {
                        *(u4 *)at = w[0];
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (oct + j >= lo && oct + j < hi) ((uint16_t *)at)[j] = (uint16_t)(w[0][j >> 1] >> (16 * (j & 1)));
                    }
                }
            }
        }
        return;
    }
    // K: (position, eight values)
    const int chunks = HD / 8;
    for (int i0 = tid; i0 < items; i0 += 256 * UN) {
        float x[UN][8];
        int pg[UN];
#pragma unroll
        for (int e = 0; e < UN; ++e) {
            const int i = i0 + 256 * e, at = base + i / chunks, c = i % chunks;
            const bool live = at >= from && at < to;
            pg[e] = live ? row[at >> p.page_shift] : -1;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[e][j] = 0.0f;
            if (live) load8(p.xk, p.x_type, (int64_t)(r.row0 + at - p0) * p.xk_stride + head * HD + 8 * c, x[e]);
        }
#pragma unroll
        for (int e = 0; e < UN; ++e) {
            const int i = i0 + 256 * e, at = base + i / chunks, c = i % chunks;
            const bool there = (uint32_t)pg[e] < (uint32_t)p.n_pages;
            uint8_t * dst = p.k + (uint64_t)(there ? pg[e] : 0) * p.k_stride + part;
            if constexpr (CT == KV_Q8) {
                float amax = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = larger(amax, x[e][j]);
                amax = larger(amax, __shfl_xor(amax, 1, 64));     // four threads hold a block of 32
                amax = larger(amax, __shfl_xor(amax, 2, 64));
                if (there) {
                    const Q8Scale s = q8_scale(amax);
                    u2 w = {0, 0};
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j >> 2] |= (uint32_t)q8_value(x[e][j], s.id) << (8 * (j & 3));
                    *(u2 *)(dst + (at & mask) * HD + 8 * c) = w;
                    if (c % 4 == 0) *(uint16_t *)(dst + page * HD + ((c / 4) * page + (at & mask)) * 2) = s.d;
                }
            } else if (there) {
                u4 w[1];
                split8<CT == KV_F16, 1>(x[e], w);
                *(u4 *)(dst + ((at & mask) * HD + 8 * c) * EL) = w[0];
            }
        }
    }
}

template <int CT>
void launch_append(const KvAppend & p, dim3 grid, hipStream_t s) {
    const dim3 wg(256);
    switch (p.head_dim) {
        case 64: hipLaunchKernelGGL((k_kv_append<CT, 64>), grid, wg, 0, s, p); break;
        case 128: hipLaunchKernelGGL((k_kv_append<CT, 128>), grid, wg, 0, s, p); break;
        case 192: hipLaunchKernelGGL((k_kv_append<CT, 192>), grid, wg, 0, s, p); break;
        case 256: hipLaunchKernelGGL((k_kv_append<CT, 256>), grid, wg, 0, s, p); break;
        case 512: hipLaunchKernelGGL((k_kv_append<CT, 512>), grid, wg, 0, s, p); break;
        default: hipLaunchKernelGGL((k_kv_append<CT, 0>), grid, wg, 0, s, p);
    }
}

// --------------------------------------------------------------- pages

// counts that loops run up to leave room for their steps in 32 bits
constexpr int KV_MAX_COUNT = 1 << 30;
constexpr int PG_CHUNK = 16384;                                   // bytes a workgroup copies at a time

// bytes [at, at + PG_CHUNK) of a page of `plane`, from one page to another: four
// 128-bit loads in flight a lane.  Bound by memory: a compaction's moves of 500 MB of
// reads and writes take 97 to 100 us, 5.0 to 5.2 TB/s; a large copy's rate is 5.0.
__device__ __forceinline__ void copy_chunk(const llapis_kv_planes & p, int plane, int from, int to, uint64_t at) {
    const uint64_t n = p.bytes[plane];
    if (at >= n) return;
    const u4 * s = (const u4 *)((const uint8_t *)p.base[plane] + (uint64_t)from * p.stride[plane] + at);
    u4 * d = (u4 *)((uint8_t *)p.base[plane] + (uint64_t)to * p.stride[plane] + at);
    const int n16 = (int)(min((uint64_t)PG_CHUNK, n - at) >> 4);
    u4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (threadIdx.x + 256 * j < n16) w[j] = s[threadIdx.x + 256 * j];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (threadIdx.x + 256 * j < n16) d[threadIdx.x + 256 * j] = w[j];
}

__device__ __forceinline__ bool in_pool(int page, int n_pages) { return (uint32_t)page < (uint32_t)n_pages; }

// pairs in the order (pair, plane, chunk); the number of pairs may be the device's
__device__ __forceinline__ void copy_pairs(const llapis_kv_planes & p, const int32_t * from, const int32_t * to, int step,
                                           int n_pairs, int chunks) {
    const int64_t per = (int64_t)p.n_planes * chunks, all = n_pairs * per;
    for (int64_t i = blockIdx.x; i < all; i += gridDim.x) {
        const int pair = (int)(i / per), rest = (int)(i - pair * per), plane = rest / chunks;
        const int a = from[(int64_t)pair * step], b = to[(int64_t)pair * step];
        if (in_pool(a, p.n_pages) && in_pool(b, p.n_pages)) copy_chunk(p, plane, a, b, (uint64_t)(rest - plane * chunks) * PG_CHUNK);
    }
}

__global__ __launch_bounds__(256) void k_kv_copy(const llapis_kv_planes p, const int32_t * pairs, int n_pairs, int chunks) {
    copy_pairs(p, pairs, pairs + 1, 2, n_pairs, chunks);
}

// workgroup (plane x chunk, fork): a part of the last page; the first of each
// fork writes the target's row and length (no workgroup reads a target's)
__global__ __launch_bounds__(256) void k_kv_fork(const llapis_kv_planes p, int32_t * table, int64_t table_stride,
                                                 int max_pages, int32_t * lens, int n_seq, const int32_t * forks, int chunks) {
    const int32_t * f = forks + 3 * (int64_t)blockIdx.y;
    const int src = f[0], dst = f[1], fresh = f[2];
    if ((uint32_t)src >= (uint32_t)n_seq || (uint32_t)dst >= (uint32_t)n_seq || src == dst) return;
    const int len = lens[src];
    if (len < 0 || (int64_t)len > (int64_t)max_pages * p.page_size) return;
    const int full = len / p.page_size;
    const bool part = len % p.page_size != 0;
    const int32_t * from = table + src * table_stride;
    const int last = part ? from[full] : -1;
    if (part && (!in_pool(last, p.n_pages) || !in_pool(fresh, p.n_pages) || fresh == last)) return;
    if (blockIdx.x == 0) {
        int32_t * to = table + dst * table_stride;
        for (int i = threadIdx.x; i < max_pages; i += 256) to[i] = i < full ? from[i] : i == full && part ? fresh : -1;
        if (threadIdx.x == 0) lens[dst] = len;
    }
    if (part) copy_chunk(p, blockIdx.x / chunks, last, fresh, (uint64_t)(blockIdx.x % chunks) * PG_CHUNK);
}

__global__ __launch_bounds__(256) void k_kv_zero(int32_t * p, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

__device__ __forceinline__ int held_pages(int len, int page_size, int max_pages) {
    return (int)min(((int64_t)max(len, 0) + page_size - 1) / page_size, (int64_t)max_pages);
}

__global__ __launch_bounds__(256) void k_kv_mark(const int32_t * table, int64_t table_stride, int max_pages,
                                                 const int32_t * lens, int page_size, int n_pages, int32_t * refs) {
    const int seq = blockIdx.x, n = held_pages(lens[seq], page_size, max_pages);
    for (int i = blockIdx.y * 256 + threadIdx.x; i < n; i += 256 * gridDim.y) {
        const int pg = table[seq * table_stride + i];
        if (in_pool(pg, n_pages)) atomicAdd(&refs[pg], 1);
    }
}

constexpr int SCAN_WG = 1024;

// exclusive sum of `x` over the workgroup; `total` gets the whole sum
__device__ __forceinline__ int block_scan(int x, int * s_part, int & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int v = x;
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(v, o, 64);
        if (lane >= o) v += u;
    }
    __syncthreads();
    if (lane == 63) s_part[wave] = v;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < SCAN_WG / 64; ++w) {
        if (w < wave) before += s_part[w];
        total += s_part[w];
    }
    return before + v - x;
}

__global__ __launch_bounds__(SCAN_WG) void k_kv_free(const int32_t * refs, int n_pages, int32_t * free_pages, int32_t * n_free) {
    __shared__ int s_part[SCAN_WG / 64];
    int at = 0;
    for (int p0 = 0; p0 < n_pages; p0 += SCAN_WG) {
        const int pg = p0 + threadIdx.x;
        const bool is_free = pg < n_pages && refs[pg] == 0;
        int total;
        const int i = block_scan(is_free, s_part, total);
        if (is_free && free_pages) free_pages[at + i] = pg;
        at += total;
    }
    if (free_pages)
        for (int i = at + threadIdx.x; i < n_pages; i += SCAN_WG) free_pages[i] = -1;
    if (n_free && threadIdx.x == 0) *n_free = at;
}

// The moves of a compaction: place[p] = where page p goes (-1: nowhere), the
// pairs (from, to), and their number.
__device__ __forceinline__ void plan_moves(const int * refs, int n_pages, int32_t * place, int32_t * from, int32_t * to,
                                           int32_t * n_moves, int32_t * n_live, int32_t * refs_out, int * s_part) {
    int live = 0, total;
    for (int p0 = threadIdx.x; p0 < n_pages; p0 += SCAN_WG) live += refs[p0] > 0;
    (void)block_scan(live, s_part, total);
    live = total;
    int n_from = 0, n_to = 0;
    for (int p0 = 0; p0 < n_pages; p0 += SCAN_WG) {
        const int pg = p0 + threadIdx.x;
        const int r = pg < n_pages ? refs[pg] : 0;
        const bool moves = r > 0 && pg >= live, hole = pg < live && pg < n_pages && r == 0;
        // at most one of the two lists gets a tile's page: one scan for both, in halves
        const int i = block_scan((moves ? 1 : 0) + (hole ? 1 << 16 : 0), s_part, total);
        if (moves) from[n_from + (i & 0xFFFF)] = pg;
        if (hole) to[n_to + (i >> 16)] = pg;
        if (pg < n_pages) {
            place[pg] = r > 0 && pg < live ? pg : -1;
            if (refs_out) refs_out[pg] = pg < live ? r : 0;
        }
        n_from += total & 0xFFFF;
        n_to += total >> 16;
    }
    __syncthreads();
    // as many pages lie behind the new end as there are holes before it
    for (int i = threadIdx.x; i < n_from; i += SCAN_WG) {
        place[from[i]] = to[i];
        if (refs_out) refs_out[to[i]] = refs[from[i]];
    }
    if (threadIdx.x == 0) {
        *n_moves = n_from;
        *n_live = live;
    }
}

__global__ __launch_bounds__(SCAN_WG) void k_kv_plan(const int32_t * refs, int n_pages, int32_t * place, int32_t * from,
                                                     int32_t * to, int32_t * n_moves, int32_t * n_live, int32_t * refs_out) {
    __shared__ int s_part[SCAN_WG / 64];
    plan_moves(refs, n_pages, place, from, to, n_moves, n_live, refs_out, s_part);
}

// All of the above for a pool and a table that one workgroup goes through in the
// time of a few launches: the counts are in LDS.  1024 pages and 64 sequences:
// 11.8 us; four kernels' launches, 3.9 us each, are more than that.  (8192 counts are
// 32 KB of LDS, 65536 entries 64 a thread.)
constexpr int SMALL_PAGES = 8192, SMALL_ENTRIES = 65536;

__global__ __launch_bounds__(SCAN_WG) void k_kv_plan_small(const int32_t * table, int64_t table_stride, int max_pages,
                                                           const int32_t * lens, int n_seq, int page_size, int n_pages,
                                                           int32_t * place, int32_t * from, int32_t * to, int32_t * n_moves,
                                                           int32_t * n_live, int32_t * refs_out, int32_t * table_out) {
    __shared__ int s_part[SCAN_WG / 64];
    __shared__ int s_refs[SMALL_PAGES];
    for (int i = threadIdx.x; i < n_pages; i += SCAN_WG) s_refs[i] = 0;
    __syncthreads();
    // a wave a row at a time
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int seq = wave; seq < n_seq; seq += SCAN_WG / 64) {
        const int n = held_pages(lens[seq], page_size, max_pages);
        for (int i = lane; i < n; i += 64) {
            const int pg = table[seq * table_stride + i];
            if (in_pool(pg, n_pages)) atomicAdd(&s_refs[pg], 1);
        }
    }
    __syncthreads();
    plan_moves(s_refs, n_pages, place, from, to, n_moves, n_live, refs_out, s_part);
    __syncthreads();
    for (int seq = wave; seq < n_seq; seq += SCAN_WG / 64) {
        const int n = held_pages(lens[seq], page_size, max_pages);
        for (int i = lane; i < max_pages; i += 64) {
            const int pg = i < n ? table[seq * table_stride + i] : -1;
            table_out[seq * table_stride + i] = in_pool(pg, n_pages) ? place[pg] : -1;
        }
    }
}

__global__ __launch_bounds__(256) void k_kv_remap(const int32_t * table, int64_t table_stride, int max_pages,
                                                  const int32_t * lens, int page_size, int n_pages, const int32_t * place,
                                                  int32_t * table_out) {
    const int seq = blockIdx.x, n = held_pages(lens[seq], page_size, max_pages);
    for (int i = blockIdx.y * 256 + threadIdx.x; i < max_pages; i += 256 * gridDim.y) {
        const int pg = i < n ? table[seq * table_stride + i] : -1;
        table_out[seq * table_stride + i] = in_pool(pg, n_pages) ? place[pg] : -1;
    }
}

__global__ __launch_bounds__(256) void k_kv_move(const llapis_kv_planes p, const int32_t * from, const int32_t * to,
                                                 const int32_t * n_moves, int chunks) {
    copy_pairs(p, from, to, 1, *n_moves, chunks);
}

}  // namespace dev

using namespace dev;

namespace {

#define KV_TRY(expr)                                                       \
    do {                                                                   \
        const hipError_t e_ = (expr);                                      \
        if (e_ != hipSuccess) return refuse(hipGetErrorString(e_));        \
    } while (0)

bool aligned16(const void * p) { return ((uintptr_t)p & 15) == 0; }

int log2_of(int x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return s;
}

int el_bytes(int type) { return type == T_F32 ? 4 : 2; }
bool act_type(int type) { return type == T_F32 || type == T_F16 || type == T_BF16; }

const char * check_cache(const llapis_kv_cache * c) {
    if (!c) return "null cache";
    const uint64_t need = llapis_kv_page_bytes(c->type, c->n_kv, c->head_dim, c->page_size);
    if (!need)
        return "need type F16, BF16 or Q8_0, head_dim 64, 96, 128, 192, 256 or 512, page_size 16, 32, 64, 128 or 256, "
               "0 < n_kv <= 1024";
    if (c->n_pages <= 0) return "need n_pages > 0";
    if (!c->k || !c->v) return "null pool";
    if (!aligned16(c->k) || !aligned16(c->v) || c->k_stride % 16 || c->v_stride % 16) return "pools and page strides must be 16-byte aligned";
    if (c->k_stride < need || c->v_stride < need) return "page stride shorter than a page";
    return nullptr;
}

const char * check_batch(const llapis_kv_batch * b, int page_size) {
    if (!b) return "null batch";
    if (b->n_seq < 0 || b->n_tokens < 0 || b->max_new < 0) return "negative batch size";
    if (b->max_pages <= 0 || b->table_stride < b->max_pages) return "need 0 < max_pages <= table_stride";
    if ((int64_t)b->max_pages * page_size > (1 << 30)) return "max_pages * page_size above 2^30";
    if (b->n_seq > 0 && (!b->page_table || !b->lens)) return "null page table or lengths";
    return nullptr;
}

int32_t refuse_as(const char * who, const char * why) noexcept {
    char msg[320];
    snprintf(msg, sizeof msg, "%s: %s", who, why);
    return refuse(msg);
}

KvSeqs seqs_of(const llapis_kv_batch * b) {
    return {b->page_table, b->lens, b->new_start, b->table_stride, b->n_seq, b->n_tokens, b->new_start ? b->max_new : 1, b->max_pages};
}

// sizes of an attention call
struct AttnPlan {
    int nt, runs, tiles;
    uint64_t base_bytes, ml_bytes, acc_bytes;
    uint64_t bytes() const { return base_bytes + ml_bytes + acc_bytes; }
};

// a launch has fewer than 2^32 threads in x: workgroups of 256
constexpr int KV_MAX_GRID = 1 << 24;

// an item may have several units, and parts to join
bool needs_join(const llapis_kv_cache * c, const llapis_kv_batch * b) { return (int64_t)b->max_pages * c->page_size > kv_unit(c->head_dim); }

const char * plan_attention(const llapis_kv_cache * c, const llapis_kv_batch * b, int n_head, AttnPlan & a) {
    const int max_new = b->new_start ? b->max_new : 1;
    if (n_head <= 0 || n_head > 1024 || n_head % c->n_kv) return "need n_head <= 1024, a multiple of n_kv";
    if (max_new > KV_MAX_NEW) return "more than 16 new tokens a sequence";
    const int rows = n_head / c->n_kv * std::max(max_new, 1);
    a.nt = kv_tiles(rows);
    a.tiles = (rows + 16 * a.nt - 1) / (16 * a.nt);
    const int unit = kv_unit(c->head_dim);
    const int64_t units = ((int64_t)b->max_pages * c->page_size + unit - 1) / unit + 1;
    if (b->n_seq > 0 && units * c->n_kv > ((1 << 29) - 1) / b->n_seq) return "the batch has 2^29 units of work or more";
    const int64_t all = units * c->n_kv * b->n_seq;
    // the join has a workgroup for each (sequence, kv head, tile)
    if (needs_join(c, b) && (int64_t)b->n_seq * c->n_kv * a.tiles >= KV_MAX_GRID)
        return "2^24 or more (sequence, kv head, 32 query rows)";
    // as many workgroups as the card holds at once
    const int64_t most = std::max(256 * kv_wgs(c->head_dim, a.nt) / a.tiles, 8);
    a.runs = (int)((std::min(most, all) + 7) / 8 * 8);
    const uint64_t parts = (uint64_t)a.runs * a.tiles * 2;
    a.base_bytes = ((uint64_t)(b->n_seq + 1) * 4 + 255) / 256 * 256;
    a.ml_bytes = parts * 16 * a.nt * 2 * 4;
    a.acc_bytes = parts * 16 * a.nt * c->head_dim * 4;
    return nullptr;
}

// chunks of the longest plane's page; 0 where a plane is refused
const char * check_planes(const llapis_kv_planes * p, int & chunks) {
    if (!p) return "null planes";
    if (p->n_planes <= 0 || p->n_planes > LLAPIS_KV_MAX_PLANES) return "need 0 < n_planes <= 128";
    if (p->n_pages <= 0 || p->n_pages > KV_MAX_COUNT || p->page_size <= 0) return "need 0 < n_pages <= 2^30 and page_size > 0";
    uint64_t most = 0;
    for (int i = 0; i < p->n_planes; ++i) {
        if (!p->base[i] || !aligned16(p->base[i]) || p->stride[i] % 16 || p->bytes[i] % 16 || !p->bytes[i] ||
            p->stride[i] < p->bytes[i])
            return "planes, strides and page bytes must be 16-byte aligned, a stride at least its page";
        most = std::max(most, p->bytes[i]);
    }
    if (most > (uint64_t)1 << 30) return "a page above 2^30 bytes";
    chunks = (int)((most + PG_CHUNK - 1) / PG_CHUNK);
    return nullptr;
}

const char * check_table(const void * table, int64_t stride, int max_pages, const void * lens, int n_seq) {
    if (n_seq < 0) return "negative n_seq";
    if (max_pages <= 0 || max_pages > KV_MAX_COUNT || stride < max_pages) return "need 0 < max_pages <= table_stride, max_pages <= 2^30";
    if (n_seq > 0 && (!table || !lens)) return "null page table or lengths";
    return nullptr;
}

// ... of calls with a workgroup for each row
const char * check_rows(const void * table, int64_t stride, int max_pages, const void * lens, int n_seq) {
    return n_seq >= KV_MAX_GRID ? "need n_seq < 2^24" : check_table(table, stride, max_pages, lens, n_seq);
}

dim3 table_grid(int n_seq, int max_pages) { return dim3(n_seq, std::min((max_pages + 255) / 256, 64)); }

hipError_t launch_refs(const int32_t * table, int64_t stride, int max_pages, const int32_t * lens, int n_seq, int page_size,
                       int n_pages, int32_t * refs, hipStream_t s) {
    hipLaunchKernelGGL(k_kv_zero, dim3((n_pages + 255) / 256), dim3(256), 0, s, refs, n_pages);
    if (n_seq > 0)
        hipLaunchKernelGGL(k_kv_mark, table_grid(n_seq, max_pages), dim3(256), 0, s, table, stride, max_pages, lens, page_size,
                           n_pages, refs);
    return hipGetLastError();
}

}  // namespace
}  // namespace llapis

using namespace llapis;

extern "C" {

uint64_t llapis_kv_page_bytes(int32_t type, int32_t n_kv, int32_t head_dim, int32_t page_size) {
    if (n_kv <= 0 || n_kv > 1024) return 0;
    if (head_dim != 64 && head_dim != 96 && head_dim != 128 && head_dim != 192 && head_dim != 256 && head_dim != 512) return 0;
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1))) return 0;
    const uint64_t values = (uint64_t)n_kv * head_dim * page_size;
    return type == T_F16 || type == T_BF16 ? 2 * values : type == LLAPIS_T_Q8_0 ? values + values / 16 : 0;
}

int32_t llapis_kv_append(const llapis_kv_cache * c, const llapis_kv_batch * b, int32_t x_type, const void * k,
                         int64_t k_stride, const void * v, int64_t v_stride, void * stream) {
    const char * who = "llapis_kv_append";
    const char * bad = check_cache(c);
    if (!bad) bad = check_batch(b, c->page_size);
    if (bad) return refuse_as(who, bad);
    if (!act_type(x_type)) return refuse_as(who, "need F32, F16 or BF16 keys and values");
    const KvSeqs q = seqs_of(b);
    if (q.n_seq == 0 || q.n_tokens == 0 || q.max_new == 0) return 0;
    if (!k || !v) return refuse_as(who, "null keys or values");
    const int es = el_bytes(x_type);
    if (!aligned16(k) || !aligned16(v) || (k_stride * es) % 16 || (v_stride * es) % 16)
        return refuse_as(who, "keys and values must be 16-byte aligned, rows too");
    if (q.n_tokens > 1 && (k_stride < (int64_t)c->n_kv * c->head_dim || v_stride < (int64_t)c->n_kv * c->head_dim))
        return refuse_as(who, "rows shorter than n_kv * head_dim");
    // a run of max_new positions touches this many aligned tiles; none lies past the table
    const int64_t tiles = std::min<int64_t>(((int64_t)q.max_new + APP_POS - 2) / APP_POS + 1,
                                            ((int64_t)b->max_pages * c->page_size + APP_POS - 1) / APP_POS);
    if (tiles > 65535) return refuse_as(who, "more than 65535 * 32 new tokens of a sequence");
    if (q.n_seq >= KV_MAX_GRID) return refuse_as(who, "need n_seq < 2^24");
    KvAppend p{q, (uint8_t *)c->k, (uint8_t *)c->v, c->k_stride, c->v_stride, c->n_pages, log2_of(c->page_size), c->n_kv,
               c->head_dim, x_type, k, v, k_stride, v_stride};
    const dim3 grid(q.n_seq, (unsigned)tiles, 2 * c->n_kv);
    hipStream_t s = (hipStream_t)stream;
    if (c->type == T_F16) launch_append<KV_F16>(p, grid, s);
    else if (c->type == T_BF16) launch_append<KV_BF16>(p, grid, s);
    else launch_append<KV_Q8>(p, grid, s);
    KV_TRY(hipGetLastError());
    return 0;
}

uint64_t llapis_kv_attention_workspace_size(const llapis_kv_cache * c, const llapis_kv_batch * b, int32_t n_head) {
    AttnPlan a;
    if (!c || !b || !llapis_kv_page_bytes(c->type, c->n_kv, c->head_dim, c->page_size) || b->n_seq < 0 || b->max_pages <= 0 ||
        (int64_t)b->max_pages * c->page_size > (1 << 30) || plan_attention(c, b, n_head, a))
        return 0;
    // three tiles a run have more workgroups in their multiple of eight runs than four:
    // the most of what fewer new tokens take
    uint64_t most = a.bytes();
    llapis_kv_batch less = *b;
    for (less.max_new = 1; b->new_start && less.max_new < b->max_new; ++less.max_new)
        if (!plan_attention(c, &less, n_head, a)) most = std::max(most, a.bytes());
    return most;
}

int32_t llapis_kv_attention(const llapis_kv_cache * c, const llapis_kv_batch * b, const llapis_kv_query * q, void * workspace,
                            uint64_t ws_bytes, void * stream) {
    const char * who = "llapis_kv_attention";
    const char * bad = check_cache(c);
    if (!bad) bad = check_batch(b, c->page_size);
    AttnPlan a{};
    if (!bad) bad = q ? plan_attention(c, b, q->n_head, a) : "null query";
    if (bad) return refuse_as(who, bad);
    if (!act_type(q->type)) return refuse_as(who, "need F32, F16 or BF16 queries");
    if (q->window < 0 || !(q->scale == q->scale)) return refuse_as(who, "negative window or no scale");
    const KvSeqs sq = seqs_of(b);
    if (sq.n_seq == 0 || sq.n_tokens == 0 || sq.max_new == 0) return 0;
    const int es = el_bytes(q->type), width = q->n_head * c->head_dim;
    if (!q->q || !q->out) return refuse_as(who, "null q or out");
    if (q->q == q->out) return refuse_as(who, "out may not be q: its rows are read by several workgroups");
    if (!aligned16(q->q) || !aligned16(q->out) || (q->q_stride * es) % 16 || (q->out_stride * es) % 16)
        return refuse_as(who, "q and out must be 16-byte aligned, rows too");
    if (sq.n_tokens > 1 && (q->q_stride < width || q->out_stride < width)) return refuse_as(who, "rows shorter than n_head * head_dim");
    if (!workspace || !aligned16(workspace) || ws_bytes < a.bytes()) return refuse_as(who, "workspace too small or not 16-byte aligned");
    KvAttn p{};
    p.b = sq;
    p.k = (const uint8_t *)c->k;
    p.v = (const uint8_t *)c->v;
    p.k_stride = c->k_stride;
    p.v_stride = c->v_stride;
    p.n_pages = c->n_pages;
    p.page_shift = log2_of(c->page_size);
    p.n_kv = c->n_kv;
    p.group = q->n_head / c->n_kv;
    p.window = std::min(q->window, 0x7FFFFF00);            // leaves room for sums with it
    p.unit = kv_unit(c->head_dim);
    p.scale = q->scale;
    p.type = q->type;
    p.q = q->q;
    p.q_stride = q->q_stride;
    p.out = q->out;
    p.out_stride = q->out_stride;
    p.lse = q->lse;
    uint8_t * ws = (uint8_t *)workspace;
    p.base = (int32_t *)ws;
    p.ml = (float *)(ws + a.base_bytes);
    p.acc = (float *)(ws + a.base_bytes + a.ml_bytes);
    p.nt = a.nt;
    p.runs = a.runs;
    p.tiles = a.tiles;
    hipStream_t s = (hipStream_t)stream;
    if (c->type == T_F16) KV_TRY(launch_kv_attn_f16(p, c->head_dim, s));
    else if (c->type == T_BF16) KV_TRY(launch_kv_attn_bf16(p, c->head_dim, s));
    else KV_TRY(launch_kv_attn_q8(p, c->head_dim, s));
    if (!needs_join(c, b)) return 0;                                   // every item is one unit
    // parts of an item, as many as the bounds suggest; workgroups by an item's rows
    const int64_t items = (int64_t)sq.n_seq * c->n_kv;
    const int parts = (int)(a.runs / items), pg = parts < 4 ? 1 : parts < 16 ? 4 : 16, per = 1024 / pg;
    const int rows = std::min(q->n_head / c->n_kv * sq.max_new, 16 * a.nt);
    const dim3 grid((unsigned)(items * a.tiles), (rows * c->head_dim + per - 1) / per), wg(256);
    const float shift = c->type == T_BF16 ? 0.0f : 15.0f;
    if (pg == 1) hipLaunchKernelGGL(k_kv_join<1>, grid, wg, 0, s, p, c->head_dim, shift);
    else if (pg == 4) hipLaunchKernelGGL(k_kv_join<4>, grid, wg, 0, s, p, c->head_dim, shift);
    else hipLaunchKernelGGL(k_kv_join<16>, grid, wg, 0, s, p, c->head_dim, shift);
    KV_TRY(hipGetLastError());
    return 0;
}

int32_t llapis_kv_copy_pages(const llapis_kv_planes * p, const int32_t * pairs, int32_t n_pairs, void * stream) {
    int chunks = 0;
    const char * bad = check_planes(p, chunks);
    if (!bad && n_pairs < 0) bad = "negative n_pairs";
    if (!bad && n_pairs > 0 && !pairs) bad = "null pairs";
    if (bad) return refuse_as("llapis_kv_copy_pages", bad);
    if (n_pairs == 0) return 0;
    const int64_t all = (int64_t)n_pairs * p->n_planes * chunks;
    hipLaunchKernelGGL(k_kv_copy, dim3((unsigned)std::min<int64_t>(all, 1 << 20)), dim3(256), 0, (hipStream_t)stream, *p, pairs,
                       n_pairs, chunks);
    KV_TRY(hipGetLastError());
    return 0;
}

int32_t llapis_kv_fork(const llapis_kv_planes * p, int32_t * page_table, int64_t table_stride, int32_t max_pages,
                       int32_t * lens, int32_t n_seq, const int32_t * forks, int32_t n_forks, void * stream) {
    int chunks = 0;
    const char * bad = check_planes(p, chunks);
    if (!bad) bad = check_table(page_table, table_stride, max_pages, lens, n_seq);
    if (!bad && (n_forks < 0 || n_forks > 65535)) bad = "need 0 <= n_forks <= 65535";
    if (!bad && n_forks > 0 && !forks) bad = "null forks";
    if (bad) return refuse_as("llapis_kv_fork", bad);
    if (n_forks == 0) return 0;
    hipLaunchKernelGGL(k_kv_fork, dim3(p->n_planes * chunks, n_forks), dim3(256), 0, (hipStream_t)stream, *p, page_table,
                       table_stride, max_pages, lens, n_seq, forks, chunks);
    KV_TRY(hipGetLastError());
    return 0;
}

int32_t llapis_kv_page_refs(int32_t n_pages, int32_t page_size, const int32_t * page_table, int64_t table_stride,
                            int32_t max_pages, const int32_t * lens, int32_t n_seq, int32_t * refs, int32_t * free_pages,
                            int32_t * n_free, void * stream) {
    const char * bad = check_rows(page_table, table_stride, max_pages, lens, n_seq);
    if (!bad && (n_pages <= 0 || n_pages > KV_MAX_COUNT || page_size <= 0)) bad = "need 0 < n_pages <= 2^30 and page_size > 0";
    if (!bad && !refs) bad = "null refs";
    if (bad) return refuse_as("llapis_kv_page_refs", bad);
    hipStream_t s = (hipStream_t)stream;
    KV_TRY(launch_refs(page_table, table_stride, max_pages, lens, n_seq, page_size, n_pages, refs, s));
    if (free_pages || n_free) {
        hipLaunchKernelGGL(k_kv_free, dim3(1), dim3(SCAN_WG), 0, s, refs, n_pages, free_pages, n_free);
        KV_TRY(hipGetLastError());
    }
    return 0;
}

uint64_t llapis_kv_compact_workspace_size(int32_t n_pages) { return n_pages > 0 && n_pages <= KV_MAX_COUNT ? ((uint64_t)n_pages * 4 + 1) * 4 : 0; }

int32_t llapis_kv_compact(const llapis_kv_planes * p, const int32_t * page_table, int64_t table_stride, int32_t max_pages,
                          const int32_t * lens, int32_t n_seq, int32_t * table_out, int32_t * refs, int32_t * n_live,
                          void * workspace, uint64_t ws_bytes, void * stream) {
    const char * who = "llapis_kv_compact";
    int chunks = 0;
    const char * bad = check_planes(p, chunks);
    if (!bad) bad = check_rows(page_table, table_stride, max_pages, lens, n_seq);
    if (!bad && ((n_seq > 0 && !table_out) || !n_live)) bad = "null table_out or n_live";
    if (!bad && (!workspace || ((uintptr_t)workspace & 3) || ws_bytes < llapis_kv_compact_workspace_size(p->n_pages)))
        bad = "workspace too small";
    if (bad) return refuse_as(who, bad);
    const int n = p->n_pages;
    int32_t * counts = (int32_t *)workspace, * place = counts + n, * from = place + n, * to = from + n, * n_moves = to + n;
    hipStream_t s = (hipStream_t)stream;
    if (n <= SMALL_PAGES && (int64_t)n_seq * max_pages <= SMALL_ENTRIES) {
        hipLaunchKernelGGL(k_kv_plan_small, dim3(1), dim3(SCAN_WG), 0, s, page_table, table_stride, max_pages, lens, n_seq,
                           p->page_size, n, place, from, to, n_moves, n_live, refs, table_out);
    } else {
        KV_TRY(launch_refs(page_table, table_stride, max_pages, lens, n_seq, p->page_size, n, counts, s));
        hipLaunchKernelGGL(k_kv_plan, dim3(1), dim3(SCAN_WG), 0, s, counts, n, place, from, to, n_moves, n_live, refs);
        KV_TRY(hipGetLastError());
        if (n_seq > 0)
            hipLaunchKernelGGL(k_kv_remap, table_grid(n_seq, max_pages), dim3(256), 0, s, page_table, table_stride, max_pages,
                               lens, p->page_size, n, place, table_out);
    }
    KV_TRY(hipGetLastError());
    // at most half of the pool moves
    const int64_t all = (int64_t)(n / 2) * p->n_planes * chunks;
    if (all > 0)
        hipLaunchKernelGGL(k_kv_move, dim3((unsigned)std::min<int64_t>(all, 256 * 8)), dim3(256), 0, s, *p, from, to, n_moves,
                           chunks);
    KV_TRY(hipGetLastError());
    return 0;
}

}  // extern "C"
