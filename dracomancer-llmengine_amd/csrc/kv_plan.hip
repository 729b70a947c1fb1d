// kv_plan.hip -- pages of a ragged batch: block tables and slot maps built on
// the GPU from the requests' lengths, and pages given back.
//
// need_s = ceil((len_s + q_s) / ps) - ceil(len_s / ps) pages; with first_s the
// exclusive prefix sum of need, the k-th page taken is free_list[n_free - 1 -
// k].  Every block computes the prefix sums of all sequences itself, 1024 at a
// time (one sequence per thread; a few KB that all blocks read from L2), and
// then serves its own part of the tokens and of the block tables, so one
// launch does without a device-wide wait.  What the call may write over its
// own inputs (kv_len_out, n_free_out) is written by the block that finishes
// last, behind every block's reads.
#include <hip/hip_runtime.h>
#include <limits.h>

#include "dev_common.h"
#include "kv4.h"

namespace draco {
namespace {

constexpr int TILE = 1024;  // sequences per pass, threads per block

// Inclusive sums of (a, b) over the block's threads (64 bits: lengths come
// unchecked from device memory).  red: 2 * 16 values of LDS.
struct Sum2 {
    long a, b;
};
__device__ __forceinline__ Sum2 block_scan(Sum2 v, long* red) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int d = 1; d < 64; d <<= 1) {
        const long a = __shfl_up(v.a, d), b = __shfl_up(v.b, d);
        if (lane >= d) {
            v.a += a;
            v.b += b;
        }
    }
    __syncthreads();
    if (lane == 63) {
        red[2 * w] = v.a;
        red[2 * w + 1] = v.b;
    }
    __syncthreads();
    for (int i = 0; i < w; i++) {
        v.a += red[2 * i];
        v.b += red[2 * i + 1];
    }
    return v;
}
__device__ __forceinline__ Sum2 block_total(const long* red) {
    Sum2 t = {0, 0};
    for (int i = 0; i < TILE / 64; i++) {
        t.a += red[2 * i];
        t.b += red[2 * i + 1];
    }
    return t;
}

__device__ __forceinline__ int pages_of(long len, int sh) { return (int)((len + (1 << sh) - 1) >> sh); }

// The last block to arrive (its counter left at 0 again); others return false.
__device__ __forceinline__ bool last_block(int* ticket, int* flag) {
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        const int n = atomicAdd(ticket, 1);
        *flag = n == (int)gridDim.x - 1;
        if (*flag) *ticket = 0;
    }
    __syncthreads();
    return *flag != 0;
}

struct Seq {  // one sequence of a tile
    int old, q, have, need;
    long cu, first;  // exclusive: rows and pages of the sequences before it
    bool ok;
};

// Sequence base + threadIdx.x; row / page: the sums of the tiles before.
__device__ __forceinline__ Seq plan_seq(const KvPlanArgs& a, int base, long& row, long& page, int n_free, long* red) {
    Seq s = {};
    const int i = base + (int)threadIdx.x;
    const long cap = (long)a.max_blocks << a.ps_shift;
    bool fits = false;
    if (i < a.n_seq) {
        s.old = max(a.kv_len[i], 0);
        s.q = max(a.q_len[i], 0);
        s.have = pages_of(s.old, a.ps_shift);
        fits = (long)s.old + s.q <= cap;
        s.need = fits ? pages_of((long)s.old + s.q, a.ps_shift) - s.have : 0;
    }
    const Sum2 in = block_scan({s.q, s.need}, red);
    s.cu = row + in.a - s.q;
    s.first = page + in.b - s.need;
    const Sum2 t = block_total(red);
    row += t.a;
    page += t.b;
    s.ok = fits && s.cu + s.q <= a.n_tok && (s.need == 0 || s.first + s.need <= n_free);
    return s;
}

__device__ __forceinline__ int taken_page(const KvPlanArgs& a, int n_free, long k) {
    const int p = a.free_list[n_free - 1 - k];
    return (unsigned)p < (unsigned)a.n_pages ? p : -1;
}

__global__ __launch_bounds__(TILE) void k_kv_plan(KvPlanArgs a) {
    __shared__ long red[2 * TILE / 64];
    __shared__ int s_cu[TILE + 1], s_old[TILE], s_first[TILE], s_have[TILE], s_need[TILE];
    __shared__ int flag;
    const int tid = threadIdx.x;
    const int n_free = min(max(*a.n_free, 0), a.n_pages);
    const int per = (a.n_tok + (int)gridDim.x - 1) / (int)gridDim.x;  // this block's tokens
    const int t0 = min(a.n_tok, per * (int)blockIdx.x), t1 = min(a.n_tok, t0 + per);
    long row = 0, page = 0;
    for (int base = 0; base < a.n_seq; base += TILE) {
        const Seq s = plan_seq(a, base, row, page, n_free, red);
        const int n = min(TILE, a.n_seq - base);
        s_cu[tid] = (int)min(s.cu, (long)a.n_tok);
        if (tid == n - 1) s_cu[n] = (int)min(s.cu + s.q, (long)a.n_tok);
        s_old[tid] = s.old;
        s_have[tid] = s.have;
        s_need[tid] = s.ok ? s.need : -1;  // -1: refused
        s_first[tid] = (int)min(s.first, (long)INT_MAX);
        __syncthreads();
        if (blockIdx.x == 0 && tid < n) {
            if (base == 0 && tid == 0) a.cu_q[0] = 0;
            a.cu_q[base + tid + 1] = s_cu[tid + 1];
        }
        // block tables: a wave per sequence, its new pages over the lanes
        for (int i = (int)blockIdx.x * (TILE / 64) + (tid >> 6); i < n; i += (int)gridDim.x * (TILE / 64))
            for (int b = tid & 63; b < s_need[i]; b += 64)
                a.block_table[(long)(base + i) * a.max_blocks + s_have[i] + b] = taken_page(a, n_free, (long)s_first[i] + b);
        // this block's tokens that belong to the tile
        for (int t = max(t0, s_cu[0]) + tid; t < min(t1, s_cu[n]); t += TILE) {
            int lo = 0, hi = n;  // the last i with s_cu[i] <= t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_cu[mid] <= t) lo = mid;
                else hi = mid;
            }
            int pos = -1, slot = -1;
            if (s_need[lo] >= 0) {
                pos = s_old[lo] + (t - s_cu[lo]);
                const int b = pos >> a.ps_shift;
                const int p = b < s_have[lo] ? a.block_table[(long)(base + lo) * a.max_blocks + b]
                                             : taken_page(a, n_free, (long)s_first[lo] + b - s_have[lo]);
                if ((unsigned)p < (unsigned)a.n_pages) slot = (p << a.ps_shift) + (pos & ((1 << a.ps_shift) - 1));
            }
            a.slot[t] = slot;
            if (a.pos) a.pos[t] = pos;
        }
        __syncthreads();
    }
    // rows behind the last sequence: no slot
    for (int t = (int)max((long)t0, min(row, (long)a.n_tok)) + tid; t < t1; t += TILE) {
        a.slot[t] = -1;
        if (a.pos) a.pos[t] = -1;
    }
    if (a.n_seq == 0 && blockIdx.x == 0 && tid == 0) a.cu_q[0] = 0;
    // lengths and the list's count, behind every block's reads of them
    if (gridDim.x > 1 && !last_block(a.ticket, &flag)) return;
    row = page = 0;
    long took = 0, refused = 0;
    for (int base = 0; base < a.n_seq; base += TILE) {
        const Seq s = plan_seq(a, base, row, page, n_free, red);
        const bool real = base + tid < a.n_seq;
        __syncthreads();
        const Sum2 in = block_scan({s.ok ? s.need : 0, real && !s.ok}, red);
        (void)in;
        const Sum2 t = block_total(red);
        took += t.a;
        refused += t.b;
        if (real) a.kv_len_out[base + tid] = s.ok ? s.old + s.q : a.kv_len[base + tid];
        __syncthreads();
    }
    if (tid == 0) {
        *a.n_free_out = n_free - (int)took;
        a.status[0] = (int)refused;
        a.status[1] = (int)min(max(row - a.n_tok, 0L), (long)INT_MAX);
    }
}

struct Rel {
    int len, keep, have, want;
    long first;
};
__device__ __forceinline__ Rel release_seq(const KvReleaseArgs& a, int base, long& page, long* red) {
    Rel s = {};
    const int i = base + (int)threadIdx.x;
    if (i < a.n_seq) {
        const long cap = (long)a.max_blocks << a.ps_shift;
        s.len = (int)min((long)max(a.kv_len[i], 0), cap);
        s.keep = min(max(a.keep[i], 0), s.len);
        s.have = pages_of(s.len, a.ps_shift);
        s.want = pages_of(s.keep, a.ps_shift);
    }
    const Sum2 in = block_scan({s.have - s.want, 0}, red);
    s.first = page + in.a - (s.have - s.want);
    page += block_total(red).a;
    return s;
}

// The released pages' ordinals run over sequences and blocks as a plan's do;
// page k of n goes to free_list[n_free + n - 1 - k], so that a release of what
// a plan took restores the list.
__global__ __launch_bounds__(TILE) void k_kv_release(KvReleaseArgs a) {
    __shared__ long red[2 * TILE / 64];
    __shared__ int s_want[TILE], s_go[TILE];
    __shared__ long s_first[TILE];
    __shared__ int flag;
    const int tid = threadIdx.x;
    const long n_free = min(max(*a.n_free, 0), a.n_pages);
    long all = 0, page = 0;
    for (int base = 0; base < a.n_seq; base += TILE) {
        release_seq(a, base, all, red);
        __syncthreads();
    }
    for (int base = 0; base < a.n_seq; base += TILE) {
        const Rel s = release_seq(a, base, page, red);
        const int n = min(TILE, a.n_seq - base);
        s_want[tid] = s.want;
        s_go[tid] = s.have - s.want;
        s_first[tid] = s.first;
        __syncthreads();
        for (int i = (int)blockIdx.x * (TILE / 64) + (tid >> 6); i < n; i += (int)gridDim.x * (TILE / 64))
            for (int b = tid & 63; b < s_go[i]; b += 64) {
                const long e = (long)(base + i) * a.max_blocks + s_want[i] + b;
                const long at = n_free + all - 1 - (s_first[i] + b);
                const int p = a.block_table[e];
                a.block_table_out[e] = -1;
                if (at < a.n_pages) a.free_list[at] = p;
            }
        __syncthreads();
    }
    if (gridDim.x > 1 && !last_block(a.ticket, &flag)) return;
    for (int base = 0; base < a.n_seq; base += TILE) {
        page = 0;
        const Rel s = release_seq(a, base, page, red);
        if (base + tid < a.n_seq) a.kv_len_out[base + tid] = s.keep;
        __syncthreads();
    }
    if (tid == 0) *a.n_free_out = (int)min(n_free + all, (long)a.n_pages);
}

}  // namespace

int kv_plan(const KvPlanArgs& a, hipStream_t st) {
    // one block serves a small batch without the wait for the last block
    const int by_tok = (a.n_tok + 2047) / 2048, by_seq = (a.n_seq + 127) / 128;
    const int grid = min(128, max(1, max(by_tok, by_seq)));
    hipLaunchKernelGGL(k_kv_plan, dim3(grid), dim3(TILE), 0, st, a);
    return 0;
}

int kv_release(const KvReleaseArgs& a, hipStream_t st) {
    const int grid = min(128, max(1, (a.n_seq + 31) / 32));
    hipLaunchKernelGGL(k_kv_release, dim3(grid), dim3(TILE), 0, st, a);
    return 0;
}

}  // namespace draco
