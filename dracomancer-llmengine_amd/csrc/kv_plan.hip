// kv_plan.hip -- pages of a ragged batch: block tables and slot maps built on
// the GPU from the requests' lengths, and pages given back.
//
// need_s = ceil((len_s + q_s) / ps) - ceil(len_s / ps) pages; with first_s the
// exclusive prefix sum of need, the k-th page taken is free_list[n_free - 1 -
// k].  Every block computes the prefix sums of all sequences itself, a tile at
// a time (one sequence per thread; a few KB that all blocks read from L2), and
// then serves its own part of the tokens and of the block tables, so one
// launch does without a device-wide wait.  What the call may write over its
// own inputs (kv_len_out, n_free_out) is written by the block that finishes
// last, behind every block's reads.
//
// Latency bound (a few KB): 8 sequences 4.2 us, 512 of up to 30000 tokens with
// 39629 rows 6.9, a release of 300 6.7, of which about 2 are any launch's (and 2
// are for entries that may be no pages: the counter waits for the table's
// entries, and the list's stores pass the L2s).
#include <hip/hip_runtime.h>
#include <limits.h>

#include "dev_common.h"
#include "kv4.h"
#include "wave_scan.h"

namespace draco {
namespace {

// Inclusive sums of (a, b) over the block's THREADS threads and their totals
// (64 bits: lengths come unchecked from device memory).  red: 2 * 16 longs of
// LDS; every wave adds up the waves before it in its own lanes.
struct Sum2 {
    long a, b;
};
template <int THREADS>
__device__ __forceinline__ Sum2 block_scan(Sum2 v, Sum2& total, long* red) {
    constexpr int W = THREADS / 64;
    const int lane = threadIdx.x & 63, w = uni((int)threadIdx.x >> 6);
    v = {wave_scan(v.a), wave_scan(v.b)};
    if constexpr (W == 1) {
        total = {lane_of(v.a, 63), lane_of(v.b, 63)};
        return v;
    }
    __syncthreads();
    if (lane == 63) {
        red[w] = v.a;
        red[16 + w] = v.b;
    }
    __syncthreads();
    const long a = wave_scan(lane < W ? red[lane] : 0L), b = wave_scan(lane < W ? red[16 + lane] : 0L);
    total = {lane_of(a, W - 1), lane_of(b, W - 1)};
    if (w) v = {v.a + lane_of(a, w - 1), v.b + lane_of(b, w - 1)};
    return v;
}

__device__ __forceinline__ int pages_of(long len, int sh) { return (int)((len + (1 << sh) - 1) >> sh); }

// The blocks that arrived with a mark, in the last one to arrive (its counter
// left at 0 again); -1 in the others.  A block's reads are done when it arrives,
// and its writes where it has waited for them.
__device__ __forceinline__ int last_block(int* ticket, bool mark, int* flag) {
    __syncthreads();
    if (threadIdx.x == 0) {
        const int add = mark ? 0x10001 : 1;  // (a grid has fewer than 2^15 blocks)
        const int n = add + __hip_atomic_fetch_add(ticket, add, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const bool last = (n & 0xFFFF) == (int)gridDim.x;
        *flag = last ? n >> 16 : -1;
        if (last) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    return *flag;
}

struct Seq {  // one sequence of a tile
    int old, q, have, need;
    long cu, first;  // exclusive: rows and pages of the sequences before it
    bool ok;
};

// Sequence base + threadIdx.x; row / page: the sums of the tiles before.
template <int TILE>
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
    Sum2 all;
    const Sum2 in = block_scan<TILE>({s.q, s.need}, all, red);
    s.cu = row + in.a - s.q;
    s.first = page + in.b - s.need;
    row += all.a;
    page += all.b;
    s.ok = fits && s.cu + s.q <= a.n_tok && (s.need == 0 || s.first + s.need <= n_free);
    return s;
}

__device__ __forceinline__ int taken_page(const KvPlanArgs& a, int n_free, long k) {
    const int p = a.free_list[n_free - 1 - k];
    return (unsigned)p < (unsigned)a.n_pages ? p : -1;
}

template <int TILE>
__global__ __launch_bounds__(TILE) void k_kv_plan(KvPlanArgs a) {
    __shared__ long red[32];
    __shared__ int s_cu[TILE + 1], s_old[TILE], s_first[TILE], s_have[TILE], s_need[TILE];
    __shared__ int flag;
    const int tid = threadIdx.x;
    const int n_free = min(max(*a.n_free, 0), a.n_pages);
    const int per = (a.n_tok + (int)gridDim.x - 1) / (int)gridDim.x;  // this block's tokens
    const int t0 = min((long)a.n_tok, (long)per * blockIdx.x), t1 = min(a.n_tok, t0 + per);
    long row = 0, page = 0;
    Seq s = {};
    for (int base = 0; base < a.n_seq; base += TILE) {
        s = plan_seq<TILE>(a, base, row, page, n_free, red);
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
        // block tables: a wave per sequence, its new pages over the lanes
        for (int i = (int)blockIdx.x * (TILE / 64) + (tid >> 6); i < n; i += (int)gridDim.x * (TILE / 64))
            for (int b = tid & 63; b < s_need[i]; b += 64)
                a.block_table[(long)(base + i) * a.max_blocks + s_have[i] + b] = taken_page(a, n_free, (long)s_first[i] + b);
        if (base + TILE < a.n_seq) __syncthreads();
    }
    // rows behind the last sequence: no slot
    for (int t = (int)max((long)t0, min(row, (long)a.n_tok)) + tid; t < t1; t += TILE) {
        a.slot[t] = -1;
        if (a.pos) a.pos[t] = -1;
    }
    if (a.n_seq == 0 && blockIdx.x == 0 && tid == 0) a.cu_q[0] = 0;
    // lengths and the list's count, behind every block's reads of them
    if (gridDim.x > 1 && last_block(a.ticket, false, &flag) < 0) return;
    const long rows = row;
    long took = 0, refused = 0;
    row = page = 0;
    for (int base = 0; base < a.n_seq; base += TILE) {
        if (a.n_seq > TILE) s = plan_seq<TILE>(a, base, row, page, n_free, red);  // (else the tile's are still here)
        const bool real = base + tid < a.n_seq;
        Sum2 all;
        block_scan<TILE>({s.ok ? s.need : 0, real && !s.ok}, all, red);
        took += all.a;
        refused += all.b;
        if (real) a.kv_len_out[base + tid] = s.ok ? s.old + s.q : a.kv_len[base + tid];
    }
    if (tid == 0) {
        *a.n_free_out = n_free - (int)took;
        a.status[0] = (int)refused;
        a.status[1] = (int)min(max(rows - a.n_tok, 0L), (long)INT_MAX);
    }
}

struct Rel {
    int len, keep, have, want;
    long first;
};
template <int TILE>
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
    Sum2 all;
    const Sum2 in = block_scan<TILE>({s.have - s.want, 0}, all, red);
    s.first = page + in.a - (s.have - s.want);
    page += all.a;
    return s;
}

// The released pages' ordinals run over sequences and blocks as a plan's do;
// page k of n goes to free_list[n_free + n - 1 - k], so that a release of what
// a plan took restores the list.  An entry that is no page of the pool (one
// behind a window, whose page the caller took back) leaves no gap: every block
// places its entries as if all were pages, past the L2s, and the last one closes
// the list up where a block met others.
template <int TILE>
__global__ __launch_bounds__(TILE) void k_kv_release(KvReleaseArgs a) {
    __shared__ long red[32];
    __shared__ int s_want[TILE], s_go[TILE];
    __shared__ long s_first[TILE];
    __shared__ int flag;
    const int tid = threadIdx.x;
    const long n_free = min(max(*a.n_free, 0), a.n_pages);
    long all = 0, page = 0;
    Rel s = {};
    for (int base = 0; base < a.n_seq; base += TILE) s = release_seq<TILE>(a, base, all, red);
    bool bad = false;
    for (int base = 0; base < a.n_seq; base += TILE) {
        if (a.n_seq > TILE) s = release_seq<TILE>(a, base, page, red);  // (else the tile's are still here)
        const int n = min(TILE, a.n_seq - base);
        s_want[tid] = s.want;
        s_go[tid] = s.have - s.want;
        s_first[tid] = s.first;
        __syncthreads();
        for (int i = (int)blockIdx.x * (TILE / 64) + (tid >> 6); i < n; i += (int)gridDim.x * (TILE / 64))
            for (int b = tid & 63; b < s_go[i]; b += 64) {
                const long e = (long)(base + i) * a.max_blocks + s_want[i] + b;
                const long at = n_free + all - 1 - (s_first[i] + b);
                if (at >= a.n_pages) continue;  // (not all of them are pages)
                const int p = a.block_table[e];
                bad |= (unsigned)p >= (unsigned)a.n_pages;
                a.block_table_out[e] = -1;
                __hip_atomic_store(a.free_list + at, p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        if (base + TILE < a.n_seq) __syncthreads();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last block may read what was stored
    int marks = __syncthreads_or(bad);
    if (gridDim.x > 1) marks = last_block(a.ticket, marks != 0, &flag);
    if (marks < 0) return;
    const long end = min(n_free + all, (long)a.n_pages);
    long count = end;
    if (marks || n_free + all > end) {
        // what was placed, closed up in its order
        count = n_free;
        for (long base = n_free; base < end; base += TILE) {
            const long i = base + tid;
            const int p = i < end ? __hip_atomic_load(a.free_list + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : -1;
            const bool ok = (unsigned)p < (unsigned)a.n_pages;
            Sum2 sum;  // (its barriers lie between the tile's loads and stores)
            const Sum2 in = block_scan<TILE>({ok, 0}, sum, red);
            if (ok) a.free_list[count + in.a - 1] = p;
            count += sum.a;
        }
        // the first ordinals, for which there was no room: counted, then placed behind the others
        const long rest = n_free + all - end;
        long left = 0;
        for (int pass = 0; pass < 2; pass++) {
            long seen = 0;
            page = 0;
            for (int base = 0; base < a.n_seq && page < rest; base += TILE) {
                const long first = page;
                s = release_seq<TILE>(a, base, page, red);
                const int n = min(TILE, a.n_seq - base);
                __syncthreads();
                s_want[tid] = s.want;
                s_first[tid] = s.first;
                __syncthreads();
                for (long k0 = first; k0 < min(page, rest); k0 += TILE) {
                    const long k = k0 + tid;
                    int p = -1;
                    long e = 0;
                    const bool mine = k < min(page, rest);
                    if (mine) {
                        int lo = 0, hi = n;  // the last sequence that starts at or before k
                        while (hi - lo > 1) {
                            const int mid = (lo + hi) >> 1;
                            if (s_first[mid] <= k) lo = mid;
                            else hi = mid;
                        }
                        e = (long)(base + lo) * a.max_blocks + s_want[lo] + (k - s_first[lo]);
                        p = a.block_table[e];
                    }
                    const bool ok = (unsigned)p < (unsigned)a.n_pages;
                    Sum2 sum;
                    const Sum2 in = block_scan<TILE>({ok, 0}, sum, red);
                    if (pass && mine) {
                        const long at = count + left - (seen + in.a);
                        if (ok && at < a.n_pages) a.free_list[at] = p;
                        a.block_table_out[e] = -1;
                    }
                    seen += sum.a;
                }
            }
            left = seen;
        }
        count = min(count + left, (long)a.n_pages);
    }
    for (int base = 0; base < a.n_seq; base += TILE) {
        if (a.n_seq > TILE) s = release_seq<TILE>(a, base, page, red);
        if (base + tid < a.n_seq) a.kv_len_out[base + tid] = s.keep;
    }
    if (tid == 0) *a.n_free_out = (int)count;
}

}  // namespace

// One tile of sequences needs one pass of loads and sums, so the tile (and the
// block) is as large as the batch; tokens and block tables are spread over more
// blocks only where they outweigh the sums that every block repeats.
int kv_plan(const KvPlanArgs& a, hipStream_t st) {
    const int tile = a.n_seq <= 256 ? 256 : 1024;
    const int by_tok = (a.n_tok + tile - 1) / tile, by_seq = (a.n_seq + 127) / 128;
    const dim3 grid(min(256, max(1, max(by_tok, by_seq))));
    if (tile == 256) hipLaunchKernelGGL(k_kv_plan<256>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_kv_plan<1024>, grid, dim3(1024), 0, st, a);
    return 0;
}

int kv_release(const KvReleaseArgs& a, hipStream_t st) {
    const int tile = a.n_seq <= 256 ? 256 : 1024;
    const dim3 grid(min(128, max(1, (a.n_seq + 15) / 16)));
    if (tile == 256) hipLaunchKernelGGL(k_kv_release<256>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_kv_release<1024>, grid, dim3(1024), 0, st, a);
    return 0;
}

}  // namespace draco
