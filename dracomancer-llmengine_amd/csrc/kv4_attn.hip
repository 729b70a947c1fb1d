// kv4_attn.hip -- causal attention of a ragged batch over the 4-bit pages
// (kv4.h), with a sliding window and sink tokens.
//
// o_r = sum_j p_rj v_j / sum_j p_rj, p = exp(scale q_r . k_j) over j <= pos_r
// and (j > pos_r - window or j < sink); 0 where no j is left.
//
// Rows of one KV head's group are packed (row = query * group + head), 16 to a
// matrix instruction.  S^T = K Q^T and O^T = V^T P^T: with keys (dims) in the
// instruction's rows and query rows in its columns, a lane keeps one query
// row's scores, so the softmax is lane-local but for two cross-row exchanges,
// and the scores leave the first product in the order in which the second
// takes them (16 consecutive keys a lane group; the contraction's order is
// free as long as both operands share it).
//
// K and V values are exact in f16 (kv4.h).  p is split into two f16 terms, 22
// bits, and so is q of fp32 rows: their products run twice into one fp32 sum.  q
// of f16 rows is exact.  A row of fp32 q is scaled by a power of two so that its
// largest value lies just below f16's range: the second term ends at 2^-24, which
// leaves 22 bits to every value down to 2^-17 of the largest.
#include <float.h>
#include <hip/hip_runtime.h>

#include <type_traits>

#include "dev_common.h"
#include "kv4.h"
#include "wave_scan.h"

namespace draco {
namespace {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef unsigned int u4v __attribute__((ext_vector_type(4)));
typedef unsigned int u2v __attribute__((ext_vector_type(2)));

constexpr int UNIT = 64;       // keys per step of a wave: four 16-row operand tiles
constexpr float PBIAS = 6.0f;  // p is held times 2^6 ..
constexpr float PSLACK = 8.0f; // .. and its maximum may lag by 2^8 (2^14 < the largest f16)

__device__ __forceinline__ f4v mfma(h8v a, h8v b, f4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The two values of byte B of w.
template <int B>
__device__ __forceinline__ h2v fp4x2(uint32_t w) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, B);
}

// Eight consecutive dims of a K row times the block's scale.
__device__ __forceinline__ h8v k_operand(uint32_t w, h2v s) {
    const h2v a = fp4x2<0>(w) * s, b = fp4x2<1>(w) * s, c = fp4x2<2>(w) * s, d = fp4x2<3>(w) * s;
    return h8v{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

__device__ __forceinline__ h2v as_h2(uint32_t u) { return __builtin_bit_cast(h2v, u); }
__device__ __forceinline__ uint32_t as_u(h2v h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ h8v as_h8(u4v u) { return __builtin_bit_cast(h8v, u); }

// a and b to f16, and to f16 what that leaves of them: one conversion for both
// (v_cvt_pk_f16_f32) and one instruction each (v_fma_mixlo_f16, v_fma_mixhi_f16).
// (Both need values that the compiler knows nothing of: it would turn a product
// with -1 into a conversion, a subtraction and another conversion, and convert a
// and b once more.)
struct Two {
    uint32_t hi, lo;
};
__device__ __forceinline__ Two split2(float a, float b) {
    typedef float f2v __attribute__((ext_vector_type(2)));
    uint32_t u = as_u(__builtin_convertvector((f2v{a, b}), h2v));
    float minus = -1.0f;
    asm("" : "+v"(u));
    asm("" : "+s"(minus));
    const h2v h = as_h2(u);
    return {u, as_u(h2v{(_Float16)__builtin_fmaf((float)h.x, minus, a), (_Float16)__builtin_fmaf((float)h.y, minus, b)})};
}
// Eight fp32 values as two f16 operands.
__device__ __forceinline__ void split8(const float x[8], h8v& hi, h8v& lo) {
    u4v h, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const Two t = split2(x[2 * i], x[2 * i + 1]);
        h[i] = t.hi, l[i] = t.lo;
    }
    hi = __builtin_bit_cast(h8v, h);
    lo = __builtin_bit_cast(h8v, l);
}

// Rows [r0, r1) of one sequence and KV head.
struct Tile {
    int seq, q0, rows, len, r0, r1, head;  // rows: of the whole sequence; head: the KV head
    bool bad;                              // the length passes the table: NaN
    long pos0;                             // position of the sequence's first query
    const int* table;
};

// The KV rows that the tile's queries can see, as units of 64: first the sink
// units [0, n_sink), then [u0, u0 + n - n_sink).
struct Units {
    int n_sink, u0, n;
    __device__ __forceinline__ int at(int i) const { return i < n_sink ? i : u0 + (i - n_sink); }
};
__device__ __forceinline__ Units units_of(long first_pos, long last_pos, int window, int sink) {
    Units u = {0, 0, 0};
    if (last_pos < 0) return u;
    const long lo = window > 0 ? max(0L, first_pos - window + 1) : 0;
    u.u0 = (int)(lo / UNIT);
    u.n_sink = lo > 0 ? min((int)((min((long)sink, lo) + UNIT - 1) / UNIT), u.u0) : 0;
    u.n = u.n_sink + (int)(last_pos / UNIT) + 1 - u.u0;
    return u;
}

// 64 sequences' rows and lengths, one a lane.
struct Batch {
    int base, q0, q1, len;
};
__device__ __forceinline__ void batch_of(const Kv4AttnArgs& a, int base, Batch& b) {
    const int s = min(base + ((int)threadIdx.x & 63), a.n_seq - 1);
    b.base = base;
    b.q0 = a.cu_q[s];
    b.q1 = a.cu_q[s + 1];
    b.len = a.kv_len[s];
}
__device__ __forceinline__ void tile_of(const Kv4AttnArgs& a, int q0, int q1, int len, Tile& t) {
    t.q0 = min(max(q0, 0), a.n_tok);
    const int qn = min(max(q1, t.q0), a.n_tok) - t.q0;
    t.rows = qn * a.group;
    t.bad = len > (long)a.max_blocks << a.c.ps_shift;
    t.len = t.bad ? 0 : max(len, 0);
    t.pos0 = (long)t.len - qn;
}
__device__ __forceinline__ void seq_of(const Kv4AttnArgs& a, Batch& b, int seq, Tile& t) {
    if (seq >= b.base + 64) batch_of(a, seq, b);
    const int l = seq - b.base;
    tile_of(a, __builtin_amdgcn_readlane(b.q0, l), __builtin_amdgcn_readlane(b.q1, l), __builtin_amdgcn_readlane(b.len, l), t);
    t.seq = seq;
    t.table = a.block_table + (long)seq * a.max_blocks;
}
__device__ __forceinline__ Units tile_units(const Kv4AttnArgs& a, const Tile& t, int r0, int r1) {
    return units_of(t.pos0 + r0 / a.group, t.pos0 + (r1 - 1) / a.group, a.window, a.sink);
}

// The batch's work, laid out as one list of units: sequences, their tiles of R
// rows, KV heads, units of keys.  A sequence's tiles all count as many units as
// any of them may have, at least one (a tile's place is then a division away;
// what is too much comes out as empty pieces).  The grid's blocks take equal
// stretches of the list, whatever the lengths are: `chunk` units from `at`.
// Lengths come from device memory, so every wave adds them up itself, 64
// sequences at a time.
struct Work {
    long at;      // this block's next unit
    int left;     // units left to it
    int chunk;
    long rem;     // `at` within sequence `seq`
    int seq;
};
// Units that a tile of the sequence has at most.
template <int R>
__device__ __forceinline__ int tile_bound(const Kv4AttnArgs& a, const Tile& t) {
    const long last = (long)t.len - 1;  // (the last row's position, behind no key)
    long n = last < 0 || t.rows == 0 ? 0 : last / UNIT + 1;
    if (a.window > 0) {
        const long span = (long)a.window + (R + a.group - 2) / a.group;  // keys under the windows of R rows
        n = min(n, (span + UNIT - 2) / UNIT + 1 + ((long)a.sink + UNIT - 1) / UNIT);
    }
    return (int)max(n, 1L);
}
template <int R>
__device__ __forceinline__ long batch_units(const Kv4AttnArgs& a, const Batch& b) {  // of this lane's sequence
    if (b.base + ((int)threadIdx.x & 63) >= a.n_seq) return 0;
    Tile t;
    tile_of(a, b.q0, b.q1, b.len, t);
    return (long)((t.rows + R - 1) / R) * tile_bound<R>(a, t) * a.c.n_kv;
}
template <int R>
__device__ __forceinline__ bool work_of(const Kv4AttnArgs& a, Work& w, Batch& b, int block, int blocks) {
    batch_of(a, 0, b);
    long mine = wave_scan(batch_units<R>(a, b)), total = lane_of(mine, 63);
    for (int s = 64; s < a.n_seq; s += 64) {
        batch_of(a, s, b);
        total += lane_of(wave_scan(batch_units<R>(a, b)), 63);
    }
    w.chunk = max(a.chunk, (int)((total + blocks - 1) / blocks));
    w.at = (long)block * w.chunk;
    w.left = (int)min((long)w.chunk, total - w.at);
    if (w.left <= 0) return false;
    long before = 0;
    for (int s = 0; s < a.n_seq; s += 64) {
        if (a.n_seq > 64) {
            batch_of(a, s, b);
            mine = wave_scan(batch_units<R>(a, b));
        }
        const unsigned long long past = __ballot(before + mine > w.at);
        if (past) {
            const int l = uni(__ffsll((long long)past) - 1);
            w.seq = s + l;
            w.rem = w.at - before - (l ? lane_of(mine, l - 1) : 0L);
            return true;
        }
        before += lane_of(mine, 63);
    }
    return false;  // (the lengths were written during the call)
}

// One tile a block, whole (prompts: enough of them, and partial rows of many
// queries cost more than they balance).  A sequence's tiles start at v(s) =
// floor(cu_q[s] * group / R) + s, which leaves it at least ceil(rows / R) of
// them; the wave looks for the last s with v(s) <= id, 64 at a time.  The last
// rows (the most keys) come first.
template <int R>
__device__ __forceinline__ bool whole_tile(const Kv4AttnArgs& a, Tile& t) {
    const int lane = threadIdx.x & 63;
    t.head = blockIdx.x % a.c.n_kv;  // neighbours on other XCDs: a head's tiles share few L2s
    const int id = blockIdx.x / a.c.n_kv;
    auto start = [&](int s) { return (int)((long)min(max(a.cu_q[s], 0), a.n_tok) * a.group / R) + s; };
    int seq = 0;
    for (int stride = a.n_seq; stride > 1;) {
        const int end = min(seq + stride, a.n_seq);
        stride = (stride + 63) / 64;
        const int s = seq + lane * stride;
        const bool in = s < end && start(s) <= id;
        seq += max((int)__popcll(__ballot(in)) - 1, 0) * stride;
    }
    t.seq = seq = uni(seq);
    t.table = a.block_table + (long)seq * a.max_blocks;
    tile_of(a, a.cu_q[seq], a.cu_q[seq + 1], a.kv_len[seq], t);
    const int n = (t.rows + R - 1) / R, k = n - 1 - (id - start(seq));
    if (k < 0 || k >= n) return false;
    t.r0 = k * R;
    t.r1 = min(t.r0 + R, t.rows);
    return true;
}

// The next piece of a block's work: units [lo, hi) of u for a tile.
struct Piece {
    int lo, hi;
    long first;  // the tile's first unit in the list
    int n;       // its units there
};
template <int R>
__device__ __forceinline__ void piece_of(const Kv4AttnArgs& a, Work& w, Batch& b, Tile& t, Units& u, Piece& p) {
    for (;; w.seq++) {
        if (w.seq >= a.n_seq) {  // lengths that are written during the call: a NaN row, and an end
            t.q0 = min(t.q0, a.n_tok - 1);
            t.bad = true;
            t.head = t.r0 = 0;
            t.r1 = 1;
            u = {0, 0, 0};
            p = {0, 0, w.at, 1};
            w.left = 0;
            return;
        }
        seq_of(a, b, w.seq, t);
        p.n = uni(tile_bound<R>(a, t));
        const long tile = (long)p.n * a.c.n_kv, all = (t.rows + R - 1) / R * tile;
        if (w.rem >= all) {  // (its rows are done; `left` says that more follow)
            w.rem -= all;
            continue;
        }
        long rem = w.rem;
        const int k = rem < tile ? 0 : (int)((unsigned long)rem / (unsigned long)tile);
        rem -= k * tile;
        for (t.head = 0; rem >= p.n; t.head++) rem -= p.n;
        t.r0 = k * R;
        t.r1 = min(t.r0 + R, t.rows);
        u = tile_units(a, t, t.r0, t.r1);
        p.lo = (int)rem;
        p.hi = min(p.lo + w.left, p.n);
        p.first = w.at - p.lo;
        const int took = p.hi - p.lo;
        w.at += took;
        w.rem += took;
        w.left -= took;
        p.lo = min(p.lo, u.n);
        p.hi = min(p.hi, u.n);
        return;
    }
}

// The table's page that holds `key` (an entry past the table, which only keys
// behind the last one have, is not read: `page_ptr` refuses it).  The loads of
// a unit are issued a turn before their use: nothing here may look at what
// they bring, or the wave would wait for it at once.
__device__ __forceinline__ int page_of(const Kv4AttnArgs& a, const int* table, int key) {
    return table[min(key >> a.c.ps_shift, a.max_blocks - 1)];
}
// The page's part of a head; a page outside the pool gives any readable one and ok = false.
__device__ __forceinline__ const uint8_t* page_ptr(const Kv4AttnArgs& a, int page, int key, int head, bool& ok) {
    ok = (unsigned)page < (unsigned)a.c.n_pages && key >> a.c.ps_shift < a.max_blocks;
    return a.c.data + (unsigned long)(ok ? (unsigned)page : 0u) * a.c.page_bytes + (unsigned long)(unsigned)head * (unsigned)a.c.head_bytes;
}

// Lane (i = lane & 15, g = lane >> 4) of operand tile t holds dims of key
// 16 (i / 4) + 4 t + i % 4: tile t's result rows are then keys 16 g' + 4 t + r
// for lane group g', so that a lane group ends with 16 consecutive keys.
__device__ __forceinline__ int k_key(int unit) {
    const int i = threadIdx.x & 15;
    return unit * UNIT + 16 * (i >> 2) + (i & 3);
}
__device__ __forceinline__ int v_key(int unit) { return unit * UNIT + 16 * ((threadIdx.x & 63) >> 4); }

// N words of 8 codes of one K row and their block scales.  Word s of a row (s =
// 0 .. HD / 32 - 1 in a lane) holds dims HD == 64: 16 g + 8 s; else
// 128 (s / 4) + 32 g + 8 (s % 4).
template <int HD, int N>
struct KRow {
    uint32_t w[N];
    uint16_t s[N > 4 ? 2 : 1];
    bool ok;
    // Scale of word j for both halves; NaN for a page that is none.
    __device__ __forceinline__ h2v scale(int j) const {
        const uint32_t x = ok ? s[N > 4 ? j >> 2 : 0] : 0x7E00u;
        return as_h2(x | x << 16);
    }
};
template <int HD, int N>
__device__ __forceinline__ void load_krow(const uint8_t* p, bool ok, int ps, int off, int s0, KRow<HD, N>& k) {
    const int g = (threadIdx.x & 63) >> 4;
    const uint8_t* sc = p + ps * HD;
    const uint8_t* row = p + off * (HD / 2) + (HD == 64 ? g * 8 + s0 * 4 : (s0 >> 2) * 64 + g * 16 + (s0 & 3) * 4);
    if constexpr (N >= 4) {
#pragma unroll
        for (int c = 0; c < N / 4; c++) {
            const u4v v = *gptr<u4v>(row + c * 64);
            k.w[4 * c] = v.x, k.w[4 * c + 1] = v.y, k.w[4 * c + 2] = v.z, k.w[4 * c + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const u2v v = *gptr<u2v>(row);
        k.w[0] = v.x, k.w[1] = v.y;
    } else {
        k.w[0] = *gptr<uint32_t>(row);
    }
#pragma unroll
    for (int c = 0; c < (N > 4 ? 2 : 1); c++) {
        const int blk = HD == 64 ? g >> 1 : ((s0 >> 2) + c) * 4 + g;
        k.s[c] = *gptr<uint16_t>(sc + (off * (HD / 32) + blk) * 2);
    }
    k.ok = ok;
}

// Eight tokens (half x of the lane group's 16) of dims 32 b + i and 32 b + 16 + i.
struct VPart {
    u2v w;
    u4v s;
};
template <int HD>
__device__ __forceinline__ void load_vpart(const uint8_t* p, int ps, int off, int b, int x, VPart& v) {
    const int i = threadIdx.x & 15, grp = off >> 4;
    v.w = *gptr<u2v>(p + ps * (HD / 2) + grp * (HD * 8) + (b * 16 + i) * 16 + x * 8);
    v.s = *gptr<u4v>(p + ps * HD + ps * (HD / 16) + grp * HD + b * 32 + x * 16);
}
// The part's values: the operand of the low nibbles' dim and of the high ones'.
__device__ __forceinline__ void v_operands(const VPart& v, h8v& lo, h8v& hi) {
    const uint32_t w0 = v.w.x, w1 = v.w.y;
    uint32_t l[4], h[4];
    const h2v c[8] = {fp4x2<0>(w0), fp4x2<1>(w0), fp4x2<2>(w0), fp4x2<3>(w0),
                      fp4x2<0>(w1), fp4x2<1>(w1), fp4x2<2>(w1), fp4x2<3>(w1)};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        l[i] = as_u(as_h2(__builtin_amdgcn_perm(as_u(c[2 * i + 1]), as_u(c[2 * i]), 0x05040100)) * as_h2(v.s[i]));
        h[i] = as_u(as_h2(__builtin_amdgcn_perm(as_u(c[2 * i + 1]), as_u(c[2 * i]), 0x07060302)) * as_h2(v.s[i]));
    }
    lo = __builtin_bit_cast(h8v, u4v{l[0], l[1], l[2], l[3]});
    hi = __builtin_bit_cast(h8v, u4v{h[0], h[1], h[2], h[3]});
}

// Rows behind the last token hold anything, NaN scales too: p = 0 would not
// hide them.  (A row that is in the cache has finite V scales.)  key: the
// part's first; n: keys that are there.
__device__ __forceinline__ void cut_vpart(VPart& v, int key, int len) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        uint32_t s = v.s[e];
        if (key + 2 * e >= len) s = 0;
        else if (key + 2 * e + 1 >= len) s &= 0xFFFFu;
        v.s[e] = s;
    }
}

// q rows of one 16-row tile as operands, fp32 ones times 2^(QTOP - e) with 2^e
// the power of two at or below the largest; f: the softmax scale less that, so
// that f times a score of the operands is the exponent of 2.  Lane (i, g): row i,
// dims in the order of load_k's words.
constexpr int QTOP = 14;  // f16 ends below 2^16; the fp32 sums reach 2^(15 + 16 + 8)
template <int HD, bool F16>
__device__ __forceinline__ void load_q(const Kv4AttnArgs& a, const Tile& t, int r, h8v* hi, h8v* lo, float& f) {
    constexpr int KS = HD / 32;
    const int g = (threadIdx.x & 63) >> 4;
    const long at = (long)(t.q0 + r / a.group) * a.q_stride + (long)(t.head * a.group + r % a.group) * HD;
    float x[KS][8];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int d = HD == 64 ? g * 16 + s * 8 : (s >> 2) * 128 + g * 32 + (s & 3) * 8;
        if constexpr (F16) {
            hi[s] = *(const h8v*)((const _Float16*)a.q + at + d);
        } else {
            const float4 u = ld4((const float*)a.q + at + d), v = ld4((const float*)a.q + at + d + 4);
            x[s][0] = u.x, x[s][1] = u.y, x[s][2] = u.z, x[s][3] = u.w;
            x[s][4] = v.x, x[s][5] = v.y, x[s][6] = v.z, x[s][7] = v.w;
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[s][e]));
        }
    }
    if constexpr (F16) {
        f = a.scale_log2;
    } else {
        top = rows_reduce(top, OpMax{});  // the row's other dims: the three other lane groups
        const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, QTOP - 100), 126);
        const float up = __uint_as_float((unsigned)(127 + QTOP - e) << 23);
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[s][j] *= up;
            split8(x[s], hi[s], lo[s]);
        }
        f = a.scale_log2 * __uint_as_float((unsigned)(127 + e - QTOP) << 23);
    }
}

// Softmax state of a lane's query row.
struct Row {
    int pos, lo;    // keys j <= pos, and j >= lo or j < sink
    float f;        // raw score -> exponent of 2
    float m;        // reference score
    float l;        // this lane group's part of the sum
};

__device__ __forceinline__ void row_init(const Kv4AttnArgs& a, const Tile& t, int r, float f, Row& w) {
    const long pos = t.pos0 + r / a.group;
    w.pos = (int)max(pos, -1L);
    w.lo = a.window > 0 ? (int)max(0L, pos - a.window + 1) : 0;
    w.f = f;
    w.m = -FLT_MAX;  // (finite: a masked score less it is -inf)
    w.l = t.bad ? __builtin_nanf("") : 0.0f;
}

// Keys that every one of rows [r0, r1) sees: [lo, hi].
struct Whole {
    int lo, hi;
    __device__ __forceinline__ bool has(int key0) const { return key0 >= lo && key0 + UNIT - 1 <= hi; }
};
__device__ __forceinline__ Whole whole_of(const Kv4AttnArgs& a, const Tile& t, int r0, int r1) {
    return {a.window > 0 ? (int)max(0L, t.pos0 + (r1 - 1) / a.group - a.window + 1) : 0, (int)(t.pos0 + r0 / a.group)};
}

template <bool MASK>
__device__ __forceinline__ float row_max(const Row& w, int key, int sink, f4v c[4]) {
    float top = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if constexpr (MASK) {
                const int j = key + 4 * t + r;
                // (& and |: three comparisons and a select a score, no branch)
                const bool see = (j <= w.pos) & ((j >= w.lo) | (j < sink));
                c[t][r] = see ? c[t][r] : -__builtin_inff();
            }
            top = fmaxf(top, c[t][r]);
        }
    return rows_reduce(top, OpMax{});
}

// p = 2^(f (c - m) + PBIAS): the reference is taken from the score before it is
// scaled.  (c f - m f with m f rounded on its own is a step of fp32 off, past
// 2^27 more than p has room for: the largest p would be 0 or infinite.)
__device__ __forceinline__ float prob(const Row& w, float c) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(c - w.m, w.f, PBIAS));
}
// The reference follows a unit's maximum, and acc and l the reference.  It
// moves only when a maximum passes it by 2^PSLACK, so that most units leave
// acc alone.
__device__ __forceinline__ bool grows(const Row& w, float top) { return top > w.m && !(w.f * (top - w.m) <= PSLACK); }
template <int MT>
__device__ __forceinline__ float follow(Row& w, float top, f4v* acc) {  // what acc was multiplied by
    float keep = 1.0f;
    if (grows(w, top)) {
        // (a maximum past fp32's range: NaN, from here to the row's end)
        const float m = fabsf(w.f * top) <= FLT_MAX ? top : __builtin_nanf("");
        keep = __builtin_amdgcn_exp2f(w.f * (w.m - m));
        w.m = m;
    }
#pragma unroll
    for (int m = 0; m < MT; m++) acc[m] *= keep;
    return keep;
}
// Scores to probabilities as the second product's operands.
__device__ __forceinline__ void probabilities(Row& w, const f4v c[4], h8v ph[2], h8v pl[2]) {
    float p[2][8], sum = 0.0f;
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const float e = prob(w, c[x][y]);
            p[x >> 1][(x & 1) * 4 + y] = e;
            sum += e;
        }
    w.l += sum;
    split8(p[0], ph[0], pl[0]);
    split8(p[1], ph[1], pl[1]);
}
// Both, for scores of keys 16 g + 4 t + r of the unit at key0.
template <int MT>
__device__ __forceinline__ void softmax(Row& w, bool whole, int key0, int sink, f4v c[4], f4v* acc, h8v ph[2], h8v pl[2]) {
    const int key = key0 + 16 * ((threadIdx.x & 63) >> 4);
    const float top = whole ? row_max<false>(w, key, sink, c) : row_max<true>(w, key, sink, c);
    if (__any(grows(w, top))) w.l *= follow<MT>(w, top, acc);
    probabilities(w, c, ph, pl);
}

template <bool F16>
__device__ __forceinline__ void store4(const Kv4AttnArgs& a, long at, f4v o) {
    if constexpr (F16) {
        typedef _Float16 h4v __attribute__((ext_vector_type(4)));
        *(h4v*)((_Float16*)a.out + at) = h4v{(_Float16)o.x, (_Float16)o.y, (_Float16)o.z, (_Float16)o.w};
    } else {
        *(f4v*)((float*)a.out + at) = o;
    }
}

__device__ __forceinline__ long out_at(const Kv4AttnArgs& a, const Tile& t, int r, int hd) {
    return (long)(t.q0 + r / a.group) * a.out_stride + (long)(t.head * a.group + r % a.group) * hd;
}

// A tile whose units several blocks share: blocks [b0, b1].  Each leaves its
// rows in a slot of its own, two slots a block (the tile that it goes on with
// and the one that it leaves unfinished; other tiles it does whole).
struct Shared {
    int b0, b1;
    __device__ __forceinline__ bool split() const { return b1 > b0; }
    __device__ __forceinline__ long slot(int b) const { return b == b0 ? 2L * b + 1 : 2L * b; }
};
__device__ __forceinline__ Shared shared_of(const Work& w, const Piece& p) {
    const int b = blockIdx.x, d = (int)(p.first - (long)b * w.chunk);  // where the tile starts, from this block's start
    return {d >= 0 ? b : b - (w.chunk - 1 - d) / w.chunk, b + (d + p.n - 1) / w.chunk};
}
template <int HD, int R>
__device__ __forceinline__ unsigned part_at(long slot, int row) {  // floats into the partial rows
    return (unsigned)((slot * R + row) * (HD + 4));
}

// The tile that a block was the first on and left unfinished, for the join's
// launch; no rows: none.
struct alignas(16) Left {
    int q0, head, r0, r1, b1, pad[3];
};
__device__ __forceinline__ Left* left_of(const Kv4AttnArgs& a, int block) { return (Left*)((char*)a.part + a.part_bytes) + block; }

// Partial rows pass between blocks on different XCDs, whose L2s do not see each
// other's lines.  They are written and read past the L2s (cache policy sc1, as
// device-scope atomics are), and the writer waits for its stores before the
// counter: fences instead would write back and drop the whole L2 once per
// block (measured: 190 -> 430 us for 64 sequences of up to 16384 tokens at 16
// splits of their keys).
constexpr int SC1 = 16;
struct Parts {
    __amdgpu_buffer_rsrc_t rsrc;
    __device__ __forceinline__ void put4(unsigned at, f4v v) const {  // at: floats
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4v, v), rsrc, (int)(at * 4), 0, SC1);
    }
    __device__ __forceinline__ f4v get4(unsigned at) const {
        return __builtin_bit_cast(f4v, __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)(at * 4), 0, SC1));
    }
};
__device__ __forceinline__ Parts parts_of(const Kv4AttnArgs& a) {
    return {__builtin_amdgcn_make_buffer_rsrc(a.part, 0, a.part_bytes, 0x00027000)};
}

// The shared pieces of a block: the one that it went on with and the one that
// it leaves unfinished.
struct Shares {
    int n = 0;
    Shared sh[2];
    Tile t[2];
    __device__ __forceinline__ void add(const Shared& s, const Tile& tile) {
        if (n == 0) sh[0] = s, t[0] = tile;
        else sh[1] = s, t[1] = tile;
        n++;
    }
};
// A shared tile's rows to one: by the block that finishes last, over the
// blocks in order.  (The counter is left at 0 for the next call.)
template <int HD, bool F16, int R, int THREADS>
__device__ __forceinline__ void join_blocks(const Kv4AttnArgs& a, const Shares& p) {
    __shared__ int last[2];
    if (p.n == 0) return;
    const Parts parts = parts_of(a);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's partial rows have arrived
    __syncthreads();
    if (threadIdx.x < (unsigned)p.n) {
        const Shared& sh = threadIdx.x ? p.sh[1] : p.sh[0];
        const bool mine = __hip_atomic_fetch_add(a.count + sh.b0, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == sh.b1 - sh.b0;
        if (mine) __hip_atomic_store(a.count + sh.b0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last[threadIdx.x] = mine;
    }
    __syncthreads();
    constexpr int LPR = HD / 4, RPB = THREADS / LPR, PB = 4;
    constexpr int RU = R / RPB >= 4 ? 4 : R / RPB >= 2 ? 2 : 1;
    const int l = threadIdx.x % LPR;
    for (int k = 0; k < p.n; k++) {
        if (!last[k]) continue;
        const Tile& t = k ? p.t[1] : p.t[0];
        const Shared& sh = k ? p.sh[1] : p.sh[0];
        // RU rows and PB blocks' parts of them are loaded together: a load past
        // the L2 takes microseconds, and one after the other they would add up
        for (int r0 = t.r0 + threadIdx.x / LPR; r0 < t.r1; r0 += RU * RPB) {
            float m[RU], sum[RU];
            f4v o[RU];
#pragma unroll
            for (int x = 0; x < RU; x++) m[x] = -FLT_MAX, sum[x] = 0.0f, o[x] = f4v{0, 0, 0, 0};
            for (int b = sh.b0; b <= sh.b1; b += PB) {
                f4v n[RU][PB], v[RU][PB];
#pragma unroll
                for (int x = 0; x < RU; x++)
#pragma unroll
                    for (int y = 0; y < PB; y++) {
                        const unsigned q = part_at<HD, R>(sh.slot(min(b + y, sh.b1)), min(r0 + x * RPB, t.r1 - 1) - t.r0);
                        n[x][y] = parts.get4(q + HD);
                        v[x][y] = parts.get4(q + 4 * l);
                    }
#pragma unroll
                for (int x = 0; x < RU; x++)
#pragma unroll
                    for (int y = 0; y < PB; y++) {
                        if (b + y > sh.b1 || n[x][y].x == 0.0f) continue;  // (no key seen)
                        const float now = fmaxf(m[x], n[x][y].y), f = n[x][y].z;
                        const float keep = sum[x] != 0.0f ? __builtin_amdgcn_exp2f(f * (m[x] - now)) : 0.0f;
                        const float w = __builtin_amdgcn_exp2f(f * (n[x][y].y - now));
                        m[x] = now;
                        sum[x] = sum[x] * keep + w * n[x][y].x;
                        o[x] = o[x] * keep + v[x][y] * w;
                    }
            }
#pragma unroll
            for (int x = 0; x < RU; x++) {
                const int r = r0 + x * RPB;
                if (r < t.r1) store4<F16>(a, out_at(a, t, r, HD) + 4 * l, o[x] * (sum[x] != 0.0f ? 1.0f / sum[x] : 0.0f));
            }
        }
    }
}

// A block's W waves hold the same rows over different keys: their sums to
// one.  acc[m]: O^T tiles, dims 16 m + 4 g + r of row i.  Wave w ends with the
// tiles m = w, w + W, ... in out.
constexpr int tiles_of_wave(int hd, int w) { return hd / 16 > w ? hd / 16 / w : 1; }
template <int HD, int W>
__device__ __forceinline__ void join_waves(f4v* acc, const Row& w, float& l, float* m_all, float* smem, f4v* out) {
    constexpr int MT = HD / 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15;
    l = rows_sum(w.l);
    float* s_m = smem;                 // [W][16]
    float* s_l = smem + 16 * W;        // [W][16]
    f4v* s_o = (f4v*)(smem + 32 * W);  // [W][MT tiles][64 lanes], each to its own wave's reference
    __syncthreads();                   // the last piece's readers are done
    if (lane < 16) {
        s_m[wave * 16 + i] = l != 0.0f ? w.m : -FLT_MAX;  // no key seen: no weight (NaN counts as seen)
        s_l[wave * 16 + i] = l;
    }
#pragma unroll
    for (int m = 0; m < MT; m++) s_o[(wave * MT + m) * 64 + lane] = acc[m];
    __syncthreads();
    float top = s_m[i];
#pragma unroll
    for (int v = 1; v < W; v++) top = fmaxf(top, s_m[v * 16 + i]);
    float sum = 0.0f, f[W];
#pragma unroll
    for (int v = 0; v < W; v++) {
        const float x = s_l[v * 16 + i];
        f[v] = x != 0.0f ? __builtin_amdgcn_exp2f(w.f * (s_m[v * 16 + i] - top)) : 0.0f;
        sum += x * f[v];
    }
    l = sum;
    *m_all = top;
#pragma unroll
    for (int c = 0; c < tiles_of_wave(HD, W); c++) {
        const int m = c * W + wave;
        f4v o = {0, 0, 0, 0};
        if (m < MT)
#pragma unroll
            for (int v = 0; v < W; v++) o += s_o[(v * MT + m) * 64 + lane] * f[v];
        out[c] = o;
    }
}

// Up to 16 NT rows of a sequence and KV head (decode, a few drafts): a block's
// waves take the units of its piece in turn, each straight into registers.  A
// wave's K words are free once the scores are done and its V words once the
// output is: the loads of the wave's next unit go there and then.  V scales (a
// lane's operands need all 16 of its tokens', the same for 16 lanes) come as
// one 64th a lane and pass through LDS, which takes 8 wide loads and 32
// registers less than loading them to every lane.
// HBM bound where the batch is long: 64 sequences of up to 16384 keys, 32 / 4
// heads of 128, fp32 rows, 395 MB in 96 us (4.12 TB/s; a copy reaches 4.80).
// Short ones are a chain of latencies: 1000 keys of 32 / 8 heads of 64 9 us.
// One unit in flight a wave: two made hardly more of the bandwidth and much
// more code, which every block fetches first (24 sequences of 16 / 2 heads of
// 256, window 6001: 43 us, 47 with two).
template <int HD>
struct Raw {
    KRow<HD, HD / 32> k[4];
    u4v v[HD / 32];
    uint32_t vs[HD / 64];
    bool v_ok;
};
template <int HD, bool F16, int W, int NT>
__global__ __launch_bounds__(64 * W) void k_kv4_attn(Kv4AttnArgs a) {
    constexpr int KS = HD / 32, MT = HD / 16, SROW = HD + 16, R = 16 * NT;
    __shared__ __align__(16) float smem[32 * W + W * MT * 64 * 4];
    __shared__ __align__(16) uint8_t s_vs[W][4 * SROW];
    const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    Work work;
    Batch batch;
    if (!work_of<R>(a, work, batch, blockIdx.x, gridDim.x)) return;
    const int ps = 1 << a.c.ps_shift;
    Tile t;
    Units u;
    Piece part;
    Raw<HD> z;
    int kp, vp;  // pages of the unit to load next
    // (Past the piece's end its last unit is loaded again: behind a branch the
    // compiler could not tell which loads are in flight and would wait for all.)
    auto unit_of = [&](int n) { return u.at(max(min(n, part.hi - 1), 0)); };
    auto pages = [&](int n, int& k, int& v) {
        k = page_of(a, t.table, k_key(unit_of(n)));
        v = page_of(a, t.table, v_key(unit_of(n)));
    };
    auto load_k = [&](int n, int page) {
        bool ok;
        const int key = k_key(unit_of(n)), off = key & (ps - 1);
        const uint8_t* p = page_ptr(a, page, key, t.head, ok);
#pragma unroll
        for (int x = 0; x < 4; x++) load_krow<HD, KS>(p, ok, ps, off + 4 * x, 0, z.k[x]);
    };
    auto load_v = [&](int n, int page) {
        const int key = v_key(unit_of(n)), grp = (key & (ps - 1)) >> 4;
        const uint8_t* p = page_ptr(a, page, key, t.head, z.v_ok);
        const uint8_t* c = p + ps * (HD / 2) + grp * (HD * 8) + i * 16;
#pragma unroll
        for (int b = 0; b < KS; b++) z.v[b] = *gptr<u4v>(c + b * 256);
        const uint8_t* s = p + ps * HD + ps * (HD / 16) + grp * HD + i * (HD / 16);
        if constexpr (HD == 64) {
            z.vs[0] = *gptr<uint32_t>(s);
        } else if constexpr (HD == 128) {
            const u2v x = *gptr<u2v>(s);
            z.vs[0] = x.x, z.vs[1] = x.y;
        } else {
            const u4v x = *gptr<u4v>(s);
            z.vs[0] = x.x, z.vs[1] = x.y, z.vs[2] = x.z, z.vs[3] = x.w;
        }
    };
    h8v qh[NT][KS], ql[NT][F16 ? 1 : KS];
    float f[NT];
    // the next piece, its q rows and its first units' loads
    auto begin = [&]() {
        piece_of<R>(a, work, batch, t, u, part);
        const int n0 = part.lo + wave;
        pages(n0, kp, vp);
#pragma unroll
        for (int x = 0; x < NT; x++)  // (rows past the last repeat it)
            load_q<HD, F16>(a, t, min(t.r0 + 16 * x + i, t.r1 - 1), qh[x], ql[x], f[x]);
        load_k(n0, kp);
        load_v(n0, vp);
        pages(n0 + W, kp, vp);
    };
    Shares shares;
    begin();
    for (;;) {
        Row w[NT];
        f4v acc[NT][MT];
#pragma unroll
        for (int x = 0; x < NT; x++) {
            row_init(a, t, min(t.r0 + 16 * x + i, t.r1 - 1), f[x], w[x]);
#pragma unroll
            for (int m = 0; m < MT; m++) acc[x][m] = f4v{0, 0, 0, 0};
        }
        const Whole whole = whole_of(a, t, t.r0, t.r1);
        for (int n = part.lo + wave; n < part.hi; n += W) {
            const int key0 = u.at(n) * UNIT, next = n + W;
            f4v c[NT][4];
#pragma unroll
            for (int x = 0; x < NT; x++)
#pragma unroll
                for (int y = 0; y < 4; y++) c[x][y] = f4v{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const h8v o = k_operand(z.k[y].w[s], z.k[y].scale(s));
#pragma unroll
                    for (int x = 0; x < NT; x++) {
                        c[x][y] = mfma(o, qh[x][s], c[x][y]);
                        if constexpr (!F16) c[x][y] = mfma(o, ql[x][s], c[x][y]);
                    }
                }
            const int vnext = vp;
            load_k(next, kp);
            pages(next + W, kp, vp);
            h8v ph[NT][2], pl[NT][2];
#pragma unroll
            for (int x = 0; x < NT; x++) softmax<MT>(w[x], whole.has(key0), key0, a.sink, c[x], acc[x], ph[x], pl[x]);
            // scales of this lane: tokens 16 g + HD / 32 * (i % (512 / HD)) .. of block i / (512 / HD)
            uint32_t vs[HD / 64];
#pragma unroll
            for (int y = 0; y < HD / 64; y++) vs[y] = z.vs[y];
            if (key0 + UNIT > t.len || !z.v_ok) {
                const int key = key0 + 16 * g + (HD / 32) * (i % (512 / HD)), len = z.v_ok ? t.len : 0;
#pragma unroll
                for (int y = 0; y < HD / 64; y++)
                    vs[y] = key + 2 * y + 1 < len ? vs[y] : key + 2 * y < len ? vs[y] & 0xFFFFu : 0;
            }
            uint8_t* sv = s_vs[wave];
            if constexpr (HD == 64) *(uint32_t*)(sv + g * SROW + i * 4) = vs[0];
            else if constexpr (HD == 128) *(u2v*)(sv + g * SROW + i * 8) = u2v{vs[0], vs[1]};
            else *(u4v*)(sv + g * SROW + i * 16) = u4v{vs[0], vs[1], vs[2], vs[3]};
#pragma unroll
            for (int b = 0; b < KS; b++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    VPart v;
                    v.w = y ? u2v{z.v[b].z, z.v[b].w} : u2v{z.v[b].x, z.v[b].y};
                    v.s = *(const u4v*)(sv + g * SROW + b * 32 + y * 16);
                    h8v lo, hi;
                    v_operands(v, lo, hi);
#pragma unroll
                    for (int x = 0; x < NT; x++) {
                        acc[x][2 * b] = mfma(lo, ph[x][y], acc[x][2 * b]);
                        acc[x][2 * b + 1] = mfma(hi, ph[x][y], acc[x][2 * b + 1]);
                        acc[x][2 * b] = mfma(lo, pl[x][y], acc[x][2 * b]);
                        acc[x][2 * b + 1] = mfma(hi, pl[x][y], acc[x][2 * b + 1]);
                    }
                }
            load_v(next, vnext);
        }
        // the next piece's loads are on their way while this one is put together
        const Tile done = t;
        const Shared sh = shared_of(work, part);
        const bool more = work.left > 0;
        if (more) begin();
#pragma unroll
        for (int x = 0; x < NT; x++) {
            float l, m;
            f4v o[tiles_of_wave(HD, W)];
            join_waves<HD, W>(acc[x], w[x], l, &m, smem, o);
            const int r = done.r0 + 16 * x + i;
            if (r >= done.r1 || wave >= MT) continue;
            if (!sh.split()) {
                const float inv = l != 0.0f ? 1.0f / l : 0.0f;
                const long at = out_at(a, done, r, HD);
#pragma unroll
                for (int c = 0; c < tiles_of_wave(HD, W); c++) store4<F16>(a, at + 16 * (c * W + wave) + 4 * g, o[c] * inv);
            } else {
                const Parts parts = parts_of(a);
                const unsigned row = part_at<HD, R>(sh.slot(blockIdx.x), r - done.r0);
#pragma unroll
                for (int c = 0; c < tiles_of_wave(HD, W); c++) parts.put4(row + 16 * (c * W + wave) + 4 * g, o[c]);
                if (wave == 0 && g == 0) parts.put4(row + HD, f4v{l, m, w[x].f, 0});
            }
        }
        if (sh.split()) shares.add(sh, done);
        if (!more) break;
    }
    join_blocks<HD, F16, R, 64 * W>(a, shares);
}

// More rows (drafts, prompts): W waves of 16 NT rows over the same units, whose
// codes they turn into f16 operands in LDS together, in the order in which a
// lane reads them (16 bytes a lane, no bank conflict).  A SIMD overlaps matrix
// products with vector work only where the two stand side by side in the
// stream (waves that share operands run in step), so a turn computes the
// exponentials of unit n among the products of unit n + 1's scores, and stages
// later units' operands among unit n's output products.  K operands are staged
// two units ahead and V operands one; one barrier a turn.
// 2048 rows of 32 / 4 heads of 128 over 8192 keys: f16 391 us, 361 GFLOP of
// products issued (p's second term makes them three for two), 923 TFLOP/s, where
// a library product of 8192^3 reaches 1123; fp32 445 us, 481 GFLOP, 1081.  The
// matrix units are busy 40 % of the time, vector instructions issue in 55 %, and
// the two overlap little: bound by their sum.  Two row tiles a wave do not fit
// the registers there (f16 441 us, 31 spilled).  With p as one f16 the f16 call
// took 273 us, and its rows were off by up to 2^-11 of the values before their
// own rounding.
template <int HD, bool F16, int W, int NT, bool SPLIT>
__global__ __launch_bounds__(64 * W, HD == 256 && W == 4 ? 1 : 2) void k_kv4_attn_prompt(Kv4AttnArgs a) {
    constexpr int KS = HD / 32, MT = HD / 16, R = 16 * NT * W;
    constexpr int KW = 4 * KS / W;                    // K words a lane stages
    constexpr int NJ = 2 * KS >= W ? 2 * KS / W : 1;  // V parts a lane stages (HD 64, 8 waves: the first 4)
    __shared__ __align__(16) h8v s_k[2][4 * KS * 64];  // [word][key tile][lane]
    __shared__ __align__(16) h8v s_v[2][4 * KS * 64];  // [block][part][low, high][lane]
    const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    Work work;
    Batch batch;
    Tile t;
    const bool one = !SPLIT || a.whole;
    if (one) {
        if (!whole_tile<R>(a, t)) return;
        work.left = 0;
    } else if constexpr (SPLIT) {
        if (!work_of<R>(a, work, batch, blockIdx.x, gridDim.x)) {
            if (threadIdx.x == 0) *left_of(a, blockIdx.x) = Left{};
            return;
        }
    }
    const int ps = 1 << a.c.ps_shift;
    const int kt = wave & 3, s0 = W == 8 ? (wave >> 2) * KW : 0, j0 = wave * NJ;
    const bool stage_v = j0 < 2 * KS;
    do {
        Units u;
        Piece part;
        if (one) {
            u = tile_units(a, t, t.r0, t.r1);
            part.lo = 0;
            part.hi = u.n;
        } else if constexpr (SPLIT) {
            piece_of<R>(a, work, batch, t, u, part);
        }
        const int units = part.hi - part.lo;
        __syncthreads();  // the last piece's operands are read
        KRow<HD, KW> k;
        VPart v[NJ];
        int kp, vp;  // pages of the units to load next
        bool v_ok = true;
        // (past the end the last unit again: no branch around loads)
        auto unit_of = [&](int n) { return u.at(max(min(part.lo + n, part.hi - 1), 0)); };
        auto load_k = [&](int n) {  // unit n's K codes, and the page of unit n + 1
            bool ok;
            const int key = k_key(unit_of(n));
            const uint8_t* p = page_ptr(a, kp, key, t.head, ok);
            load_krow<HD, KW>(p, ok, ps, (key & (ps - 1)) + 4 * kt, s0, k);
            kp = page_of(a, t.table, k_key(unit_of(n + 1)));
        };
        auto load_v = [&](int n) {
            const int key = v_key(unit_of(n));
            const uint8_t* p = page_ptr(a, vp, key, t.head, v_ok);
#pragma unroll
            for (int j = 0; j < NJ; j++) load_vpart<HD>(p, ps, key & (ps - 1), ((j0 + j) >> 1) & (KS - 1), (j0 + j) & 1, v[j]);
            vp = page_of(a, t.table, v_key(unit_of(n + 1)));
        };
        auto stage_k = [&](int n) {
            h8v* bk = s_k[n & 1];
#pragma unroll
            for (int s = 0; s < KW; s++) bk[((s0 + s) * 4 + kt) * 64 + lane] = k_operand(k.w[s], k.scale(s));
        };
        auto cut_v = [&](int n) {
            const int key0 = unit_of(n) * UNIT;
            if (key0 + UNIT > t.len || !v_ok) {
#pragma unroll
                for (int j = 0; j < NJ; j++) cut_vpart(v[j], key0 + 16 * g + 8 * ((j0 + j) & 1), v_ok ? t.len : 0);
            }
        };
        auto stage_v_ops = [&](int n) {
            h8v* bv = s_v[n & 1];
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                h8v lo, hi;
                v_operands(v[j], lo, hi);
                if (2 * KS >= W || stage_v) {
                    bv[((j0 + j) * 2 + 0) * 64 + lane] = lo;
                    bv[((j0 + j) * 2 + 1) * 64 + lane] = hi;
                }
            }
        };
        kp = page_of(a, t.table, k_key(unit_of(0)));
        vp = page_of(a, t.table, v_key(unit_of(0)));
        // this wave's rows; a wave without any repeats the tile's last and stores nothing
        const int mine = t.r0 + wave * 16 * NT, r0 = min(mine, t.r1 - 1), r1 = min(mine + 16 * NT, t.r1);
        h8v qh[NT][KS], ql[NT][F16 ? 1 : KS];
        Row w[NT];
        f4v acc[NT][MT], c[NT][4], d[NT][4];
#pragma unroll
        for (int x = 0; x < NT; x++) {
            const int r = min(r0 + 16 * x + i, t.r1 - 1);
            float f;
            load_q<HD, F16>(a, t, r, qh[x], ql[x], f);
            row_init(a, t, r, f, w[x]);
#pragma unroll
            for (int m = 0; m < MT; m++) acc[x][m] = f4v{0, 0, 0, 0};
        }
        const Whole whole = whole_of(a, t, r0, max(r1, r0 + 1));
        load_k(0);
        load_v(0);
        stage_k(0);
        cut_v(0);
        stage_v_ops(0);
        load_k(1);
        load_v(1);
        stage_k(1);
        load_k(2);
        lds_barrier();
        // Operands are read one step ahead of their products, and each step's
        // products have a share of the vector work between them: left to itself the
        // compiler reads an operand where it is used and waits out the LDS.
        h8v cur[4], nxt[4];
        auto read = [&](const h8v* p, h8v (&o)[4]) {
#pragma unroll
            for (int y = 0; y < 4; y++) o[y] = p[y * 64 + lane];
        };
        auto products = [&](int e, f4v (&s)[NT][4]) {
#pragma unroll
            for (int y = 0; y < 4; y++)
#pragma unroll
                for (int x = 0; x < NT; x++) s[x][y] = mfma(cur[y], qh[x][e], s[x][y]);
            if constexpr (!F16) {
#pragma unroll
                for (int y = 0; y < 4; y++)
#pragma unroll
                    for (int x = 0; x < NT; x++) s[x][y] = mfma(cur[y], ql[x][e], s[x][y]);
            }
        };
        auto clear = [&](f4v (&s)[NT][4]) {
#pragma unroll
            for (int x = 0; x < NT; x++)
#pragma unroll
                for (int y = 0; y < 4; y++) s[x][y] = f4v{0, 0, 0, 0};
        };
        constexpr int QM = 4 * NT * (F16 ? 1 : 2), PM = 8 * NT;  // products of a step: scores, output
        auto interleave = [&](auto n, auto vec) {                // n.value products, vec.value vector instructions behind each
#pragma unroll
            for (int m = 0; m < decltype(n)::value; m++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, decltype(vec)::value, 0);
            }
        };
        clear(c);
#pragma unroll
        for (int e = 0; e < KS; e++) {
            read(s_k[0] + e * 256, cur);
            products(e, c);
        }
        lds_barrier();  // unit 0's K buffer goes to unit 2
        // Sums of the rounded p, by products with ones (a lane's column is its row):
        // less work than adding, and the weights that are applied sum to one.
        f4v sum[NT];
        h8v ones;
#pragma unroll
        for (int e = 0; e < 8; e++) ones[e] = (_Float16)1.0f;
#pragma unroll
        for (int x = 0; x < NT; x++) sum[x] = f4v{w[x].l, w[x].l, w[x].l, w[x].l};
        auto turn = [&](int n, f4v (&c)[NT][4], f4v (&d)[NT][4]) {
            const int key0 = unit_of(n) * UNIT;
            const bool all = whole.has(key0);
            const h8v *bk = s_k[(n + 1) & 1], *bv = s_v[n & 1];
            read(bk, cur);
            float top[NT];
            if (all) {
#pragma unroll
                for (int x = 0; x < NT; x++) top[x] = row_max<false>(w[x], key0 + 16 * g, a.sink, c[x]);
            } else {
#pragma unroll
                for (int x = 0; x < NT; x++) top[x] = row_max<true>(w[x], key0 + 16 * g, a.sink, c[x]);
            }
            bool grow = false;
#pragma unroll
            for (int x = 0; x < NT; x++) grow |= grows(w[x], top[x]);
            if (__any(grow)) {
#pragma unroll
                for (int x = 0; x < NT; x++) {
                    const float keep = follow<MT>(w[x], top[x], acc[x]);
                    sum[x] *= keep;
                }
            }
            cut_v(n + 1);
            // scores of unit n + 1, probabilities of unit n
            u4v ph[NT][2], pl[NT][2];
            clear(d);
#pragma unroll
            for (int e = 0; e < KS; e++) {
                read(e + 1 < KS ? bk + (e + 1) * 256 : bv, nxt);
                __builtin_amdgcn_sched_barrier(0);
                products(e, d);
#pragma unroll
                for (int y = e * 4 / KS; y < (e + 1) * 4 / KS; y++)
#pragma unroll
                    for (int x = 0; x < NT; x++)
#pragma unroll
                        for (int z = 0; z < 2; z++) {
                            float p[2];
#pragma unroll
                            for (int k = 0; k < 2; k++) p[k] = prob(w[x], c[x][y][2 * z + k]);
                            const Two t = split2(p[0], p[1]);
                            ph[x][y >> 1][2 * (y & 1) + z] = t.hi;
                            pl[x][y >> 1][2 * (y & 1) + z] = t.lo;
                        }
                interleave(std::integral_constant<int, QM>(), std::integral_constant<int, 16 * NT * 4 / KS / QM>());
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < 4; y++) cur[y] = nxt[y];
            }
            // output of unit n; operands of units n + 2 and n + 1, codes of the units after them
#pragma unroll
            for (int b = 0; b < KS; b++) {
                if (b + 1 < KS) read(bv + (b + 1) * 256, nxt);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < 2; y++) {
#pragma unroll
                    for (int x = 0; x < NT; x++) {
                        acc[x][2 * b] = mfma(cur[2 * y], as_h8(ph[x][y]), acc[x][2 * b]);
                        acc[x][2 * b + 1] = mfma(cur[2 * y + 1], as_h8(ph[x][y]), acc[x][2 * b + 1]);
                    }
#pragma unroll
                    for (int x = 0; x < NT; x++) {
                        acc[x][2 * b] = mfma(cur[2 * y], as_h8(pl[x][y]), acc[x][2 * b]);
                        acc[x][2 * b + 1] = mfma(cur[2 * y + 1], as_h8(pl[x][y]), acc[x][2 * b + 1]);
                    }
                }
                if (b == 0) {
                    stage_k(n + 2);
                    load_k(n + 3);
                }
                if (b == KS / 2) {
                    stage_v_ops(n + 1);
                    load_v(n + 2);
                }
                if (b == KS - 1) {
#pragma unroll
                    for (int x = 0; x < NT; x++)
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            sum[x] = mfma(ones, as_h8(ph[x][y]), sum[x]);
                            sum[x] = mfma(ones, as_h8(pl[x][y]), sum[x]);
                        }
                }
                interleave(std::integral_constant<int, PM>(), std::integral_constant<int, 4>());
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < 4; y++) cur[y] = nxt[y];
            }
            lds_barrier();
        };
        for (int n = 0; n < units; n += 2) {  // (two turns: the scores change places without copies)
            turn(n, c, d);
            if (n + 1 < units) turn(n + 1, d, c);
        }
        const Shared sh = one ? Shared{0, 0} : shared_of(work, part);
        if (SPLIT && !one && work.left == 0 && threadIdx.x == 0)  // (a block's last piece is the one that others may share)
            *left_of(a, blockIdx.x) = sh.split() && sh.b0 == (int)blockIdx.x ? Left{t.q0, t.head, t.r0, t.r1, sh.b1, {}} : Left{};
#pragma unroll
        for (int x = 0; x < NT; x++) {
            const float l = sum[x][0];
            const int r = mine + 16 * x + i;
            if (r >= r1) continue;
            if (!sh.split()) {
                const float inv = l != 0.0f ? 1.0f / l : 0.0f;
                const long at = out_at(a, t, r, HD);
#pragma unroll
                for (int m = 0; m < MT; m++) store4<F16>(a, at + 16 * m + 4 * g, acc[x][m] * inv);
            } else {
                float* row = a.part + part_at<HD, R>(sh.slot(blockIdx.x), r - t.r0);
#pragma unroll
                for (int m = 0; m < MT; m++) *(f4v*)(row + 16 * m + 4 * g) = acc[x][m];
                if (g == 0) *(f4v*)(row + HD) = f4v{l, w[x].m, w[x].f, 0};
            }
        }
    } while (SPLIT && work.left > 0);
}

// The shared tiles of 64 rows to one, in a launch of its own: block (b, s) has
// some rows of the tile that block b was the first on and left unfinished, one
// a lane group.  (By the block that finishes last, as above, one block read all
// parts of 64 rows: 16 rows a sequence of 9000 keys, 8 sequences, 64 us, now 48.
// With the record of `Left` a block knows its tile after one read: 24 sequences
// of 5 rows, window 6001, 16 / 2 heads of 256 8 us, 17 where it searched.)
template <int HD, bool F16, int R>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4AttnArgs a) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR, PB = 8;  // (eight blocks' parts in flight)
    const Left left = *left_of(a, blockIdx.x);
    const Shared sh = {(int)blockIdx.x, left.b1};
    Tile t;
    t.q0 = left.q0, t.head = left.head, t.r0 = left.r0, t.r1 = left.r1;
    const int l = threadIdx.x % LPR, r = t.r0 + (int)blockIdx.y * RPB + threadIdx.x / LPR;
    if (r < t.r1) {
        float m = -FLT_MAX, sum = 0.0f;
        f4v o = {0, 0, 0, 0};
        for (int b = sh.b0; b <= sh.b1; b += PB) {
            f4v n[PB], v[PB];
#pragma unroll
            for (int y = 0; y < PB; y++) {
                const float* q = a.part + part_at<HD, R>(sh.slot(min(b + y, sh.b1)), r - t.r0);
                n[y] = *(const f4v*)(q + HD);
                v[y] = *(const f4v*)(q + 4 * l);
            }
#pragma unroll
            for (int y = 0; y < PB; y++) {
                if (b + y > sh.b1 || n[y].x == 0.0f) continue;  // (no key seen)
                const float now = fmaxf(m, n[y].y), f = n[y].z;
                const float keep = sum != 0.0f ? __builtin_amdgcn_exp2f(f * (m - now)) : 0.0f;
                const float w = __builtin_amdgcn_exp2f(f * (n[y].y - now));
                m = now;
                sum = sum * keep + w * n[y].x;
                o = o * keep + v[y] * w;
            }
        }
        store4<F16>(a, out_at(a, t, r, HD) + 4 * l, o * (sum != 0.0f ? 1.0f / sum : 0.0f));
    }
}

template <int HD, bool F16>
void attn_run(const Kv4AttnArgs& a, const Kv4AttnPlan& p, hipStream_t st) {
    const dim3 grid((unsigned)p.grid);
    constexpr int NT = HD == 64 ? 2 : 1;  // row tiles a wave of the large tiles
    if (p.rows == 16) {
        hipLaunchKernelGGL((k_kv4_attn<HD, F16, 4, 1>), grid, dim3(256), 0, st, a);
    } else if (HD == 128 && p.rows == 32) {
        hipLaunchKernelGGL((k_kv4_attn<128, F16, 4, 2>), grid, dim3(256), 0, st, a);
    } else if (p.rows == 64) {
        hipLaunchKernelGGL((k_kv4_attn_prompt<HD, F16, 4, 1, true>), grid, dim3(256), 0, st, a);
        if (p.whole) return;
        constexpr int RPB = 256 / (HD / 4);
        hipLaunchKernelGGL((k_kv4_join<HD, F16, 64>), dim3((unsigned)p.grid, 64 / RPB), dim3(256), 0, st, a);
    } else if constexpr (HD != 256 || F16) {
        hipLaunchKernelGGL((k_kv4_attn_prompt<HD, F16, 8, NT, false>), grid, dim3(512), 0, st, a);
    }
}

}  // namespace

// Which kernel, by the caller's largest row count (a hint: every kernel serves
// every batch).  Measured on 256 CUs, us:
// - up to 16 rows a sequence and KV head the decode kernel, whose waves share
//   nothing but the rows; more rows would read the pages once per 16 of them.
// - up to 32 at head dim 128 the same with two row tiles (352 registers in f16,
//   387 in fp32, so one block a CU): 24 sequences of 5 drafts over 20011 keys,
//   window 6001, 32 / 8 heads, 76 against 116 in tiles of 64 in fp32 and 75
//   against 102 in f16.  At 64 (12 drafts of 32 / 8 heads over 8000 keys 73
//   against 55) and at 256, where they spill (5 drafts 98 against 71), the tiles
//   of 64 are faster.
// - tiles of 64 rows, and of 128 (256 at head dim 64; at 256 in fp32 the
//   registers leave no larger one) where there is one for every CU: 2048 rows of
//   32 / 4 heads of 128 over 8192 keys 409 against 435 in f16, 461 against 487 in
//   fp32.  At head dim 64, where staging is a smaller part, from two a CU on: five
//   prompts of 777 are as fast either way, one of 8000 (1000 tiles) 584 against
//   682.  At 256, whose small tiles leave one wave a SIMD, from one for two CUs:
//   1500 rows over 3000 keys 134 against 158.
// - tiles whole, one a block, where there is one for every CU (four prompts of
//   300: 15 against 31 split); else equal stretches of their units for two
//   blocks a CU (one at head dim 256, whose operands fill the LDS), and the
//   join's launch: 300 rows over 5000 keys 62 against 90 whole.
// - the decode kernel at head dims 64 and 128: two blocks a CU where the batch
//   has tiles or units for them (64 sequences of 1000 keys, 8 KV heads of 128
//   32 against 45 with one; 64 of 16384 95 against 112), else one, whose longer
//   stretches leave fewer parts to join (20 of 3000, 8 KV heads of 128 25
//   against 29; 24 windows of 6001, 4 KV heads 31 against 35).
// A block takes `chunk` units at least.  Of a tile of n units the decode kernel's
// blocks go through chunk / 4 turns and its last one through n / chunk parts
// of 4 a turn, each a round trip: least near sqrt(2 n), a multiple of the 4
// waves (one token over 10000 keys, 32 / 4 heads of 128: 27 us, 42 at 4 units
// always; over 100000 keys of 64 38 against 48).  The join's launch reads all
// parts at once: 2 (4 drafts of 30 rows over 700 keys of 256 29 us, 33 at 4).
Kv4AttnPlan kv4_attn_plan(int hd, bool f16, int n_seq, int n_tok, int n_head, int n_kv, int max_q, long max_keys,
                          int cus) {
    Kv4AttnPlan p = {};
    const int group = n_head / n_kv;
    const int big = hd == 64 ? 256 : hd == 256 && !f16 ? 64 : 128;
    const long rows = (long)max_q * group;
    auto tiles = [&](int r) { return (long)n_tok * group / r * n_kv; };
    p.rows = rows <= 16 ? 16 : rows > 64 && 2 * tiles(big) >= (hd == 64 ? 4 : hd == 128 ? 2 : 1) * cus ? big : 64;
    if (hd == 128 && p.rows == 64 && rows <= 32) p.rows = 32;
    p.whole = p.rows > 64 || (p.rows == 64 && tiles(64) >= cus);
    const long decode = (long)n_seq * n_kv;  // tiles of the decode kernel
    const bool two = hd != 256 && (p.rows == 64 || (p.rows == 16 && (3 * decode >= 2 * cus || (double)decode * max_keys >= 64.0 * UNIT * cus)));
    p.grid = p.whole ? ((long)n_tok * group / p.rows + n_seq) * n_kv : (two ? 2 : 1) * cus;
    p.chunk = p.rows <= 32 ? 4 * (int)fmax(1.0, 0.25 * sqrt(2.0 * (double)max_keys / UNIT) + 0.5) : 2;
    p.part_bytes = p.whole ? 0 : (size_t)p.grid * 2 * p.rows * (hd + 4) * sizeof(float);
    p.work = p.whole ? 0 : KV4_COUNT_BYTES + p.part_bytes + (p.rows == 64 ? p.grid * sizeof(Left) : 0);
    return p;
}

// Of split tiles of 64 rows, the most of any plan.
size_t kv4_attn_workspace(int hd, int cus) {
    return KV4_COUNT_BYTES + (size_t)(hd != 256 ? 2 : 1) * cus * (2 * 64 * (hd + 4) * sizeof(float) + sizeof(Left));
}

int kv4_attn(Kv4AttnArgs a, bool f16, const Kv4AttnPlan& p, void* work, hipStream_t st) {
    if (p.grid > KV4_MAX_GRID / (p.rows > 64 ? 2 : 1)) return -1;  // (512 threads from 128 rows on)
    a.whole = p.whole;
    a.part_bytes = (unsigned)p.part_bytes;
    a.chunk = p.chunk;
    a.count = (int*)work;
    a.part = (float*)((char*)work + KV4_COUNT_BYTES);
    switch (a.c.hd) {
    case 64: f16 ? attn_run<64, true>(a, p, st) : attn_run<64, false>(a, p, st); return 0;
    case 128: f16 ? attn_run<128, true>(a, p, st) : attn_run<128, false>(a, p, st); return 0;
    case 256: f16 ? attn_run<256, true>(a, p, st) : attn_run<256, false>(a, p, st); return 0;
    }
    return -1;
}

}  // namespace draco
