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
// K and V values are exact in f16 (kv4.h).  fp32 rows: q (scaled by a power of
// two to [1, 2) of its largest) and p are split into two f16 terms, 22 bits of
// each, and every product runs twice into one fp32 sum.  f16 rows: q is exact
// and p is rounded once, to nearest (2^-12 of itself, as the output's own
// rounding).
#include <hip/hip_runtime.h>

#include "dev_common.h"
#include "kv4.h"

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

// Eight consecutive tokens' bytes (w0, w1) of a pair of dims, times the
// tokens' scales: the operand of the low nibbles' dim and of the high ones'.
__device__ __forceinline__ void v_operands(uint32_t w0, uint32_t w1, const uint32_t s[4], h8v& lo, h8v& hi) {
    uint32_t l[4], h[4];
    const h2v c[8] = {fp4x2<0>(w0), fp4x2<1>(w0), fp4x2<2>(w0), fp4x2<3>(w0),
                      fp4x2<0>(w1), fp4x2<1>(w1), fp4x2<2>(w1), fp4x2<3>(w1)};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        l[i] = as_u(as_h2(__builtin_amdgcn_perm(as_u(c[2 * i + 1]), as_u(c[2 * i]), 0x05040100)) * as_h2(s[i]));
        h[i] = as_u(as_h2(__builtin_amdgcn_perm(as_u(c[2 * i + 1]), as_u(c[2 * i]), 0x07060302)) * as_h2(s[i]));
    }
    lo = __builtin_bit_cast(h8v, u4v{l[0], l[1], l[2], l[3]});
    hi = __builtin_bit_cast(h8v, u4v{h[0], h[1], h[2], h[3]});
}

// Eight fp32 values as one (F16) or two f16 operands.
template <bool F16>
__device__ __forceinline__ void split8(const float x[8], h8v& hi, h8v& lo) {
#pragma unroll
    for (int i = 0; i < 8; i++) hi[i] = (_Float16)x[i];
    if constexpr (!F16) {
#pragma unroll
        for (int i = 0; i < 8; i++) lo[i] = (_Float16)__builtin_fmaf((float)hi[i], -1.0f, x[i]);
    }
}

// What a block works on: one sequence's rows [r0, r0 + rows) of a KV head.
struct Tile {
    int q0, qn, len, rows, r0, head;  // head: the KV head
    bool bad;                         // the length passes the table: NaN
    long pos0;                        // position of the sequence's first query
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

__device__ __forceinline__ void seq_of(const Kv4AttnArgs& a, int seq, int head, Tile& t) {
    t.q0 = min(max(a.cu_q[seq], 0), a.n_tok);
    t.qn = min(max(a.cu_q[seq + 1], t.q0), a.n_tok) - t.q0;
    t.rows = t.qn * a.group;
    t.head = head;
    const int len = max(a.kv_len[seq], 0);
    const long cap = (long)a.max_blocks << a.c.ps_shift;
    t.bad = len > cap;
    t.len = t.bad ? 0 : len;
    t.pos0 = (long)t.len - t.qn;
}

// Address of a page's head, or null for a page outside the pool.
__device__ __forceinline__ const uint8_t* page_ptr(const Kv4AttnArgs& a, const int* table, int key, int head) {
    const int b = key >> a.c.ps_shift;
    const int p = b < a.max_blocks ? table[b] : 0;  // past the table only behind the last key
    return (unsigned)p < (unsigned)a.c.n_pages ? a.c.data + (long)p * a.c.page_bytes + (long)head * a.c.head_bytes : nullptr;
}

template <int HD>
struct KRaw {  // one wave's K of a unit
    static constexpr int W = HD / 32;  // 8-code words per lane and tile
    uint32_t w[4][W];
    uint16_t s[4][HD == 256 ? 2 : 1];
};
template <int HD>
struct VRaw {
    static constexpr int B = HD / 32;
    u4v w[B], s[B][2];
};

// Lane (i = lane & 15, g = lane >> 4) of operand tile t holds dims of key
// 16 (i / 4) + 4 t + i % 4: tile t's result rows are then keys 16 g' + 4 t + r
// for lane group g', so that a lane group ends with 16 consecutive keys.
template <int HD>
__device__ __forceinline__ void load_k(const Kv4AttnArgs& a, const int* table, int head, int unit, KRaw<HD>& k) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int ps = 1 << a.c.ps_shift;
    const int key = unit * UNIT + 16 * (i >> 2) + (i & 3);
    const uint8_t* p = page_ptr(a, table, key, head);
    const bool ok = p != nullptr;
    if (!ok) p = a.c.data;  // any readable page; its scores become NaN
    const int off = key & (ps - 1);
    const uint8_t* sc = p + ps * HD;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint8_t* row = p + (off + 4 * t) * (HD / 2);
        if constexpr (HD == 64) {
            const u2v v = *gptr<u2v>(row + g * 8);
            k.w[t][0] = v.x, k.w[t][1] = v.y;
            k.s[t][0] = *gptr<uint16_t>(sc + ((off + 4 * t) * 2 + (g >> 1)) * 2);
        } else {
#pragma unroll
            for (int c = 0; c < HD / 128; c++) {
                const u4v v = *gptr<u4v>(row + c * 64 + g * 16);
                k.w[t][4 * c] = v.x, k.w[t][4 * c + 1] = v.y, k.w[t][4 * c + 2] = v.z, k.w[t][4 * c + 3] = v.w;
                k.s[t][c] = *gptr<uint16_t>(sc + ((off + 4 * t) * (HD / 32) + c * 4 + g) * 2);
            }
        }
        if (!ok) k.s[t][0] = 0x7E00;
    }
}

// Lane (i, g): bytes of 16 tokens (the page group of keys 16 g ..) for dims
// 32 b + i and 32 b + 16 + i.
template <int HD>
__device__ __forceinline__ void load_v(const Kv4AttnArgs& a, const int* table, int head, int unit, int len, VRaw<HD>& v) {
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int ps = 1 << a.c.ps_shift;
    const int key = unit * UNIT + 16 * g;
    const uint8_t* p = page_ptr(a, table, key, head);
    const bool ok = p != nullptr && key < len;
    if (p == nullptr) p = a.c.data;
    const int grp = (key & (ps - 1)) >> 4;
    const uint8_t* w = p + ps * (HD / 2) + grp * (HD * 8) + i * 16;
    const uint8_t* s = p + ps * HD + ps * (HD / 16) + grp * HD;
#pragma unroll
    for (int b = 0; b < HD / 32; b++) {
        v.w[b] = *gptr<u4v>(w + b * 256);
        v.s[b][0] = *gptr<u4v>(s + b * 32);
        v.s[b][1] = *gptr<u4v>(s + b * 32 + 16);
    }
    // Rows behind the last token hold anything, NaN scales too: p = 0 would not
    // hide them.  (A row that is in the cache has finite V scales.)
    if (unit * UNIT + UNIT > len || !ok) {
#pragma unroll
        for (int b = 0; b < HD / 32; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                uint32_t x = v.s[b][e >> 2][e & 3];
                if (!ok || key + 2 * e >= len) x = 0;
                else if (key + 2 * e + 1 >= len) x &= 0xFFFFu;
                v.s[b][e >> 2][e & 3] = x;
            }
    }
}

// q rows of one 16-row tile as operands; f: 2^-e with max |q 2^e| in [1, 2),
// times nothing else (the softmax scale is in q).  Lane (i, g): row i, dims in
// the order of load_k's words.
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
        const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 126);
        const float up = __uint_as_float((unsigned)(127 - e) << 23);
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[s][j] *= up;
            split8<false>(x[s], hi[s], lo[s]);
        }
        f = a.scale_log2 * __uint_as_float((unsigned)(127 + e) << 23);
    }
}

// Scores of a unit against a 16-row tile: c[t][r] for key 16 g + 4 t + r.
template <int HD, bool F16>
__device__ __forceinline__ void scores(const KRaw<HD>& k, const h8v* hi, const h8v* lo, f4v c[4]) {
    constexpr int KS = HD / 32;
#pragma unroll
    for (int t = 0; t < 4; t++) {
        c[t] = f4v{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const uint32_t sc = k.s[t][HD == 256 ? s >> 2 : 0];
            const h8v w = k_operand(k.w[t][s], as_h2(sc | sc << 16));
            c[t] = mfma(w, hi[s], c[t]);
            if constexpr (!F16) c[t] = mfma(w, lo[s], c[t]);
        }
    }
}

// Softmax state of a lane's query row.
struct Row {
    int pos, lo;    // keys j <= pos, and j >= lo or j < sink
    float f;        // raw score -> exponent of 2
    float m, nfm;   // reference score, PBIAS - f m
    float l;        // this lane group's part of the sum
};

__device__ __forceinline__ void row_init(const Kv4AttnArgs& a, const Tile& t, int r, float f, Row& w) {
    const long pos = t.pos0 + r / a.group;
    w.pos = (int)max(pos, -1L);
    w.lo = a.window > 0 ? (int)max(0L, pos - a.window + 1) : 0;
    w.f = f;
    w.m = -__builtin_inff();
    w.nfm = 0.0f;
    w.l = t.bad ? __builtin_nanf("") : 0.0f;
}

template <bool MASK>
__device__ __forceinline__ bool row_max(const Row& w, int key, int sink, f4v c[4], float& top) {
    top = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if constexpr (MASK) {
                const int j = key + 4 * t + r;
                const bool see = j <= w.pos && (j >= w.lo || j < sink);
                c[t][r] = see ? c[t][r] : -__builtin_inff();
            }
            top = fmaxf(top, c[t][r]);
        }
    top = rows_reduce(top, OpMax{});
    return top > w.m && !(w.f * (top - w.m) <= PSLACK);
}

// A block's four waves hold the same rows over different keys: their sums to
// one.  acc[m]: O^T tiles, dims 16 m + 4 g + r of row i.  Wave w ends with the
// tiles m = 4 c + w of every chunk c, in out[c].
template <int HD>
__device__ __forceinline__ void join_waves(f4v* acc, float nfm, float& l, float* nfm_all, float* smem, f4v* out) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15;
    l = rows_sum(l);
    float* s_n = smem;        // [4][16]
    float* s_l = smem + 64;   // [4][16]
    f4v* s_o = (f4v*)(smem + 128);  // [4 waves][4 tiles][64 lanes]
    __syncthreads();
    if (lane < 16) {
        s_n[wave * 16 + i] = l != 0.0f ? nfm : __builtin_inff();  // no key seen: no weight (NaN counts as seen)
        s_l[wave * 16 + i] = l;
    }
    __syncthreads();
    float n = s_n[i];
#pragma unroll
    for (int w = 1; w < 4; w++) n = fminf(n, s_n[w * 16 + i]);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float x = s_l[w * 16 + i];
        if (x != 0.0f) sum += x * exp2f(n - s_n[w * 16 + i]);
    }
    const float mine = l != 0.0f ? exp2f(n - nfm) : 0.0f;
    l = sum;
    *nfm_all = n;
#pragma unroll
    for (int c = 0; c < HD / 64; c++) {
#pragma unroll
        for (int m = 0; m < 4; m++) s_o[(wave * 4 + m) * 64 + lane] = acc[4 * c + m] * mine;
        __syncthreads();
        f4v o = s_o[wave * 64 + lane];
#pragma unroll
        for (int w = 1; w < 4; w++) o += s_o[(w * 4 + wave) * 64 + lane];
        out[c] = o;
        __syncthreads();
    }
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

// Few rows (decode, drafts): a block's waves take the units of its split in
// turn, 16 rows each.
template <int HD, bool F16>
__device__ __forceinline__ void stream_tile(const Kv4AttnArgs& a, const Tile& t, const int* table, int split, float* smem) {
    constexpr int KS = HD / 32, MT = HD / 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int last = min(t.r0 + 15, t.rows - 1);
    const Units u = units_of(t.pos0 + t.r0 / a.group, t.pos0 + last / a.group, a.window, a.sink);
    const int u_lo = (int)((long)u.n * split / a.n_split), u_hi = (int)((long)u.n * (split + 1) / a.n_split);
    const int r = min(t.r0 + i, last);  // rows past the last repeat it
    h8v qh[KS], ql[F16 ? 1 : KS];
    float f;
    load_q<HD, F16>(a, t, r, qh, ql, f);
    Row w;
    row_init(a, t, r, f, w);
    const int full_hi = (int)(t.pos0 + t.r0 / a.group);  // every row sees keys up to here ..
    const int full_lo = a.window > 0 ? (int)max(0L, t.pos0 + last / a.group - a.window + 1) : 0;  // .. from here on
    f4v acc[MT];
#pragma unroll
    for (int m = 0; m < MT; m++) acc[m] = f4v{0, 0, 0, 0};
    for (int n = u_lo + wave; n < u_hi; n += 4) {
        const int unit = u.at(n), key0 = unit * UNIT;
        KRaw<HD> k;
        load_k<HD>(a, table, t.head, unit, k);
        VRaw<HD> v;
        load_v<HD>(a, table, t.head, unit, t.len, v);
        f4v c[4];
        scores<HD, F16>(k, qh, ql, c);
        float top;
        const bool whole = key0 + UNIT - 1 <= full_hi && key0 >= full_lo;
        const bool grow = whole ? row_max<false>(w, key0 + 16 * g, a.sink, c, top) : row_max<true>(w, key0 + 16 * g, a.sink, c, top);
        if (__any(grow)) {
            const float nfm = grow ? PBIAS - w.f * top : w.nfm;
            const float keep = !grow ? 1.0f : w.m == -__builtin_inff() ? 0.0f : exp2f(nfm - w.nfm);
            if (grow) w.m = top;
            w.nfm = nfm;
            w.l *= keep;
#pragma unroll
            for (int m = 0; m < MT; m++) acc[m] *= keep;
        }
        float p[2][8];
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(c[x][y], w.f, w.nfm));
                p[x >> 1][(x & 1) * 4 + y] = e;
                w.l += e;
            }
        h8v ph[2], pl[2];
        split8<F16>(p[0], ph[0], pl[0]);
        split8<F16>(p[1], ph[1], pl[1]);
#pragma unroll
        for (int b = 0; b < HD / 32; b++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
                h8v lo, hi;
                const uint32_t sc[4] = {v.s[b][s].x, v.s[b][s].y, v.s[b][s].z, v.s[b][s].w};
                v_operands(s ? v.w[b].z : v.w[b].x, s ? v.w[b].w : v.w[b].y, sc, lo, hi);
                acc[2 * b] = mfma(lo, ph[s], acc[2 * b]);
                acc[2 * b + 1] = mfma(hi, ph[s], acc[2 * b + 1]);
                if constexpr (!F16) {
                    acc[2 * b] = mfma(lo, pl[s], acc[2 * b]);
                    acc[2 * b + 1] = mfma(hi, pl[s], acc[2 * b + 1]);
                }
            }
    }
    float l = w.l, nfm;
    f4v o[HD / 64];
    join_waves<HD>(acc, w.nfm, l, &nfm, smem, o);
    if (t.r0 + i > last) return;
    const int tok = t.q0 + r / a.group, h = t.head * a.group + r % a.group;
    if (a.n_split == 1) {
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        const long at = (long)tok * a.out_stride + (long)h * HD;
#pragma unroll
        for (int c = 0; c < HD / 64; c++) store4<F16>(a, at + 16 * (4 * c + wave) + 4 * g, o[c] * inv);
    } else {
        float* row = a.part + (((long)tok * a.n_head + h) * a.n_split + split) * (HD + 4);
#pragma unroll
        for (int c = 0; c < HD / 64; c++) *(f4v*)(row + 16 * (4 * c + wave) + 4 * g) = o[c];
        if (wave == 0 && g == 0) *(f4v*)(row + HD) = f4v{l, nfm, 0, 0};
    }
}

template <int HD, bool F16>
__global__ __launch_bounds__(256) void k_kv4_attn(Kv4AttnArgs a) {
    __shared__ __align__(16) float smem[128 + 4 * 4 * 64 * 4];
    unsigned id = blockIdx.x;
    const int split = id % a.n_split;
    id /= a.n_split;
    const int head = id % a.c.n_kv;
    id /= a.c.n_kv;
    const int tile = id % a.tiles, seq = id / a.tiles;
    Tile t;
    seq_of(a, seq, head, t);
    const int* table = a.block_table + (long)seq * a.max_blocks;
    // (more tiles than the caller's max_q said: the blocks go round again)
    for (t.r0 = tile * 16; t.r0 < t.rows; t.r0 += a.tiles * 16) stream_tile<HD, F16>(a, t, table, split, smem);
}

// Splits of a row to one.  A row's lanes: HD / 4, four dims each.
template <int HD, bool F16>
__global__ __launch_bounds__(256) void k_kv4_join(Kv4AttnArgs a) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR;
    const long row = (long)blockIdx.x * RPB + threadIdx.x / LPR;
    if (row >= (long)a.n_tok * a.n_head) return;
    const int tok = (int)(row / a.n_head), h = (int)(row - (long)tok * a.n_head);
    if (tok < a.cu_q[0] || tok >= a.cu_q[a.n_seq]) return;  // rows of no sequence stay as they are
    const int l = threadIdx.x % LPR;
    const float* p = a.part + row * a.n_split * (HD + 4);
    float n = __builtin_inff();
    for (int s = 0; s < a.n_split; s++)
        if (p[s * (HD + 4) + HD] != 0.0f) n = fminf(n, p[s * (HD + 4) + HD + 1]);
    float sum = 0.0f;
    f4v o = {0, 0, 0, 0};
    for (int s = 0; s < a.n_split; s++) {
        const float* q = p + s * (HD + 4);
        if (q[HD] == 0.0f) continue;
        const float w = exp2f(n - q[HD + 1]);
        sum += w * q[HD];
        o += *(const f4v*)(q + 4 * l) * w;
    }
    const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
    store4<F16>(a, (long)tok * a.out_stride + (long)h * HD + 4 * l, o * inv);
}

template <int HD, bool F16>
int attn_run(const Kv4AttnArgs& a, const Kv4AttnPlan& p, hipStream_t st) {
    const long grid = (long)a.n_seq * p.tiles * a.c.n_kv * p.n_split;
    if (grid > 0x7FFFFFFFL) return -1;
    hipLaunchKernelGGL((k_kv4_attn<HD, F16>), dim3((unsigned)grid), dim3(256), 0, st, a);
    if (p.n_split > 1) {
        constexpr int RPB = 256 / (HD / 4);
        const long rows = (long)a.n_tok * a.n_head;
        hipLaunchKernelGGL((k_kv4_join<HD, F16>), dim3((unsigned)((rows + RPB - 1) / RPB)), dim3(256), 0, st, a);
    }
    return 0;
}

}  // namespace

Kv4AttnPlan kv4_attn_plan(int hd, bool f16, int n_seq, int n_tok, int n_head, int n_kv, int max_q, long max_len,
                          int window, int sink, int cus) {
    Kv4AttnPlan p = {};
    (void)f16;
    const int group = n_head / n_kv;
    p.rows = 16;
    p.tiles = (int)(((long)max_q * group + p.rows - 1) / p.rows);
    long keys = max_len;
    if (window > 0) keys = min(keys, (long)window + max_q + sink);
    const long units = max(1L, (keys + UNIT - 1) / UNIT), base = (long)n_seq * p.tiles * n_kv;
    const long want = 3L * cus;
    p.n_split = (int)max(1L, min(min((want + base - 1) / base, (units + 3) / 4), 128L));
    p.work = p.n_split > 1 ? (size_t)n_tok * n_head * p.n_split * (hd + 4) * sizeof(float) : 0;
    return p;
}

int kv4_attn(Kv4AttnArgs a, bool f16, const Kv4AttnPlan& p, hipStream_t st) {
    a.tiles = p.tiles;
    a.n_split = p.n_split;
    switch (a.c.hd) {
    case 64: return f16 ? attn_run<64, true>(a, p, st) : attn_run<64, false>(a, p, st);
    case 128: return f16 ? attn_run<128, true>(a, p, st) : attn_run<128, false>(a, p, st);
    case 256: return f16 ? attn_run<256, true>(a, p, st) : attn_run<256, false>(a, p, st);
    }
    return -1;
}

}  // namespace draco
