// kv4.hip -- rows into and out of the 4-bit pages (kv4.h): rotary positions
// on several axes, quantization, and the values a page stands for.
//
// Quantization of a block of 32 values: a = max |x|, scale = a / 6 rounded to
// 9 significant bits (and a multiple of 2^-23, at most 10912 so that 6 * scale
// stays an f16 number), code = the E2M1 number nearest to x / scale, ties to
// the even code.  Every decision is made exactly: a midpoint of two codes
// times the scale has at most 4 + 9 bits, so x is compared with an exact fp32
// product and nothing is divided.
//
// Rotation: a c - b s and a s + b c with products and sum in 64 bits and one
// rounding to fp32 (f16 q: another to its type): an fp32 sum could round
// differently on another machine and move a value over a code's border.
//
// The append is HBM bound where it is long: 8192 tokens of 32 / 4 heads of 128,
// fp32, 307 MB in 64 us (4.8 TB/s, a copy's rate).  Short ones wait for slot,
// position and angles one after the other: 1 token 4.2 us, 1037 of 16 / 2 heads
// of 256 with three axes 9.3.
#include <hip/hip_runtime.h>

#include "dev_common.h"
#include "kv4.h"

namespace draco {
namespace {

template <bool F16>
__device__ __forceinline__ float4 load4(const void* p, long i) {
    if constexpr (F16) {
        const uint2 u = *(const uint2*)((const uint16_t*)p + i);
        return make_float4(h2f(u.x & 0xFFFF), h2f(u.x >> 16), h2f(u.y & 0xFFFF), h2f(u.y >> 16));
    } else {
        return ld4((const float*)p + i);
    }
}

// f16 by way of fp32, whose rounding moves one value in 2^13 to the other side
// of a tie (a conversion from 64 bits is a dozen instructions).
__device__ __forceinline__ uint16_t d2h(double x) { return __builtin_bit_cast(uint16_t, (_Float16)(float)x); }

// a / 6 to 9 significant bits, a multiple of 2^-23, at most 10912: exact
// comparisons decide where the fp32 quotient is a midpoint.
__device__ __forceinline__ float block_scale(float amax) {
    const float t = amax / 6.0f;
    // candidates below and above t: multiples of the step of t's binade
    const int e = max((int)(__float_as_uint(t) >> 23) - 127 - 8, -23);
    const float step = __uint_as_float((unsigned)(e + 127) << 23), inv = __uint_as_float((unsigned)(127 - e) << 23);
    const float k = floorf(t * inv);  // exact: a power of two, at most 2^9
    const float mid6 = (k + 0.5f) * step * 6.0f;  // exact: 11 bits times 3
    const bool up = amax > mid6 || (amax == mid6 && ((int)k & 1));
    return fminf((up ? k + 1.0f : k) * step, 10912.0f);
}

// Code of x at scale s: the number of midpoints below |x| (or on it, where the
// upper code is the even one), and the sign.
__device__ __forceinline__ uint32_t code_of(float x, float s) {
    const float v = fabsf(x);
    uint32_t c = 0;
    c += v > 0.25f * s;
    c += v >= 0.75f * s;
    c += v > 1.25f * s;
    c += v >= 1.75f * s;
    c += v > 2.5f * s;
    c += v >= 3.5f * s;
    c += v > 5.0f * s;
    if (!(s > 0.0f)) c = 0;
    return c | (x < 0.0f ? 8u : 0u);
}

// A lane's cos and sin of the N pairs from `pair`, in 64 bits; NaN for a
// position outside the table.
template <int N>
__device__ __forceinline__ void angles(const Kv4AppendArgs& a, long t, int pair, double c[N], double s[N]) {
    const int half = a.rot >> 1;
    float2 cs[N];
    bool ok[N];
    // the pairs' axes, two bits each, 16 pairs a word (selected, not loaded: one round trip less)
    uint32_t ax = a.axis[0];
    if (a.n_axes > 1) {
#pragma unroll
        for (int w = 1; w < 8; w++) ax = pair >> 4 == w ? a.axis[w] : ax;
        ax >>= 2 * (pair & 15);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int p = a.pos[(long)((ax >> 2 * i) & 3) * a.pos_stride + t];
        ok[i] = (unsigned)p < (unsigned)a.table_rows;
        cs[i] = *(const float2*)(a.table + 2 * ((long)(ok[i] ? p : 0) * half + pair + i));
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        c[i] = ok[i] ? cs[i].x : __builtin_nanf("");
        s[i] = ok[i] ? cs[i].y : __builtin_nanf("");
    }
}

template <bool F16>
__device__ __forceinline__ void store4(void* p, long i, const double y[4]) {
    if constexpr (F16) {
        uint2 u;
        u.x = d2h(y[0]) | (uint32_t)d2h(y[1]) << 16;
        u.y = d2h(y[2]) | (uint32_t)d2h(y[3]) << 16;
        *(uint2*)((uint16_t*)p + i) = u;
    } else {
        *(float4*)((float*)p + i) = make_float4((float)y[0], (float)y[1], (float)y[2], (float)y[3]);
    }
}

// q heads of one token: a lane has the eight dims of four pairs (halves: dims
// d .. and d + rot / 2 ..; consecutive: d .. d + 7; behind rot, d .. d + 7 as
// they are), keeps their angles and goes through the heads, QU rows in flight.
constexpr int QU = 2;
template <int HD, bool F16, bool HALVES>
__device__ __forceinline__ void append_q(const Kv4AppendArgs& a, long block) {
    constexpr int LPR = HD / 8, RPB = 256 / LPR;
    const int per = (a.n_head + RPB * QU - 1) / (RPB * QU);
    const long t = block / per;
    const int h0 = (int)(block - t * per) * RPB * QU + threadIdx.x / LPR, j = threadIdx.x % LPR;
    const int slot = a.slot[t];  // (looked at behind the loads: nothing waits for it)
    const bool turn = 8 * j < a.rot;
    const int d0 = HALVES && turn ? 4 * j : 8 * j, d1 = HALVES && turn ? d0 + (a.rot >> 1) : d0 + 4;
    float4 x[QU], y[QU];
#pragma unroll
    for (int u = 0; u < QU; u++) {
        const long at = t * a.q_stride + (long)min(h0 + u * RPB, a.n_head - 1) * HD;
        x[u] = load4<F16>(a.q, at + d0);
        y[u] = load4<F16>(a.q, at + d1);
    }
    double c[4] = {1, 1, 1, 1}, s[4] = {0, 0, 0, 0};
    if (turn) angles<4>(a, t, 4 * j, c, s);
    if (slot < 0 || slot >> a.c.ps_shift >= a.c.n_pages) return;
#pragma unroll
    for (int u = 0; u < QU; u++) {
        const int h = h0 + u * RPB;
        const float v[8] = {x[u].x, x[u].y, x[u].z, x[u].w, y[u].x, y[u].y, y[u].z, y[u].w};
        double o[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int p0 = HALVES ? i : 2 * i, p1 = HALVES ? i + 4 : 2 * i + 1;
            const double e0 = v[turn ? p0 : i], e1 = v[turn ? p1 : i + 4];
            o[turn ? p0 : i] = turn ? e0 * c[i] - e1 * s[i] : e0;
            o[turn ? p1 : i + 4] = turn ? e0 * s[i] + e1 * c[i] : e1;
        }
        if (h < a.n_head) {
            const long at = t * a.q_out_stride + (long)h * HD;
            store4<F16>(a.q_out, at + d0, o);
            store4<F16>(a.q_out, at + d1, o + 4);
        }
    }
}

// 16 tokens of one KV head (their V bytes share lines, so they share a block;
// a short call spreads them, one pass of 256 / LPR rows a block, as each pass
// waits out its loads: 1037 tokens at head dim 256 15 -> 9 us), HD / 4 lanes a
// row, four dims a lane.  A K or V row that is not finite marks
// the row: NaN in every K scale, 0 in every V scale (the attention's scores
// carry the NaN to the rows that see the token, and to no others).
constexpr int KV_TOKENS = 16;
template <int HD, bool F16, bool HALVES>
__device__ __forceinline__ void append_kv(const Kv4AppendArgs& a, long block) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR;
    const int l = threadIdx.x % LPR, d = 4 * l, b = l >> 3;
    const long group = block / a.c.n_kv;
    const int g = (int)(block - group * a.c.n_kv);
    const int half = a.rot >> 1;
    const bool turn = d < a.rot;
    const int pair = HALVES ? (d < half ? d : d - half) : d >> 1;
    constexpr int NP = HALVES ? 4 : 2;  // pairs of a lane
    for (int k = 0; k < a.kv_passes; k++) {
        const long t = (group * a.kv_passes + k) * RPB + threadIdx.x / LPR;
        if (t >= a.n_tok) return;  // (whole groups of LPR lanes)
        const int slot = a.slot[t], page = slot >> a.c.ps_shift;
        const long at = t * a.k_stride + (long)g * HD;
        const float4 k4 = load4<F16>(a.k, at + d);
        const float4 v4 = load4<F16>(a.v, t * a.v_stride + (long)g * HD + d);
        float x[2][4] = {{k4.x, k4.y, k4.z, k4.w}, {v4.x, v4.y, v4.z, v4.w}};
        if (turn) {
            float4 o4;
            if constexpr (HALVES) o4 = load4<F16>(a.k, at + (d < half ? d + half : d - half));
            double c[NP], s[NP];
            angles<NP>(a, t, pair, c, s);
            if constexpr (HALVES) {
                const float o[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const double e = x[0][i], p = o[i];
                    x[0][i] = (float)(d < half ? e * c[i] - p * s[i] : p * s[i] + e * c[i]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const double e0 = x[0][2 * i], e1 = x[0][2 * i + 1];
                    x[0][2 * i] = (float)(e0 * c[i] - e1 * s[i]);
                    x[0][2 * i + 1] = (float)(e0 * s[i] + e1 * c[i]);
                }
            }
        }
        if (slot < 0 || page >= a.c.n_pages) continue;
        // largest magnitude of a block as bits: NaN and infinity rank above every number
        const auto larger = [](uint32_t p, uint32_t q) { return p > q ? p : q; };
        uint32_t top[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(x[r][i]) & 0x7FFFFFFFu);
            top[r] = group_reduce<8>(m, larger);
        }
        const bool bad = group_reduce<LPR>(max(top[0], top[1]), larger) >= 0x7F800000u;
        uint32_t code[2];
        uint16_t sc[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const float s = bad ? 0.0f : block_scale(__uint_as_float(top[r]));
            code[r] = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) code[r] |= (bad ? 0u : code_of(x[r][i], s)) << (4 * i);
            sc[r] = __builtin_bit_cast(uint16_t, (_Float16)s);
        }
        if (bad) sc[0] = 0x7E00;
        const int ps = 1 << a.c.ps_shift, off = slot & (ps - 1);
        uint8_t* base = a.c.data + (unsigned long)(unsigned)page * a.c.page_bytes + (unsigned long)(unsigned)g * (unsigned)a.c.head_bytes;
        *(uint16_t*)(base + (long)off * (HD / 2) + 2 * l) = (uint16_t)code[0];
        // V bytes: dim a with dim a + 16 of the block, from the lane four
        // further; lanes 0-3 of a block write a = 4i, 4i + 1, lanes 4-7 the other two
        const uint32_t part = (uint32_t)__shfl((int)code[1], (threadIdx.x & 63) ^ 4);
        const uint32_t lo = (l & 4) ? part >> 8 : code[1], hi = (l & 4) ? code[1] >> 8 : part;
        uint8_t* vrow = base + ps * (HD / 2) + (off >> 4) * (HD * 8) + (off & 15) + (b * 16 + 4 * (l & 3) + ((l & 4) ? 2 : 0)) * 16;
        vrow[0] = (uint8_t)((lo & 15) | (hi & 15) << 4);
        vrow[16] = (uint8_t)(((lo >> 4) & 15) | ((hi >> 4) & 15) << 4);
        if ((l & 7) == 0) {
            uint8_t* ksc = base + ps * HD;
            ((uint16_t*)ksc)[off * (HD / 32) + b] = sc[0];
            ((uint16_t*)(ksc + ps * (HD / 16)))[((off >> 4) * (HD / 32) + b) * 16 + (off & 15)] = sc[1];
        }
    }
}

// The first kv_blocks blocks write K and V, the others rotate q.
template <int HD, bool F16, bool HALVES>
__global__ __launch_bounds__(256) void k_kv4_append(Kv4AppendArgs a, unsigned kv_blocks) {
    if (blockIdx.x < kv_blocks) append_kv<HD, F16, HALVES>(a, blockIdx.x);
    else append_q<HD, F16, HALVES>(a, (long)blockIdx.x - kv_blocks);
}

__device__ __forceinline__ float value_of(uint32_t c, float s) {
    const uint32_t m = c & 7;
    const float v = m < 2 ? 0.5f * (float)m : (float)(2 + (m & 1)) * (float)(1 << (m >> 1)) * 0.25f;
    return (c & 8) ? -v * s : v * s;
}

// One row of a slot and KV head per HD / 4 lanes: 8192 slots of 4 heads of 128 in
// 12 us, HBM bound on what it writes (38 MB, 3.2 TB/s).
template <int HD>
__global__ __launch_bounds__(256) void k_kv4_read(Kv4View c, const int* slots, int n, float* k, float* v) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR;
    const int l = threadIdx.x % LPR, d = 4 * l, b = l >> 3;
    const long id = (long)blockIdx.x * RPB + threadIdx.x / LPR;
    const long t = id / c.n_kv;
    if (t >= n) return;
    const int g = (int)(id - t * c.n_kv);
    const int slot = slots[t], page = slot >> c.ps_shift;
    if (slot < 0 || page >= c.n_pages) return;
    const int ps = 1 << c.ps_shift, off = slot & (ps - 1);
    const uint8_t* base = c.data + (unsigned long)(unsigned)page * c.page_bytes + (unsigned long)(unsigned)g * (unsigned)c.head_bytes;
    const uint8_t* ksc = base + ps * HD;
    const float sk = h2f(((const uint16_t*)ksc)[off * (HD / 32) + b]);
    float sv = h2f(((const uint16_t*)(ksc + ps * (HD / 16)))[((off >> 4) * (HD / 32) + b) * 16 + (off & 15)]);
    if (sk != sk) sv = sk;  // a row that was not finite
    const long o = (t * c.n_kv + g) * HD + d;
    const uint32_t w = *(const uint16_t*)(base + (long)off * (HD / 2) + 2 * l);
    *(float4*)(k + o) = make_float4(value_of(w & 15, sk), value_of((w >> 4) & 15, sk), value_of((w >> 8) & 15, sk),
                                    value_of(w >> 12, sk));
    const uint8_t* vrow = base + ps * (HD / 2) + (off >> 4) * (HD * 8) + (off & 15) + (b * 16 + 4 * (l & 3)) * 16;
    const int sh = (l & 4) ? 4 : 0;
    *(float4*)(v + o) = make_float4(value_of((vrow[0] >> sh) & 15, sv), value_of((vrow[16] >> sh) & 15, sv),
                                    value_of((vrow[32] >> sh) & 15, sv), value_of((vrow[48] >> sh) & 15, sv));
}

template <int HD>
int append_hd(const Kv4AppendArgs& a, const Kv4AppendGrid& g, bool f16, bool halves, hipStream_t st) {
    const dim3 gr((unsigned)g.blocks), bl(256);
    const unsigned n = (unsigned)g.kv;
    if (f16 && halves) hipLaunchKernelGGL((k_kv4_append<HD, true, true>), gr, bl, 0, st, a, n);
    else if (f16) hipLaunchKernelGGL((k_kv4_append<HD, true, false>), gr, bl, 0, st, a, n);
    else if (halves) hipLaunchKernelGGL((k_kv4_append<HD, false, true>), gr, bl, 0, st, a, n);
    else hipLaunchKernelGGL((k_kv4_append<HD, false, false>), gr, bl, 0, st, a, n);
    return 0;
}

}  // namespace

Kv4AppendGrid kv4_append_grid(const Kv4AppendArgs& a) {
    const int rpb = 256 / (a.c.hd / 8) * QU;  // q heads a block
    const int kpb = 256 / (a.c.hd / 4);       // K and V rows a pass
    Kv4AppendGrid g;
    g.kv_passes = (long)a.n_tok / KV_TOKENS * a.c.n_kv >= 1024 ? KV_TOKENS / kpb : 1;
    const int per = kpb * g.kv_passes;
    g.kv = ((long)a.n_tok + per - 1) / per * a.c.n_kv;
    g.blocks = g.kv + (long)a.n_tok * ((a.n_head + rpb - 1) / rpb);
    return g;
}

int kv4_append(Kv4AppendArgs a, bool f16, bool halves, hipStream_t st) {
    const Kv4AppendGrid g = kv4_append_grid(a);
    if (g.blocks > KV4_MAX_GRID) return -1;
    a.kv_passes = g.kv_passes;
    switch (a.c.hd) {
    case 64: return append_hd<64>(a, g, f16, halves, st);
    case 128: return append_hd<128>(a, g, f16, halves, st);
    case 256: return append_hd<256>(a, g, f16, halves, st);
    }
    return -1;
}

long kv4_read_grid(const Kv4View& c, int n) {
    const int rpb = 256 / (c.hd / 4);
    return ((long)n * c.n_kv + rpb - 1) / rpb;
}

int kv4_read(const Kv4View& c, const int* slot, int n, float* k, float* v, hipStream_t st) {
    const long grid = kv4_read_grid(c, n);
    if (grid > KV4_MAX_GRID) return -1;
    const dim3 gr((unsigned)grid), bl(256);
    switch (c.hd) {
    case 64: hipLaunchKernelGGL(k_kv4_read<64>, gr, bl, 0, st, c, slot, n, k, v); return 0;
    case 128: hipLaunchKernelGGL(k_kv4_read<128>, gr, bl, 0, st, c, slot, n, k, v); return 0;
    case 256: hipLaunchKernelGGL(k_kv4_read<256>, gr, bl, 0, st, c, slot, n, k, v); return 0;
    }
    return -1;
}

}  // namespace draco
