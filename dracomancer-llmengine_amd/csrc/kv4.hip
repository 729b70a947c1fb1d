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
// rounding to fp32 (q: to its type): an fp32 sum could round differently on
// another machine and move a value over a code's border.
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

// f16 nearest to x (one rounding from 64 bits: the rotated q).
__device__ __forceinline__ uint16_t d2h(double x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }

// The four dims d .. d + 3 of a rotated row in 64 bits.  Dims from rot on pass
// through; a position outside the table makes its pairs NaN.
template <bool F16, bool HALVES>
__device__ __forceinline__ void rotate4(const Kv4AppendArgs& a, const void* row, long at, int d, long t, double y[4]) {
    const float4 x = load4<F16>(row, at + d);
    const float xv[4] = {x.x, x.y, x.z, x.w};
    if (d >= a.rot) {
        for (int i = 0; i < 4; i++) y[i] = xv[i];
        return;
    }
    const int half = a.rot >> 1;
    float pv[4];  // the pairs' other halves
    if constexpr (HALVES) {
        const float4 p = load4<F16>(row, at + (d < half ? d + half : d - half));
        pv[0] = p.x, pv[1] = p.y, pv[2] = p.z, pv[3] = p.w;
    } else {
        pv[0] = xv[1], pv[1] = xv[0], pv[2] = xv[3], pv[3] = xv[2];
    }
    for (int i = 0; i < 4; i++) {
        const int pair = HALVES ? (d < half ? d + i : d + i - half) : (d + i) >> 1;
        const bool second = HALVES ? d >= half : (i & 1);
        const int p = a.pos[(long)a.axis[pair] * a.pos_stride + t];
        const bool ok = (unsigned)p < (unsigned)a.table_rows;
        const float2 cs = *(const float2*)(a.table + 2 * ((long)(ok ? p : 0) * half + pair));
        const double c = ok ? cs.x : __builtin_nanf(""), s = ok ? cs.y : __builtin_nanf("");
        y[i] = second ? (double)pv[i] * s + (double)xv[i] * c : (double)xv[i] * c - (double)pv[i] * s;
    }
}

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

// One token and head per group of HD / 4 lanes, four dims a lane.  Group h of
// a token: q heads first (rotated into q_out), then KV heads (k rotated and
// quantized, v quantized).  A K or V row that is not finite marks the row:
// NaN in every K scale, 0 in every V scale (the attention's scores carry the
// NaN to the rows that see the token, and to no others).
template <int HD, bool F16, bool HALVES>
__global__ __launch_bounds__(256) void k_kv4_append(Kv4AppendArgs a) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR;
    const int l = threadIdx.x % LPR, d = 4 * l;
    const int rows = a.n_head + a.c.n_kv;
    const long id = (long)blockIdx.x * RPB + threadIdx.x / LPR;
    const long t = id / rows;
    if (t >= a.n_tok) return;
    const int h = (int)(id - t * rows);
    const int slot = a.slot[t];
    const int page = slot >> a.c.ps_shift;
    if (slot < 0 || page >= a.c.n_pages) return;
    double y[4];
    if (h < a.n_head) {
        rotate4<F16, HALVES>(a, a.q, t * a.q_stride + (long)h * HD, d, t, y);
        const long o = t * a.q_out_stride + (long)h * HD + d;
        if constexpr (F16) {
            uint2 u;
            u.x = d2h(y[0]) | (uint32_t)d2h(y[1]) << 16;
            u.y = d2h(y[2]) | (uint32_t)d2h(y[3]) << 16;
            *(uint2*)((uint16_t*)a.q_out + o) = u;
        } else {
            *(float4*)((float*)a.q_out + o) = make_float4((float)y[0], (float)y[1], (float)y[2], (float)y[3]);
        }
        return;
    }
    const int g = h - a.n_head;
    rotate4<F16, HALVES>(a, a.k, t * a.k_stride + (long)g * HD, d, t, y);
    const float4 v4 = load4<F16>(a.v, t * a.v_stride + (long)g * HD + d);
    const float x[2][4] = {{(float)y[0], (float)y[1], (float)y[2], (float)y[3]}, {v4.x, v4.y, v4.z, v4.w}};
    // largest magnitude of a block as bits: NaN and infinity rank above every number
    uint32_t top[2];
    for (int r = 0; r < 2; r++) {
        uint32_t m = 0;
        for (int i = 0; i < 4; i++) m = max(m, __float_as_uint(x[r][i]) & 0x7FFFFFFFu);
        top[r] = group_reduce<8>(m, [](uint32_t p, uint32_t q) { return p > q ? p : q; });
    }
    const uint32_t any = group_reduce<LPR>(max(top[0], top[1]), [](uint32_t p, uint32_t q) { return p > q ? p : q; });
    const bool bad = any >= 0x7F800000u;
    uint16_t code[2], sc[2];
    uint32_t codes[2][4];
    for (int r = 0; r < 2; r++) {
        const float s = bad ? 0.0f : block_scale(__uint_as_float(top[r]));
        for (int i = 0; i < 4; i++) codes[r][i] = bad ? 0u : code_of(x[r][i], s);
        sc[r] = __builtin_bit_cast(uint16_t, (_Float16)s);
        code[r] = (uint16_t)(codes[r][0] | codes[r][1] << 4 | codes[r][2] << 8 | codes[r][3] << 12);
    }
    if (bad) sc[0] = 0x7E00;
    const int ps = 1 << a.c.ps_shift, off = slot & (ps - 1), b = l >> 3;
    uint8_t* base = a.c.data + (long)page * a.c.page_bytes + (long)g * a.c.head_bytes;
    *(uint16_t*)(base + (long)off * (HD / 2) + 2 * l) = code[0];
    // V bytes: dim a with dim a + 16 of the block, from the lane four further
    uint8_t* vrow = base + ps * (HD / 2) + (off >> 4) * (HD * 8) + (off & 15);
    const uint32_t part = (uint32_t)__shfl((int)code[1], (threadIdx.x & 63) ^ 4);
    const uint32_t lo = (l & 4) ? part : code[1], hi = (l & 4) ? code[1] : part;
    const int first = (l & 4) ? 2 : 0;  // lanes 0-3 of a block write a = 4i, 4i + 1; lanes 4-7 a = 4i + 2, 4i + 3
    for (int i = first; i < first + 2; i++) {
        const uint32_t byte = ((lo >> (4 * i)) & 15) | ((hi >> (4 * i)) & 15) << 4;
        vrow[(b * 16 + 4 * (l & 3) + i) * 16] = (uint8_t)byte;
    }
    if ((l & 7) == 0) {
        uint8_t* ksc = base + ps * HD;
        ((uint16_t*)ksc)[off * (HD / 32) + b] = sc[0];
        ((uint16_t*)(ksc + ps * (HD / 16)))[((off >> 4) * (HD / 32) + b) * 16 + (off & 15)] = sc[1];
    }
}

__device__ __forceinline__ float value_of(uint32_t c, float s) {
    const uint32_t m = c & 7;
    const float v = m < 2 ? 0.5f * (float)m : (float)(2 + (m & 1)) * (float)(1 << (m >> 1)) * 0.25f;
    return (c & 8) ? -v * s : v * s;
}

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
    const uint8_t* base = c.data + (long)page * c.page_bytes + (long)g * c.head_bytes;
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
int append_hd(const Kv4AppendArgs& a, bool f16, bool halves, hipStream_t st) {
    constexpr int RPB = 256 / (HD / 4);
    const long rows = (long)a.n_tok * (a.n_head + a.c.n_kv);
    const long grid = (rows + RPB - 1) / RPB;
    if (grid > 0x7FFFFFFFL) return -1;
    const dim3 gr((unsigned)grid), bl(256);
    if (f16 && halves) hipLaunchKernelGGL((k_kv4_append<HD, true, true>), gr, bl, 0, st, a);
    else if (f16) hipLaunchKernelGGL((k_kv4_append<HD, true, false>), gr, bl, 0, st, a);
    else if (halves) hipLaunchKernelGGL((k_kv4_append<HD, false, true>), gr, bl, 0, st, a);
    else hipLaunchKernelGGL((k_kv4_append<HD, false, false>), gr, bl, 0, st, a);
    return 0;
}

}  // namespace

int kv4_append(const Kv4AppendArgs& a, bool f16, bool halves, hipStream_t st) {
    switch (a.c.hd) {
    case 64: return append_hd<64>(a, f16, halves, st);
    case 128: return append_hd<128>(a, f16, halves, st);
    case 256: return append_hd<256>(a, f16, halves, st);
    }
    return -1;
}

int kv4_read(const Kv4View& c, const int* slot, int n, float* k, float* v, hipStream_t st) {
    const int rpb = 256 / (c.hd / 4);
    const long grid = ((long)n * c.n_kv + rpb - 1) / rpb;
    if (grid > 0x7FFFFFFFL) return -1;
    const dim3 gr((unsigned)grid), bl(256);
    switch (c.hd) {
    case 64: hipLaunchKernelGGL(k_kv4_read<64>, gr, bl, 0, st, c, slot, n, k, v); return 0;
    case 128: hipLaunchKernelGGL(k_kv4_read<128>, gr, bl, 0, st, c, slot, n, k, v); return 0;
    case 256: hipLaunchKernelGGL(k_kv4_read<256>, gr, bl, 0, st, c, slot, n, k, v); return 0;
    }
    return -1;
}

}  // namespace draco
