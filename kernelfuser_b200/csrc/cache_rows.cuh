// Rows into a paged key-value cache and back.
//
// append: K row x -> rotate(x * rsqrt(mean x^2 + eps) * gamma) at the row's own position, V row as it is, both written
// to row (position % page_size) of page table[b][position / page_size].
// read:   rows 0 .. length-1 of every sequence as contiguous [B, H, S, D], zeros behind them.
// Everything between the input's 16 bits and the cache's type is done in 32 bits and rounded once.  An 8-bit cache
// holds a row as e4m3 values times ONE power of two, kept as its exponent byte (e8m0): the smallest that brings the
// row's largest magnitude to at most 448.  A power of two costs no precision that e4m3 has (only its subnormals begin
// up to a factor of two earlier) and makes scaling exact, so that each value is rounded once and reading back to 16
// bits is exact.  (Magnitudes above 448 * 2^119 = 2.98e38 become that.)  A row whose largest magnitude is not finite gets the NaN scale and reads back as NaN.
#pragma once
#include "ptx.cuh"
#include "rounding.cuh"

namespace kf {

// Codes in the status word.
constexpr int kStatusBadPage = 911;      // a table entry that a sequence's rows need is not a page of the cache
constexpr int kStatusBadLength = 912;    // a position or length outside what the sequence's table entries can hold
constexpr int kStatusBadPosition = 913;  // a position behind the last row of the rotary tables

struct CacheView {
    unsigned char *k, *v;                        // [n_pages, H, page_size, D]; strides in BYTES
    unsigned char *k_scale, *v_scale;            // [n_pages, H, page_size] exponent bytes (8-bit cache)
    long long k_sp, k_sh, k_ss, v_sp, v_sh, v_ss;
    long long ks_sp, ks_sh, vs_sp, vs_sh;
    const int* pages;                            // [B, max_pages]
    long long pages_sb;
    int n_pages, page_size, max_pages;
    int capacity;                                // max_pages * page_size, at most 2^31 - 1
};

__device__ __forceinline__ void report(int* status, int code) { atomicCAS(status, 0, code); }

// Two floats to two e4m3 (in the low 16 bits, `lo` first), to nearest even; values above 448 saturate.
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// The low two e4m3 of x as f16x2 (exact).
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t x) {
    uint32_t r;
    asm("{.reg .b16 t; cvt.u16.u32 t, %1; cvt.rn.f16x2.e4m3x2 %0, t;}" : "=r"(r) : "r"(x));
    return r;
}
// Exponent byte of the power of two for a row whose largest magnitude has the bits `amax`: 448 = 1.75 * 2^8.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
    if (amax >= 0x7f800000u) return 255;  // inf or NaN
    const int e = static_cast<int>(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u);
    return static_cast<uint32_t>(min(max(e, 1), 246));  // (2^119: 448 times the next would not be a number of 16 or 32 bits)
}
// 2^(byte - 127), NaN for 255.
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return __uint_as_float(byte == 255 ? 0x7fffffffu : byte == 0 ? 0x00400000u : byte << 23);
}

struct AppendArgs {
    CacheView c;
    const void *k, *v, *gamma, *cos, *sin;       // gamma, tables: may be null
    long long k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;  // element strides
    const int *start, *counts;                   // counts may be null: all S rows
    int newest;                                  // one row per sequence, at start[b] - 1 where start[b] > 0
    int B, H, S, n_pos, heads_per_group;
    float eps;
    int* status;
};

constexpr int kRowsThreads = 256;

// A row's lane owns columns [8i, 8i+8) and their rotation partners, as in the row-prepare kernel; a group of D/16 lanes
// walks over heads of one position, so that the tables are read once for them.
template <int D, typename T, bool E8>
__global__ void __launch_bounds__(kRowsThreads) append_rows_kernel(const AppendArgs a) {
    constexpr int LPR = D / 16;
    if (*reinterpret_cast<volatile int*>(a.status) != 0) return;
    const int sub = threadIdx.x % LPR;
    const long long task = static_cast<long long>(blockIdx.x) * (kRowsThreads / LPR) + threadIdx.x / LPR;
    const int b = static_cast<int>(task / a.S), s = static_cast<int>(task - static_cast<long long>(b) * a.S);
    bool valid = b < a.B;
    int pos = 0, page = 0, row = 0;
    if (valid) {
        if (a.counts != nullptr) valid = s < a.counts[b];
        long long p = static_cast<long long>(a.start[b]) + s;
        if (a.newest) valid = --p >= 0;
        if (valid && (p < 0 || p >= a.c.capacity)) {
            report(a.status, kStatusBadLength);
            valid = false;
        }
        pos = static_cast<int>(p);
        if (valid && a.cos != nullptr && pos >= a.n_pos) {
            report(a.status, kStatusBadPosition);
            valid = false;
        }
        if (valid) {
            page = a.c.pages[b * a.c.pages_sb + pos / a.c.page_size];
            row = pos % a.c.page_size;
            if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.c.n_pages)) {
                report(a.status, kStatusBadPage);
                valid = false;
            }
        }
    }
    const bool rope = a.cos != nullptr;
    uint4 glo = make_uint4(0, 0, 0, 0), ghi = glo, clo = glo, chi = glo, slo = glo, shi = glo;
    if (a.gamma != nullptr) {
        const uint4* g4 = reinterpret_cast<const uint4*>(a.gamma);
        glo = __ldg(g4 + sub);
        ghi = __ldg(g4 + LPR + sub);
    }
    if (rope && valid) {
        const uint4* c4 = reinterpret_cast<const uint4*>(a.cos) + static_cast<long long>(pos) * (D / 8);
        const uint4* s4 = reinterpret_cast<const uint4*>(a.sin) + static_cast<long long>(pos) * (D / 8);
        clo = __ldg(c4 + sub);
        chi = __ldg(c4 + LPR + sub);
        slo = __ldg(s4 + sub);
        shi = __ldg(s4 + LPR + sub);
    }
    const int h0 = blockIdx.y * a.heads_per_group, h1 = min(h0 + a.heads_per_group, a.H);
    const T* kb = reinterpret_cast<const T*>(a.k) + b * a.k_sb + s * a.k_ss;
    const T* vb = reinterpret_cast<const T*>(a.v) + b * a.v_sb + s * a.v_ss;
    unsigned char* kd = a.c.k + page * a.c.k_sp + row * a.c.k_ss;
    unsigned char* vd = a.c.v + page * a.c.v_sp + row * a.c.v_ss;

    // one row of 16 floats a lane to the cache
    auto put = [&](const float (&x)[16], unsigned char* dst, unsigned char* scale) {
        if constexpr (E8) {
            uint32_t amax = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);  // (a NaN is the largest)
#pragma unroll
            for (int m = LPR / 2; m >= 1; m >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, m));
            const uint32_t e = scale_byte(amax);
            const float f = e == 255 ? 1.f : __uint_as_float((254u - e) << 23);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = pack_e4m3(x[4 * i] * f, x[4 * i + 1] * f) | (pack_e4m3(x[4 * i + 2] * f, x[4 * i + 3] * f) << 16);
            if (valid) {
                reinterpret_cast<uint2*>(dst)[sub] = make_uint2(w[0], w[1]);
                reinterpret_cast<uint2*>(dst)[LPR + sub] = make_uint2(w[2], w[3]);
                if (sub == 0) *scale = static_cast<unsigned char>(e);
            }
        } else if (valid) {
            const float(&lo)[8] = *reinterpret_cast<const float(*)[8]>(&x[0]);
            const float(&hi)[8] = *reinterpret_cast<const float(*)[8]>(&x[8]);
            reinterpret_cast<uint4*>(dst)[sub] = pack8<T>(lo);
            reinterpret_cast<uint4*>(dst)[LPR + sub] = pack8<T>(hi);
        }
    };
    for (int h = h0; h < h1; ++h) {
        uint4 klo = make_uint4(0, 0, 0, 0), khi = klo, vlo = klo, vhi = klo;
        if (valid) {
            const uint4* k4 = reinterpret_cast<const uint4*>(kb + h * a.k_sh);
            const uint4* v4 = reinterpret_cast<const uint4*>(vb + h * a.v_sh);
            klo = __ldcs(k4 + sub);
            khi = __ldcs(k4 + LPR + sub);
            vlo = __ldcs(v4 + sub);
            vhi = __ldcs(v4 + LPR + sub);
        }
        float x[16];
        unpack8<T>(klo, *reinterpret_cast<float(*)[8]>(&x[0]));
        unpack8<T>(khi, *reinterpret_cast<float(*)[8]>(&x[8]));
        if (a.gamma != nullptr) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int m = LPR / 2; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            const float inv = rsqrtf(ss * (1.0f / static_cast<float>(D)) + a.eps);
            float g[16];
            unpack8<T>(glo, *reinterpret_cast<float(*)[8]>(&g[0]));
            unpack8<T>(ghi, *reinterpret_cast<float(*)[8]>(&g[8]));
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = x[i] * inv * g[i];
        }
        if (rope) {
            float cl[8], ch[8], sl[8], sh[8];
            unpack8<T>(clo, cl);
            unpack8<T>(chi, ch);
            unpack8<T>(slo, sl);
            unpack8<T>(shi, sh);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float lo = x[i], hi = x[8 + i];
                x[i] = lo * cl[i] - hi * sl[i];
                x[8 + i] = hi * ch[i] + lo * sh[i];
            }
        }
        const long long ks = E8 ? page * a.c.ks_sp + h * a.c.ks_sh + row : 0;
        const long long vs = E8 ? page * a.c.vs_sp + h * a.c.vs_sh + row : 0;
        if constexpr (!E8) {
            put(x, kd + h * a.c.k_sh, nullptr);
            if (valid) {
                reinterpret_cast<uint4*>(vd + h * a.c.v_sh)[sub] = vlo;
                reinterpret_cast<uint4*>(vd + h * a.c.v_sh)[LPR + sub] = vhi;
            }
        } else {
            put(x, kd + h * a.c.k_sh, a.c.k_scale + ks);
            unpack8<T>(vlo, *reinterpret_cast<float(*)[8]>(&x[0]));
            unpack8<T>(vhi, *reinterpret_cast<float(*)[8]>(&x[8]));
            put(x, vd + h * a.c.v_sh, a.c.v_scale + vs);
        }
    }
}

struct ReadArgs {
    CacheView c;
    void *k, *v;
    long long k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;  // element strides
    const int* lengths;
    int B, H, S;
    int* status;
};

constexpr int kReadUnroll = 4;  // rows of K and of V in flight per lane

// A lane owns 8 columns of a row: one 16-byte store, and a 16-byte (16-bit cache) or 8-byte load.  A CTA takes
// kReadUnroll * (threads / lanes per row) rows of one head of one sequence.
template <int D, typename T, bool E8>
__global__ void __launch_bounds__(kRowsThreads) read_rows_kernel(const ReadArgs a) {
    constexpr int LPR = D / 8, RPB = kRowsThreads / LPR;
    if (*reinterpret_cast<volatile int*>(a.status) != 0) return;
    const int sub = threadIdx.x % LPR, r0 = blockIdx.x * (RPB * kReadUnroll) + threadIdx.x / LPR;
    for (long long bh = blockIdx.y; bh < static_cast<long long>(a.B) * a.H; bh += gridDim.y) {
        const int b = static_cast<int>(bh / a.H), h = static_cast<int>(bh - static_cast<long long>(b) * a.H);
        int len = a.lengths[b];
        if (len > a.c.capacity) {
            report(a.status, kStatusBadLength);
            len = a.c.capacity;
        }
        uint4 kx[kReadUnroll], vx[kReadUnroll];
        float kf[kReadUnroll], vf[kReadUnroll];
#pragma unroll
        for (int u = 0; u < kReadUnroll; ++u) {
            const int s = r0 + u * RPB;
            kx[u] = vx[u] = make_uint4(0, 0, 0, 0);
            kf[u] = vf[u] = 0.f;
            if (s >= a.S || s >= len) continue;
            const int page = a.c.pages[b * a.c.pages_sb + s / a.c.page_size], row = s % a.c.page_size;
            if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.c.n_pages)) {
                report(a.status, kStatusBadPage);
                continue;
            }
            const unsigned char* kp = a.c.k + page * a.c.k_sp + h * a.c.k_sh + row * a.c.k_ss;
            const unsigned char* vp = a.c.v + page * a.c.v_sp + h * a.c.v_sh + row * a.c.v_ss;
            if constexpr (E8) {
                const uint2 k2 = __ldcs(reinterpret_cast<const uint2*>(kp) + sub);
                const uint2 v2 = __ldcs(reinterpret_cast<const uint2*>(vp) + sub);
                kx[u].x = k2.x;
                kx[u].y = k2.y;
                vx[u].x = v2.x;
                vx[u].y = v2.y;
                kf[u] = scale_value(a.c.k_scale[page * a.c.ks_sp + h * a.c.ks_sh + row]);
                vf[u] = scale_value(a.c.v_scale[page * a.c.vs_sp + h * a.c.vs_sh + row]);
            } else {
                kx[u] = __ldcs(reinterpret_cast<const uint4*>(kp) + sub);
                vx[u] = __ldcs(reinterpret_cast<const uint4*>(vp) + sub);
            }
        }
        auto widen = [](uint4& x, float f) {
            const uint32_t w[4] = {x.x, x.x >> 16, x.y, x.y >> 16};
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t h2 = e4m3_to_half2(w[i]);
                const float2 y = Num<__half>::unpack(h2);
                o[i] = Num<T>::pack(y.x * f, y.y * f);
            }
            x = make_uint4(o[0], o[1], o[2], o[3]);
        };
#pragma unroll
        for (int u = 0; u < kReadUnroll; ++u) {
            const int s = r0 + u * RPB;
            if (s >= a.S) continue;
            if constexpr (E8) {
                widen(kx[u], kf[u]);
                widen(vx[u], vf[u]);
            }
            T* ko = reinterpret_cast<T*>(a.k) + b * a.k_sb + h * a.k_sh + s * a.k_ss;
            T* vo = reinterpret_cast<T*>(a.v) + b * a.v_sb + h * a.v_sh + s * a.v_ss;
            __stcs(reinterpret_cast<uint4*>(ko) + sub, kx[u]);
            __stcs(reinterpret_cast<uint4*>(vo) + sub, vx[u]);
        }
    }
}

}  // namespace kf
