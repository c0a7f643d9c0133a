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
    int k_sp, k_sh, k_ss, v_sp, v_sh, v_ss;      // (a page's place: a 32 x 32 -> 64 bit product)
    int ks_sp, ks_sh, vs_sp, vs_sh;
    const int* pages;                            // [B, max_pages]
    long long pages_sb;
    int n_pages, page_size, max_pages;
    int capacity;                                // max_pages * page_size, at most 2^31 - 1
};

__device__ __forceinline__ long long wide(int a, int b) { return static_cast<long long>(a) * b; }
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

// A row of D values over LPR lanes: lane i holds columns W i .. W i + W - 1 and their rotation partners D/2 further.  The
// arithmetic (order of the sum of squares included) does not depend on LPR: a row gets the same bits wherever it is done.
template <int D, int LPR> struct Row {
    static constexpr int W = D / 2 / LPR, kWords = W / 2;
    using Words = uint32_t[2][kWords];  // packed 16-bit values of both halves
    float x[2][W];

    template <bool STREAM> __device__ static __forceinline__ void load(Words& w, const void* row, int lane) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const char* const p = static_cast<const char*>(row) + half * D + lane * (2 * W);  // (bytes)
            if constexpr (kWords == 4) {
                const uint4 v = STREAM ? __ldcs(reinterpret_cast<const uint4*>(p)) : __ldg(reinterpret_cast<const uint4*>(p));
                w[half][0] = v.x;
                w[half][1] = v.y;
                w[half][2] = v.z;
                w[half][3] = v.w;
            } else if constexpr (kWords == 2) {
                const uint2 v = STREAM ? __ldcs(reinterpret_cast<const uint2*>(p)) : __ldg(reinterpret_cast<const uint2*>(p));
                w[half][0] = v.x;
                w[half][1] = v.y;
            } else {
                w[half][0] = STREAM ? __ldcs(reinterpret_cast<const uint32_t*>(p)) : __ldg(reinterpret_cast<const uint32_t*>(p));
            }
        }
    }
    template <typename T> __device__ __forceinline__ void unpack(const Words& w) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const float2 v = Num<T>::unpack(w[half][i]);
                x[half][2 * i] = v.x;
                x[half][2 * i + 1] = v.y;
            }
    }
    template <typename T> __device__ __forceinline__ void norm(const Words& gamma, float eps) {
        constexpr int kUnit = D / 64, kUnits = W / kUnit;  // a thirty-second of the row at a time
        float ss[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            ss[u] = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int i = 0; i < kUnit; ++i) ss[u] = fmaf(x[half][u * kUnit + i], x[half][u * kUnit + i], ss[u]);
        }
#pragma unroll
        for (int m = 1; m < kUnits; m *= 2)
#pragma unroll
            for (int u = 0; u < kUnits; u += 2 * m) ss[u] += ss[u + m];
#pragma unroll
        for (int m = 1; m < LPR; m *= 2) ss[0] += __shfl_xor_sync(0xffffffffu, ss[0], m);
        const float inv = rsqrtf(fmaf(ss[0], 1.0f / static_cast<float>(D), eps));
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const float2 g = Num<T>::unpack(gamma[half][i]);
                x[half][2 * i] = __fmul_rn(__fmul_rn(x[half][2 * i], inv), g.x);
                x[half][2 * i + 1] = __fmul_rn(__fmul_rn(x[half][2 * i + 1], inv), g.y);
            }
    }
    template <typename T> __device__ __forceinline__ void rotate(const Words& c, const Words& s) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const float2 cl = Num<T>::unpack(c[0][i]), ch = Num<T>::unpack(c[1][i]);
            const float2 sl = Num<T>::unpack(s[0][i]), sh = Num<T>::unpack(s[1][i]);
            const float lo0 = x[0][2 * i], lo1 = x[0][2 * i + 1], hi0 = x[1][2 * i], hi1 = x[1][2 * i + 1];
            x[0][2 * i] = fmaf(lo0, cl.x, -__fmul_rn(hi0, sl.x));
            x[0][2 * i + 1] = fmaf(lo1, cl.y, -__fmul_rn(hi1, sl.y));
            x[1][2 * i] = fmaf(hi0, ch.x, __fmul_rn(lo0, sh.x));
            x[1][2 * i + 1] = fmaf(hi1, ch.y, __fmul_rn(lo1, sh.y));
        }
    }
    // bits of the largest magnitude of the row (a NaN is the largest)
    __device__ __forceinline__ uint32_t largest() const {
        uint32_t m = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < W; ++i) m = max(m, __float_as_uint(x[half][i]) & 0x7fffffffu);
#pragma unroll
        for (int d = 1; d < LPR; d *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
        return m;
    }
    // The row in the cache's type: `put(byte offset, value)` with a value of 2, 4, 8 or 16 bytes.  Returns the scale's byte.
    template <typename T, bool E8, typename F> __device__ __forceinline__ uint32_t store(int lane, F&& put) const {
        uint32_t e = 0;
        if constexpr (E8) {
            e = scale_byte(largest());
            const float f = e == 255 ? 1.f : __uint_as_float((254u - e) << 23);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t w[(W + 3) / 4] = {};
#pragma unroll
                for (int i = 0; i < W; i += 2) w[i / 4] |= pack_e4m3(x[half][i] * f, x[half][i + 1] * f) << (8 * (i % 4));
                const int at = half * (D / 2) + lane * W;
                if constexpr (W == 8) put(at, make_uint2(w[0], w[1]));
                else if constexpr (W == 4) put(at, w[0]);
                else put(at, static_cast<uint16_t>(w[0]));
            }
        } else {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t w[kWords];
#pragma unroll
                for (int i = 0; i < kWords; ++i) w[i] = Num<T>::pack(x[half][2 * i], x[half][2 * i + 1]);
                const int at = half * D + lane * (2 * W);
                if constexpr (kWords == 4) put(at, make_uint4(w[0], w[1], w[2], w[3]));
                else if constexpr (kWords == 2) put(at, make_uint2(w[0], w[1]));
                else put(at, w[0]);
            }
        }
        return e;
    }
};

struct AppendArgs {
    CacheView c;
    const void *k, *v, *gamma, *cos, *sin;       // gamma, tables: may be null
    long long k_sb, k_sh, k_ss, v_sb, v_sh, v_ss;  // element strides
    const int *start, *counts;                   // counts may be null: all S rows
    int B, H, S, n_pos, heads_per_group;
    float eps;
    int* status;
};

constexpr int kRowsThreads = 256;

// A group of D/16 lanes walks over heads of one position, so that the tables are read once for them; a lane's columns are
// two 16-byte pieces of a row.
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
        const long long p = static_cast<long long>(a.start[b]) + s;
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
    using R = Row<D, LPR>;
    typename R::Words gamma, cos, sin;
    if (a.gamma != nullptr) R::template load<false>(gamma, a.gamma, sub);
    if (a.cos != nullptr) {
        R::template load<false>(cos, reinterpret_cast<const T*>(a.cos) + static_cast<long long>(valid ? pos : 0) * D, sub);
        R::template load<false>(sin, reinterpret_cast<const T*>(a.sin) + static_cast<long long>(valid ? pos : 0) * D, sub);
    }
    const int h0 = blockIdx.y * a.heads_per_group, h1 = min(h0 + a.heads_per_group, a.H);
    const T* kb = reinterpret_cast<const T*>(a.k) + b * a.k_sb + s * a.k_ss;
    const T* vb = reinterpret_cast<const T*>(a.v) + b * a.v_sb + s * a.v_ss;
    unsigned char* kd = a.c.k + wide(page, a.c.k_sp) + wide(row, a.c.k_ss);
    unsigned char* vd = a.c.v + wide(page, a.c.v_sp) + wide(row, a.c.v_ss);
    for (int h = h0; h < h1; ++h) {
        typename R::Words kw = {}, vw = {};
        if (valid) {
            R::template load<true>(kw, kb + h * a.k_sh, sub);
            R::template load<true>(vw, vb + h * a.v_sh, sub);
        }
        R k, v;
        k.template unpack<T>(kw);
        v.template unpack<T>(vw);
        if (a.gamma != nullptr) k.template norm<T>(gamma, a.eps);
        if (a.cos != nullptr) k.template rotate<T>(cos, sin);
        auto to = [&](unsigned char* dst) {
            return [=](int at, auto value) {
                if (valid) *reinterpret_cast<decltype(value)*>(dst + at) = value;
            };
        };
        const uint32_t ke = k.template store<T, E8>(sub, to(kd + wide(h, a.c.k_sh)));
        const uint32_t ve = v.template store<T, E8>(sub, to(vd + wide(h, a.c.v_sh)));
        if (E8 && valid && sub == 0) {
            a.c.k_scale[wide(page, a.c.ks_sp) + wide(h, a.c.ks_sh) + row] = static_cast<unsigned char>(ke);
            a.c.v_scale[wide(page, a.c.vs_sp) + wide(h, a.c.vs_sh) + row] = static_cast<unsigned char>(ve);
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
            const unsigned char* kp = a.c.k + wide(page, a.c.k_sp) + wide(h, a.c.k_sh) + wide(row, a.c.k_ss);
            const unsigned char* vp = a.c.v + wide(page, a.c.v_sp) + wide(h, a.c.v_sh) + wide(row, a.c.v_ss);
            if constexpr (E8) {
                const uint2 k2 = __ldcs(reinterpret_cast<const uint2*>(kp) + sub);
                const uint2 v2 = __ldcs(reinterpret_cast<const uint2*>(vp) + sub);
                kx[u].x = k2.x;
                kx[u].y = k2.y;
                vx[u].x = v2.x;
                vx[u].y = v2.y;
                kf[u] = scale_value(a.c.k_scale[wide(page, a.c.ks_sp) + wide(h, a.c.ks_sh) + row]);
                vf[u] = scale_value(a.c.v_scale[wide(page, a.c.vs_sp) + wide(h, a.c.vs_sh) + row]);
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
