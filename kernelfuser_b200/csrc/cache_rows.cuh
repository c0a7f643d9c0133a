// Rows into a paged key-value cache and back.
//
// append: K row x -> rotate(x * rsqrt(mean x^2 + eps) * gamma) at the row's own position, V row as it is, both written
// to row (position % page_size) of page table[b][position / page_size].
// read:   rows 0 .. length-1 of every sequence as contiguous [B, H, S, D], zeros behind them.
// Everything between the input's 16 bits and the cache's type is done in 32 bits and rounded once.  An 8-bit cache
// holds a row as e4m3 values times ONE power of two, kept as its exponent byte (e8m0): the smallest that brings the
// row's largest magnitude to at most 448.  A power of two costs no precision that e4m3 has (only its subnormals begin
// up to a factor of two earlier) and makes scaling exact, so that each value is rounded once and reading back to 16
// bits is exact.  (Magnitudes above 448 * 2^119 = 2.98e38 become that.)  A row whose largest magnitude is not finite
// gets the NaN scale and reads back as NaN.
#pragma once
#include <type_traits>

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
        float m = 0.f;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < W; ++i) asm("max.NaN.xorsign.abs.f32 %0, %0, %1;" : "+f"(m) : "f"(x[half][i]));
        uint32_t bits = __float_as_uint(m) & 0x7fffffffu;
#pragma unroll
        for (int d = 1; d < LPR; d *= 2) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
        return bits;
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

// A group of D/16 lanes takes up to kAppendHeads heads of one position, so that the tables are read once for them and their
// rows are in flight together; K rows and V rows are different CTAs' work (blockIdx.z).  Bound by HBM (16 bits: 16384 rows
// of eight heads in 27.3 us = 5.0 TB/s, launches in a graph; one head in flight 33, K and V in one lane 43) and by the latency
// of a CTA's chain of loads: 80 registers, three CTAs an SM (e4m3 30.5 -> 27.1 us).
constexpr int kAppendHeads = 4;

template <int D, typename T, bool E8>
__global__ void __launch_bounds__(kRowsThreads, 3) append_rows_kernel(const AppendArgs a) {
    constexpr int LPR = D / 16;
    using R = Row<D, LPR>;
    const int failed = *reinterpret_cast<volatile int*>(a.status);  // (looked at when there is something to write)
    const bool is_k = blockIdx.z == 0;
    const int sub = threadIdx.x % LPR;
    const long long task = static_cast<long long>(blockIdx.x) * (kRowsThreads / LPR) + threadIdx.x / LPR;
    const int b = static_cast<int>(task / a.S), s = static_cast<int>(task - static_cast<long long>(b) * a.S);
    bool valid = b < a.B;
    int start = 0, count = 0;
    if (valid) {
        start = __ldg(a.start + b);
        count = a.counts != nullptr ? __ldg(a.counts + b) : a.S;
    }
    valid = s < count;
    // the rows are asked for before their place is known
    const int h0 = blockIdx.y * a.heads_per_group, heads = min(a.heads_per_group, a.H - h0);
    const T* const src = is_k ? reinterpret_cast<const T*>(a.k) + b * a.k_sb + s * a.k_ss + h0 * a.k_sh
                              : reinterpret_cast<const T*>(a.v) + b * a.v_sb + s * a.v_ss + h0 * a.v_sh;
    const long long src_h = is_k ? a.k_sh : a.v_sh;
    typename R::Words rows[kAppendHeads] = {};
#pragma unroll
    for (int i = 0; i < kAppendHeads; ++i)
        if (valid && i < heads) R::template load<true>(rows[i], src + i * src_h, sub);
    int pos = 0, page = 0, row = 0;
    if (valid) {
        const long long p = static_cast<long long>(start) + s;
        if (p < 0 || p >= a.c.capacity) {
            report(a.status, kStatusBadLength);
            valid = false;
        } else if (a.cos != nullptr && p >= a.n_pos) {
            report(a.status, kStatusBadPosition);
            valid = false;
        } else {
            pos = static_cast<int>(p);
            page = __ldg(a.c.pages + b * a.c.pages_sb + pos / a.c.page_size);
            row = pos % a.c.page_size;
            if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.c.n_pages)) {
                report(a.status, kStatusBadPage);
                valid = false;
            }
        }
    }
    typename R::Words gamma, cos, sin;
    if (is_k && a.gamma != nullptr) R::template load<false>(gamma, a.gamma, sub);
    if (is_k && a.cos != nullptr) {
        R::template load<false>(cos, reinterpret_cast<const T*>(a.cos) + static_cast<long long>(pos) * D, sub);
        R::template load<false>(sin, reinterpret_cast<const T*>(a.sin) + static_cast<long long>(pos) * D, sub);
    }
    valid = valid && failed == 0;
    unsigned char* dst = is_k ? a.c.k + wide(page, a.c.k_sp) + wide(row, a.c.k_ss) + wide(h0, a.c.k_sh)
                              : a.c.v + wide(page, a.c.v_sp) + wide(row, a.c.v_ss) + wide(h0, a.c.v_sh);
    unsigned char* scale = nullptr;
    if constexpr (E8)
        scale = is_k ? a.c.k_scale + wide(page, a.c.ks_sp) + wide(h0, a.c.ks_sh) + row
                     : a.c.v_scale + wide(page, a.c.vs_sp) + wide(h0, a.c.vs_sh) + row;
    const int dst_h = is_k ? a.c.k_sh : a.c.v_sh, scale_h = is_k ? a.c.ks_sh : a.c.vs_sh;
#pragma unroll
    for (int i = 0; i < kAppendHeads; ++i) {
        if (i >= heads) break;
        R x;
        x.template unpack<T>(rows[i]);
        if (is_k && a.gamma != nullptr) x.template norm<T>(gamma, a.eps);
        if (is_k && a.cos != nullptr) x.template rotate<T>(cos, sin);
        const uint32_t e = x.template store<T, E8>(sub, [&](int at, auto value) {
            if (valid) *reinterpret_cast<decltype(value)*>(dst + at) = value;
        });
        if (E8 && valid && sub == 0) *scale = static_cast<unsigned char>(e);
        dst += dst_h;
        if constexpr (E8) scale += scale_h;
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

// A lane owns 8 columns of a row: one 16-byte store, and a 16-byte (16-bit cache) or 8-byte load.  A CTA takes some blocks of
// rows of one head of one sequence; a block lies in one page, whose place is looked up once for all its lanes.
constexpr int kReadBlocks = 4;  // in flight per lane, of K and of V
template <int D> __host__ __device__ constexpr int read_block() { return kRowsThreads / (D / 8); }  // rows; divides 16

template <int D, typename T, bool E8>
__global__ void __launch_bounds__(kRowsThreads) read_rows_kernel(const ReadArgs a) {
    constexpr int LPR = D / 8, RPB = read_block<D>();
    using Raw = typename std::conditional<E8, uint2, uint4>::type;
    const int failed = *reinterpret_cast<volatile int*>(a.status);  // (looked at when there is something to write)
    const int sub = threadIdx.x % LPR, r = threadIdx.x / LPR, first = blockIdx.x * (RPB * kReadBlocks);
    for (long long bh = blockIdx.y; bh < static_cast<long long>(a.B) * a.H; bh += gridDim.y) {
        const int b = static_cast<int>(bh / a.H), h = static_cast<int>(bh - static_cast<long long>(b) * a.H);
        int len = a.lengths[b];
        if (len > a.c.capacity) {
            report(a.status, kStatusBadLength);
            len = a.c.capacity;
        }
        len = min(len, a.S);
        const unsigned char* const kh = a.c.k + wide(h, a.c.k_sh) + wide(r, a.c.k_ss);
        const unsigned char* const vh = a.c.v + wide(h, a.c.v_sh) + wide(r, a.c.v_ss);
        Raw kx[kReadBlocks], vx[kReadBlocks];
        float kf[kReadBlocks], vf[kReadBlocks];
        int i = first / a.c.page_size, row = first - i * a.c.page_size;  // page of the sequence and row in it
#pragma unroll
        for (int u = 0; u < kReadBlocks; ++u) {
            const int s0 = first + u * RPB;
            kx[u] = vx[u] = Raw{};
            kf[u] = vf[u] = 0.f;
            if (s0 >= len) continue;  // (all lanes alike)
            const int page = __ldg(a.c.pages + b * a.c.pages_sb + i), at = row;
            row += RPB;
            if (row >= a.c.page_size) {
                row = 0;
                ++i;
            }
            if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.c.n_pages)) {
                report(a.status, kStatusBadPage);
                continue;
            }
            if (s0 + r >= len) continue;
            kx[u] = __ldcs(reinterpret_cast<const Raw*>(kh + wide(page, a.c.k_sp) + wide(at, a.c.k_ss)) + sub);
            vx[u] = __ldcs(reinterpret_cast<const Raw*>(vh + wide(page, a.c.v_sp) + wide(at, a.c.v_ss)) + sub);
            if constexpr (E8) {
                kf[u] = scale_value(a.c.k_scale[wide(page, a.c.ks_sp) + wide(h, a.c.ks_sh) + at + r]);
                vf[u] = scale_value(a.c.v_scale[wide(page, a.c.vs_sp) + wide(h, a.c.vs_sh) + at + r]);
            }
        }
        auto put = [&](T* row, const Raw& x, float f) {
            if constexpr (E8) {
                const uint32_t w[4] = {x.x, x.x >> 16, x.y, x.y >> 16};
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 y = Num<__half>::unpack(e4m3_to_half2(w[i]));
                    o[i] = Num<T>::pack(y.x * f, y.y * f);
                }
                __stcs(reinterpret_cast<uint4*>(row) + sub, make_uint4(o[0], o[1], o[2], o[3]));
            } else {
                __stcs(reinterpret_cast<uint4*>(row) + sub, x);
            }
        };
        T* ko = reinterpret_cast<T*>(a.k) + b * a.k_sb + h * a.k_sh + (first + r) * a.k_ss;
        T* vo = reinterpret_cast<T*>(a.v) + b * a.v_sb + h * a.v_sh + (first + r) * a.v_ss;
#pragma unroll
        for (int u = 0; u < kReadBlocks; ++u) {
            if (first + r + u * RPB >= a.S || failed != 0) continue;
            put(ko, kx[u], kf[u]);
            put(vo, vx[u], vf[u]);
            ko += RPB * a.k_ss;
            vo += RPB * a.v_ss;
        }
    }
}

}  // namespace kf
