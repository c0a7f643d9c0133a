// Attention of one new token per sequence over a paged key-value cache.
//
// For sequence b with n cached rows, KV head h and its G query heads:  q' = rotate(rmsnorm(q) * gamma) at position n-1
// (either part may be absent),  s_j = scale * q' . k_j,  out = sum_j softmax(s)_j v_j  over j < n;  n <= 0 gives zeros.
//
// What bounds it.  Every cached byte is read once and serves G query heads: 4 D G operations per 4 D bytes of a 16-bit
// cache, a few operations a byte, so HBM sets the time and everything else has to stay out of its way.
//
// Work split.  The unit of work is 64 keys of one (sequence, KV head).  All units of the launch are laid in one line and
// every CTA takes an equal piece of it, found from the lengths on the device: ragged batches and single long sequences
// load all SMs alike, and a captured launch follows its lengths.  A CTA's piece covers whole (sequence, head) items and
// at most two broken ones; a broken item's pieces meet in the workspace and are joined by decode_join_kernel.
//
// Inside a CTA each of the four warps is a stream of its own: of every unit it takes 16 keys, copies their K and V rows
// into its own ring in shared memory (cp.async, across item borders), and keeps its own running maximum, sum and output;
// the four meet once per item.  S^T = K Q^T and O^T = V^T P^T: the 16 keys (16 columns of V) are the m16 of
// mma.m16n8k16 and the query heads its n8, so up to eight heads cost one instruction per 16 x 16 block of the cache.
// (The 128-row MMAs of the prefill kernels have nothing to fill their rows with here.)
// Rounding: q' and the probabilities are rounded to the 16-bit type of the product they enter; scores, maxima, sums and
// outputs are 32 bits.  An e4m3 cache is widened to f16 (exact) on the way into the product; q' is scaled there by a power
// of two per head so that its largest value is between 2^14 and 2^15; a key's scale multiplies its score, and a value row's scale
// goes into the exponent of its probability, whose running maximum for O is kept apart from the one for the sum.
#pragma once
#include <type_traits>

#include "cache_rows.cuh"

namespace kf {

struct DecodeArgs {
    CacheView c;
    const void *q, *gamma, *cos, *sin;  // gamma, tables: may be null
    void* out;
    long long q_sb, q_sh, o_sb, o_sh;   // element strides
    const int* lengths;
    float* ws;                          // decode_workspace_floats() floats
    int B, Hkv, G, row_blocks;          // G query heads per KV head in row_blocks blocks
    int n_pos;
    float eps, scale_log2e;
    int* status;
};

constexpr int kDecWarps = 4, kDecThreads = 32 * kDecWarps;
constexpr int kDecKeys = 16;                    // keys of a warp's step
constexpr int kDecUnit = kDecKeys * kDecWarps;  // keys of a unit
constexpr int kDecMinUnits = 4;                 // a CTA's piece is at least this long

template <int D, bool E8, int NT> struct DecodeCfg {
    static constexpr int kRowBytes = D * (E8 ? 1 : 2);
    static constexpr int kTileBytes = kDecKeys * kRowBytes;  // K or V of a step
    static constexpr int kScaleBytes = E8 ? 2 * kDecKeys : 0;
    static constexpr int kStageBytes = 2 * kTileBytes + kScaleBytes;
    static constexpr int kCtasPerSm = D == 256 && !E8 ? 1 : 2;
    static constexpr int kStages = kTileBytes == 2048 ? 6 : 3;
    static constexpr int kRows = 8 * NT;
    static constexpr int kMergeCols = 128, kPad = kMergeCols + 4;  // columns that meet at a time; a row in shared memory
    static constexpr int kRingBytes = kDecWarps * kStages * kStageBytes;
    static constexpr int kMergeBytes = 2 * 8 * kPad * 4 + 2 * kDecWarps * kRows * 4;
    static constexpr int kSmemBytes = kRingBytes + kMergeBytes;
    static constexpr int kPartFloats = kRows * D + 2 * kRows;  // output, maximum, sum of a broken item
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
    const int n = take ? 16 : 0;  // (0: zeros, nothing is read)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ int cached_rows(const DecodeArgs& a, int b) { return min(max(__ldg(a.lengths + b), 0), a.c.capacity); }
__device__ __forceinline__ int units_of(int len) { return (len + kDecUnit - 1) / kDecUnit; }

// A place in the line of units: unit t of nt of item hk of sequence b.
struct DecodeCursor {
    int b, hk, t, nt, len;
    int left;  // units up to the end of the CTA's piece
    // to the next item; only called with units left
    __device__ __forceinline__ void next_item(const DecodeArgs& a, int HK) {
        t = 0;
        if (++hk < HK) return;
        hk = 0;
        do len = cached_rows(a, ++b); while (len == 0 && b + 1 < a.B);
        nt = units_of(len);
    }
};

// The 16-bit fragments of a row block's query heads.  Lane l holds row l/4 of each n8 block; the columns are those that a
// K fragment of the same step has: of 16 columns 2t, 2t+1, 2t+8, 2t+9 (16-bit cache) or 4t .. 4t+3 (8-bit), t = l%4.
// A column and its rotation partner D/2 further are in the same lane.  Returns what the row's scores are to be multiplied
// with to undo the scaling of its values.
template <int D, typename T, bool E8>
__device__ __forceinline__ float query_fragment(const DecodeArgs& a, int b, int head, bool valid, int pos, uint32_t (&f)[D / 16][2]) {
    constexpr int N = D / 4;  // values a lane holds
    const int t = threadIdx.x % 4;
    float x[N];
    auto load = [&](const void* p, float (&y)[N]) {
        const T* const base = reinterpret_cast<const T*>(p);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            uint32_t w[2];
            if constexpr (E8) {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(base + 16 * j) + t);
                w[0] = u.x;
                w[1] = u.y;
            } else {
                w[0] = __ldg(reinterpret_cast<const uint32_t*>(base + 16 * j) + t);
                w[1] = __ldg(reinterpret_cast<const uint32_t*>(base + 16 * j + 8) + t);
            }
            const float2 u0 = Num<T>::unpack(w[0]), u1 = Num<T>::unpack(w[1]);
            y[4 * j] = u0.x;
            y[4 * j + 1] = u0.y;
            y[4 * j + 2] = u1.x;
            y[4 * j + 3] = u1.y;
        }
    };
    if (valid) {
        load(reinterpret_cast<const T*>(a.q) + b * a.q_sb + head * a.q_sh, x);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = 0.f;
    }
    if (a.gamma != nullptr) {
        float ss = 0.f, g[N];
#pragma unroll
        for (int i = 0; i < N; ++i) ss = fmaf(x[i], x[i], ss);
        ss += __shfl_xor_sync(0xffffffffu, ss, 1);
        ss += __shfl_xor_sync(0xffffffffu, ss, 2);
        const float inv = rsqrtf(ss * (1.0f / static_cast<float>(D)) + a.eps);
        load(a.gamma, g);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = x[i] * inv * g[i];
    }
    if (a.cos != nullptr && pos < a.n_pos) {
        float c[N], s[N];
        load(reinterpret_cast<const T*>(a.cos) + static_cast<long long>(pos) * D, c);
        load(reinterpret_cast<const T*>(a.sin) + static_cast<long long>(pos) * D, s);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float lo = x[i], hi = x[i + N / 2];
            x[i] = lo * c[i] - hi * s[i];
            x[i + N / 2] = hi * c[i + N / 2] + lo * s[i + N / 2];
        }
    }
    float back = 1.f;
    if constexpr (E8) {
        uint32_t amax = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7fffffffu);
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // largest value to [2^14, 2^15) (an infinity or a NaN stays what it is)
        const uint32_t e = min(max(amax >> 23, 15u), 254u);
        const float up = __uint_as_float((268u - e) << 23);  // 2^(141 - e)
        back = __uint_as_float((e - 14u) << 23);             // 2^(e - 141)
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] *= up;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            f[j][0] = Num<__half>::pack(x[4 * j], x[4 * j + 1]);
            f[j][1] = Num<__half>::pack(x[4 * j + 2], x[4 * j + 3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
            f[j][0] = Num<T>::pack(x[4 * j], x[4 * j + 1]);
            f[j][1] = Num<T>::pack(x[4 * j + 2], x[4 * j + 3]);
        }
    }
    return back;
}

// Where the broken items' parts and what joins them lie in the workspace: for each CTA two parts (0: an item that began
// in an earlier CTA, 1: one that begins here), then for each CTA {item that begins here and goes on, or -1; last CTA of it}.
template <int D, bool E8, int NT> __host__ __device__ constexpr long long decode_part_at(int cta, int which) {
    return (2LL * cta + which) * DecodeCfg<D, E8, NT>::kPartFloats;
}
template <int D, bool E8, int NT> __host__ __device__ constexpr long long decode_workspace_floats(int ctas) {
    return decode_part_at<D, E8, NT>(ctas, 0) + 4LL * ctas;
}

template <int D, typename T, bool E8, int NT>
__global__ void __launch_bounds__(kDecThreads, DecodeCfg<D, E8, NT>::kCtasPerSm) decode_kernel(const DecodeArgs a) {
    using C = DecodeCfg<D, E8, NT>;
    using M = typename std::conditional<E8, __half, T>::type;  // type of the products' operands
    constexpr int kDT = D / 16, kRows = C::kRows;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ long long s_sum[kDecWarps], s_first;
    __shared__ int s_b, s_dead;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int HK = a.Hkv * a.row_blocks, n_ctas = gridDim.x;
    int* const meta = reinterpret_cast<int*>(a.ws + decode_part_at<D, E8, NT>(n_ctas, 0));
    if (tid == 0) s_dead = *reinterpret_cast<volatile int*>(a.status);  // (one reading for the whole CTA)

    // ---- this CTA's piece of the line of units
    const int per_thread = (a.B + kDecThreads - 1) / kDecThreads, b_lo = tid * per_thread;
    long long mine = 0;
    for (int b = b_lo; b < min(b_lo + per_thread, a.B); ++b) {
        const int n = __ldg(a.lengths + b);
        if (n > a.c.capacity) report(a.status, kStatusBadLength);
        if (a.cos != nullptr && n > a.n_pos) report(a.status, kStatusBadPosition);
        mine += units_of(cached_rows(a, b));
    }
    long long before = mine;  // inclusive sums within the warp
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += x;
    }
    if (lane == 31) s_sum[warp] = before;
    __syncthreads();
    if (s_dead != 0) return;
    long long total = 0;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
        if (w < warp) before += s_sum[w];
        total += s_sum[w];
    }
    before -= mine;
    total *= HK;
    long long piece = (total + n_ctas - 1) / n_ctas;
    if (piece < kDecMinUnits) piece = kDecMinUnits;
    const long long u0 = piece * blockIdx.x, u1 = min(u0 + piece, total);
    if (u0 < total && before * HK <= u0 && u0 < (before + mine) * HK) {  // (one thread of the CTA)
        int b = b_lo;
        long long at = before;
        for (;;) {
            const int n = units_of(cached_rows(a, b));
            if (u0 < (at + n) * HK) break;
            at += n;
            ++b;
        }
        s_b = b;
        s_first = at;
    }
    // sequences without rows have no units: their output is zero
    for (int b = blockIdx.x; b < a.B; b += n_ctas)
        if (cached_rows(a, b) == 0) {
            const int Hq = a.Hkv * a.G;
            for (int i = tid; i < Hq * (D / 8); i += kDecThreads)
                reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + b * a.o_sb + (i / (D / 8)) * a.o_sh)[i % (D / 8)] =
                    make_uint4(0, 0, 0, 0);
        }
    if (u0 >= total) {
        if (tid == 0) meta[2 * blockIdx.x] = -1;
        return;
    }
    __syncthreads();
    DecodeCursor cc;
    cc.b = s_b;
    cc.len = cached_rows(a, cc.b);
    cc.nt = units_of(cc.len);
    {
        const long long in_b = u0 - s_first * HK;
        cc.hk = static_cast<int>(in_b / cc.nt);
        cc.t = static_cast<int>(in_b - static_cast<long long>(cc.hk) * cc.nt);
    }
    cc.left = static_cast<int>(u1 - u0);

    // ---- the warp's ring of stages: K rows, V rows (16-byte pieces xor-ed with the row so that eight rows of a column
    // block lie in different banks), scales
    const uint32_t ring = smem_u32(smem) + warp * C::kStages * C::kStageBytes;
    DecodeCursor pc = cc;
    int table_at = 0, my_page = 0, my_row = 0;  // lane i: page and row in it of the warp's keys of unit table_at + i
    bool fresh = true;                           // the producer stands at an item whose pages it has not looked up
    auto issue = [&](int stage) {
        const int key0 = pc.t * kDecUnit + warp * kDecKeys;
        if (fresh || pc.t - table_at >= 32) {
            fresh = false;
            table_at = pc.t;
            const int key = (pc.t + lane) * kDecUnit + warp * kDecKeys;
            my_page = 0;
            if (pc.t + lane < pc.nt && key < pc.len) {
                const int i = key / a.c.page_size;
                my_row = key - i * a.c.page_size;
                my_page = __ldg(a.c.pages + pc.b * a.c.pages_sb + i);
                if (static_cast<unsigned>(my_page) >= static_cast<unsigned>(a.c.n_pages)) {
                    report(a.status, kStatusBadPage);
                    my_page = -1;
                }
            }
        }
        const int page = __shfl_sync(0xffffffffu, my_page, pc.t - table_at);
        const int row0 = __shfl_sync(0xffffffffu, my_row, pc.t - table_at);
        if (key0 < pc.len) {
            constexpr int kPieces = C::kRowBytes / 16, kRowsAtOnce = 32 / kPieces == 0 ? 1 : 32 / kPieces;
            const int h = pc.hk / a.row_blocks, piece16 = lane % kPieces, r0 = lane / kPieces;
            const long long row = page < 0 ? 0 : row0 + r0, pg = page < 0 ? 0 : page;
            const int rows = page < 0 ? 0 : min(kDecKeys, pc.len - key0);
            const unsigned char* kp = a.c.k + pg * a.c.k_sp + h * a.c.k_sh + row * a.c.k_ss + piece16 * 16;
            const unsigned char* vp = a.c.v + pg * a.c.v_sp + h * a.c.v_sh + row * a.c.v_ss + piece16 * 16;
            const uint32_t base = ring + stage * C::kStageBytes;
#pragma unroll
            for (int i = 0; i < kDecKeys / kRowsAtOnce; ++i) {
                const int r = r0 + i * kRowsAtOnce;
                const uint32_t at = base + r * C::kRowBytes + ((piece16 ^ (r & 7)) << 4);
                cp_async16(at, kp + (r < rows ? i * kRowsAtOnce * a.c.k_ss : 0), r < rows);
                cp_async16(at + C::kTileBytes, vp + (r < rows ? i * kRowsAtOnce * a.c.v_ss : 0), r < rows);
            }
            if constexpr (E8) {
                // (all 16 scales: a page holds a multiple of 16 rows)
                if (lane == 0) cp_async16(base + 2 * C::kTileBytes, a.c.k_scale + pg * a.c.ks_sp + h * a.c.ks_sh + (row - r0), page >= 0);
                if (lane == 0) cp_async16(base + 2 * C::kTileBytes + kDecKeys, a.c.v_scale + pg * a.c.vs_sp + h * a.c.vs_sh + (row - r0), page >= 0);
            }
        }
        ++pc.t;
        --pc.left;
        if (pc.t == pc.nt && pc.left > 0) {
            pc.next_item(a, HK);
            fresh = true;
        }
    };
#pragma unroll
    for (int s = 0; s < C::kStages - 1; ++s) {
        if (pc.left > 0) issue(s);
        cp_async_commit();
    }

    float* const merge_o = reinterpret_cast<float*>(smem + C::kRingBytes);  // two copies of [8][kPad]
    float* const merge_m = merge_o + 2 * 8 * C::kPad;                       // [warps][rows]
    float* const merge_l = merge_m + kDecWarps * kRows;
    // ldmatrix: the row (key) of the stage and the 16-byte piece that this lane names
    const int q8 = lane >> 3;
    const int k_row = (q8 & 1) * 8 + (lane & 7), k_piece = q8 >> 1;
    const int v_row = E8 ? k_row : (q8 >> 1) * 8 + (lane & 7), v_piece = E8 ? k_piece : (q8 & 1);

    int stage = 0, continues = -1, last_cta = 0;
    while (cc.left > 0) {
        // ---- one item's part: units cc.t .. cc.t + n - 1
        const int n = min(cc.nt - cc.t, cc.left);
        if (n <= 0) break;
        const int h = cc.hk / a.row_blocks, row0 = (cc.hk - h * a.row_blocks) * kRows;
        uint32_t qf[NT][kDT][2];
        float mul[NT][2];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            const int r = row0 + u * 8 + g;
            const float back = query_fragment<D, T, E8>(a, cc.b, h * a.G + r, r < a.G, cc.len - 1, qf[u]);
            mul[u][0] = a.scale_log2e * __shfl_sync(0xffffffffu, back, 8 * t4);      // row 2 t4
            mul[u][1] = a.scale_log2e * __shfl_sync(0xffffffffu, back, 8 * t4 + 4);  // row 2 t4 + 1
        }
        float o[NT][kDT][4], m[NT][2], l[NT][2], mv[NT][2];  // mv: reference of O (its own only for an 8-bit cache)
#pragma unroll
        for (int u = 0; u < NT; ++u) {
#pragma unroll
            for (int i = 0; i < kDT; ++i) o[u][i][0] = o[u][i][1] = o[u][i][2] = o[u][i][3] = 0.f;
            m[u][0] = m[u][1] = mv[u][0] = mv[u][1] = -INFINITY;
            l[u][0] = l[u][1] = 0.f;
        }
        for (int i_unit = 0; i_unit < n; ++i_unit) {
            cp_async_wait<C::kStages - 2>();
            __syncwarp();  // all lanes' copies of this stage are there, and all lanes are done with the stage before it
            {
                const int next = stage == 0 ? C::kStages - 1 : stage - 1;
                if (pc.left > 0) issue(next);
                cp_async_commit();
            }
            const int key0 = (cc.t + i_unit) * kDecUnit + warp * kDecKeys;
            if (key0 < cc.len) {
                const uint32_t ks = ring + stage * C::kStageBytes, vs = ks + C::kTileBytes;
                // S^T: keys g, g + 8 (rows), heads 2 t4, 2 t4 + 1 (columns)
                float s[NT][4];
#pragma unroll
                for (int u = 0; u < NT; ++u) s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
                const uint32_t k_at = ks + k_row * C::kRowBytes;
                if constexpr (E8) {
#pragma unroll
                    for (int j = 0; j < kDT; j += 2) {
                        uint32_t r[4];
                        ldmatrix4(r, k_at + (((j + k_piece) ^ (k_row & 7)) << 4));
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t a0 = e4m3_to_half2(r[2 * x]), a2 = e4m3_to_half2(r[2 * x] >> 16);
                            const uint32_t a1 = e4m3_to_half2(r[2 * x + 1]), a3 = e4m3_to_half2(r[2 * x + 1] >> 16);
#pragma unroll
                            for (int u = 0; u < NT; ++u) mma16816<M>(s[u], a0, a1, a2, a3, qf[u][j + x][0], qf[u][j + x][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < kDT; ++j) {
                        uint32_t r[4];
                        ldmatrix4(r, k_at + (((2 * j + k_piece) ^ (k_row & 7)) << 4));
#pragma unroll
                        for (int u = 0; u < NT; ++u) mma16816<M>(s[u], r[0], r[1], r[2], r[3], qf[u][j][0], qf[u][j][1]);
                    }
                }
                const bool in0 = key0 + g < cc.len, in1 = key0 + g + 8 < cc.len;
                float ks0 = 1.f, ks1 = 1.f, ve0 = 0.f, ve1 = 0.f;  // factors of the keys, exponents of the value rows
                if constexpr (E8) {
                    const unsigned char* sc = smem + (vs + C::kTileBytes - smem_u32(smem));
                    ks0 = scale_value(sc[g]);
                    ks1 = scale_value(sc[g + 8]);
                    ve0 = sc[16 + g] == 255 ? NAN : static_cast<float>(sc[16 + g]) - 127.f;
                    ve1 = sc[24 + g] == 255 ? NAN : static_cast<float>(sc[24 + g]) - 127.f;
                }
                uint32_t pb[NT][2];
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    float x[4], w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = (i < 2 ? in0 : in1) ? s[u][i] * mul[u][i & 1] * (i < 2 ? ks0 : ks1) : -INFINITY;
                        w[i] = E8 ? ((i < 2 ? in0 : in1) ? x[i] + (i < 2 ? ve0 : ve1) : -INFINITY) : x[i];
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float mx = fmaxf(x[c], x[c + 2]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(m[u][c], fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)));
                        const float base = mx == -INFINITY ? 0.f : mx;
                        l[u][c] = l[u][c] * ex2(m[u][c] - base) + (ex2(x[c] - base) + ex2(x[c + 2] - base));
                        m[u][c] = mx;
                        float base_v = base;
                        float from = mv[u][c];
                        if constexpr (E8) {
                            float my = fmaxf(w[c], w[c + 2]);
                            my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 4));
                            my = fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 8));
                            mx = fmaxf(from, fmaxf(my, __shfl_xor_sync(0xffffffffu, my, 16)));
                            base_v = mx == -INFINITY ? 0.f : mx;
                        }
                        mv[u][c] = mx;
                        if (__any_sync(0xffffffffu, from != mx)) {
                            const float f = ex2(from - base_v);
#pragma unroll
                            for (int i = 0; i < kDT; ++i) {
                                o[u][i][c] *= f;
                                o[u][i][c + 2] *= f;
                            }
                        }
                        w[c] = ex2(w[c] - base_v);
                        w[c + 2] = ex2(w[c + 2] - base_v);
                    }
                    pb[u][0] = transpose8x8(Num<M>::pack(w[0], w[1]));
                    pb[u][1] = transpose8x8(Num<M>::pack(w[2], w[3]));
                }
                // O^T += V^T P^T
                const uint32_t v_at = vs + v_row * C::kRowBytes;
                if constexpr (E8) {
#pragma unroll
                    for (int i = 0; i < kDT; i += 2) {
                        uint32_t r[4];
                        ldmatrix4_trans(r, v_at + (((i + v_piece) ^ (v_row & 7)) << 4));
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            // bytes {key 2t col 2g, key 2t col 2g+1, key 2t+1 col 2g, key 2t+1 col 2g+1}
                            const uint32_t y0 = __byte_perm(r[2 * x], 0, 0x3120), y1 = __byte_perm(r[2 * x + 1], 0, 0x3120);
                            const uint32_t a0 = e4m3_to_half2(y0), a1 = e4m3_to_half2(y0 >> 16);
                            const uint32_t a2 = e4m3_to_half2(y1), a3 = e4m3_to_half2(y1 >> 16);
#pragma unroll
                            for (int u = 0; u < NT; ++u) mma16816<M>(o[u][i + x], a0, a1, a2, a3, pb[u][0], pb[u][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < kDT; ++i) {
                        uint32_t r[4];
                        ldmatrix4_trans(r, v_at + (((2 * i + v_piece) ^ (v_row & 7)) << 4));
#pragma unroll
                        for (int u = 0; u < NT; ++u) mma16816<M>(o[u][i], r[0], r[1], r[2], r[3], pb[u][0], pb[u][1]);
                    }
                }
            }
            stage = stage + 1 == C::kStages ? 0 : stage + 1;
        }

        // ---- the four warps' parts of the item together
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = l[u][c];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                l[u][c] = x;
                if (g == 0) {
                    merge_m[warp * kRows + u * 8 + 2 * t4 + c] = m[u][c];
                    merge_l[warp * kRows + u * 8 + 2 * t4 + c] = x;
                }
            }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < kDecWarps; ++w) top = fmaxf(top, merge_m[w * kRows + u * 8 + 2 * t4 + c]);
                const float f = mv[u][c] == -INFINITY ? 0.f : exp2f(mv[u][c] - (top == -INFINITY ? 0.f : top));
                // (a warp without keys has a zero output; one whose scores are all -inf keeps a NaN that it may hold)
#pragma unroll
                for (int i = 0; i < kDT; ++i) {
                    o[u][i][c] = f == 0.f && o[u][i][c] == 0.f ? 0.f : o[u][i][c] * f;
                    o[u][i][c + 2] = f == 0.f && o[u][i][c + 2] == 0.f ? 0.f : o[u][i][c + 2] * f;
                }
            }
        const bool whole = n == cc.nt;
        if (!whole && cc.t == 0) {  // begins here and goes on: to its last unit
            continues = cc.b * HK + cc.hk;
            last_cta = static_cast<int>((u1 - 1 + (cc.nt - n)) / piece);
        }
        float* const part = a.ws + decode_part_at<D, E8, NT>(blockIdx.x, cc.t == 0 ? 1 : 0);
        float* const copy = merge_o + (warp & 1) * 8 * C::kPad;
        // eight rows and 128 columns at a time: warps 2 and 3 leave theirs, 0 and 1 add theirs, all add the two copies
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += C::kMergeCols) {
                auto each = [&](auto&& f) {  // f(place in a copy, value)
#pragma unroll
                    for (int i = 0; i < C::kMergeCols / 16; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            f((2 * t4 + (k & 1)) * C::kPad + 16 * i + (E8 ? 2 * g + (k >> 1) : g + 8 * (k >> 1)), o[u][c0 / 16 + i][k]);
                };
                if (warp >= 2) each([&](int at, float x) { copy[at] = x; });
                __syncthreads();
                if (warp < 2) each([&](int at, float x) { copy[at] += x; });
                __syncthreads();
                for (int i = tid; i < 8 * (C::kMergeCols / 4); i += kDecThreads) {
                    const int r8 = i / (C::kMergeCols / 4), d8 = (i % (C::kMergeCols / 4)) * 4, r = u * 8 + r8, d = c0 + d8;
                    if (row0 + r >= a.G) break;  // (rows go up with i)
                    const float4 x = *reinterpret_cast<const float4*>(merge_o + r8 * C::kPad + d8);
                    const float4 y = *reinterpret_cast<const float4*>(merge_o + (8 + r8) * C::kPad + d8);
                    const float4 z = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
                    float top = -INFINITY, sum = 0.f;
#pragma unroll
                    for (int w = 0; w < kDecWarps; ++w) top = fmaxf(top, merge_m[w * kRows + r]);
#pragma unroll
                    for (int w = 0; w < kDecWarps; ++w) {
                        const float lw = merge_l[w * kRows + r];
                        sum += lw == 0.f ? 0.f : lw * exp2f(merge_m[w * kRows + r] - (top == -INFINITY ? 0.f : top));
                    }
                    if (whole) {
                        T* const dst = reinterpret_cast<T*>(a.out) + cc.b * a.o_sb + (h * a.G + row0 + r) * a.o_sh + d;
                        const float inv = 1.f / sum;
                        *reinterpret_cast<uint2*>(dst) = make_uint2(Num<T>::pack(z.x * inv, z.y * inv), Num<T>::pack(z.z * inv, z.w * inv));
                    } else {
                        *reinterpret_cast<float4*>(part + r * D + d) = z;
                        if (d == 0) {
                            part[kRows * D + r] = top;
                            part[kRows * D + kRows + r] = sum;
                        }
                    }
                }
                __syncthreads();  // the copies are free
            }
        cc.t += n;
        cc.left -= n;
        if (cc.left > 0) cc.next_item(a, HK);
    }
    cp_async_wait<0>();
    if (tid == 0) {
        meta[2 * blockIdx.x] = continues;
        meta[2 * blockIdx.x + 1] = last_cta;
    }
}

// Joins the broken items: CTA i the one that begins in CTA i of decode_kernel, in the order of the parts.
template <int D, typename T, bool E8, int NT>
__global__ void __launch_bounds__(kDecThreads) decode_join_kernel(const DecodeArgs a) {
    using C = DecodeCfg<D, E8, NT>;
    constexpr int kRows = C::kRows;
    const int n_ctas = gridDim.x, HK = a.Hkv * a.row_blocks, first = blockIdx.x;
    if (*reinterpret_cast<volatile int*>(a.status) != 0) return;
    const int* const meta = reinterpret_cast<const int*>(a.ws + decode_part_at<D, E8, NT>(n_ctas, 0));
    const int item = meta[2 * first], last = meta[2 * first + 1];
    if (item < 0) return;
    const int b = item / HK, hk = item - b * HK, h = hk / a.row_blocks, row0 = (hk - h * a.row_blocks) * kRows;
    for (int i = threadIdx.x; i < kRows * (D / 4); i += kDecThreads) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        if (row0 + r >= a.G) break;
        float top = -INFINITY, sum = 0.f;
        float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = first; c <= last; ++c) top = fmaxf(top, a.ws[decode_part_at<D, E8, NT>(c, c == first) + kRows * D + r]);
        for (int c = first; c <= last; ++c) {
            const float* part = a.ws + decode_part_at<D, E8, NT>(c, c == first);
            const float m = part[kRows * D + r], f = m == -INFINITY ? 0.f : exp2f(m - top);
            const float4 x = *reinterpret_cast<const float4*>(part + r * D + d);
            sum += part[kRows * D + kRows + r] * f;
            z.x += x.x * f;
            z.y += x.y * f;
            z.z += x.z * f;
            z.w += x.w * f;
        }
        T* const dst = reinterpret_cast<T*>(a.out) + b * a.o_sb + (h * a.G + row0 + r) * a.o_sh + d;
        const float inv = 1.f / sum;
        *reinterpret_cast<uint2*>(dst) = make_uint2(Num<T>::pack(z.x * inv, z.y * inv), Num<T>::pack(z.z * inv, z.w * inv));
    }
}

}  // namespace kf
