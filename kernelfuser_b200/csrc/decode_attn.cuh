// Attention of one new token per sequence over a paged key-value cache.
//
// For sequence b with n cached rows, KV head h and its G query heads:  q' = rotate(rmsnorm(q) * gamma) at position n-1
// (either part may be absent),  s_j = scale * q' . k_j,  out = sum_j softmax(s)_j v_j  over j < n;  n <= 0 gives zeros.
//
// What bounds it.  Every cached byte is read once and serves G query heads: 4 D G operations per 4 D bytes of a 16-bit
// cache, a few operations a byte, so HBM sets the time and everything else has to stay out of its way.
//
// Work split.  The unit of work is 64 keys of one (sequence, KV head), 128 where a warp's step is 32 keys or a CTA has
// eight warps.  All units of the launch are laid in one line and every CTA takes an equal piece of it, found from the
// lengths on the device: ragged batches and single long sequences load all SMs alike, and a captured launch follows its
// lengths.  A CTA's piece covers whole (sequence, head) items and at most two broken ones; a broken item's parts meet in
// the workspace, where the CTA that comes last joins them, in the order of the line whoever that is: as many at a time as
// its ring holds, and if there are more, the joined groups once more.  (A second kernel for it cost 2 us of a call, and
// its serial pass over 37 parts of a long sequence 12 us.)
//
// More than sixteen query heads of a KV head are blocks of sixteen, a CTA each for the same piece of the line: they run side
// by side, so that HBM gives a row to one of them and L2 to the others (128 sequences of 8192 rows, 24 heads: 173 us when
// the blocks were items one behind the other, 148; 48/2 heads of 256, 32 sequences: 176 -> 132).
//
// Inside a CTA each of the four (or eight) warps is a stream of its own: of every unit it takes a step of 16 keys (32 of an
// 8-bit cache), copies their K and V rows into its own ring of slots in shared memory (cp.async, across item borders), and
// keeps its own sum and output; they meet once per item.  S^T = K Q^T and O^T = V^T P^T: the 16 keys (16 columns of V) are
// the m16 of mma.m16n8k16 and the query heads its n8, so up to eight heads cost one instruction per 16 x 16 block of the
// cache.  (128 keys would fill the rows of a tcgen05.mma in the same way, with more heads as its columns: not built.)  Q is
// prepared once per item, a row to a warp, from values that are loaded while the item before is computed.
// The exponentials are taken against a base that is only moved when a score exceeds it by more than a factor of 2^8 (2^4
// where probabilities enter in f16), which is exact after the division by the sum: as a rule no lane waits for a maximum
// over lanes.
// A new token's K and V rows are prepared by the warp that has their step, which puts them into the cache and, for itself,
// behind the step's cached rows in shared memory: nobody else reads them, so nobody has to wait.
// Rounding: q' and the probabilities enter the products as the sum of two 16-bit numbers, so that what is left of them is
// 2^-16 (bf16) or 2^-22 (fp16) of each: a single rounding there doubled the error of a bf16 result (1.6e-3 -> 3.1e-3
// relative), and the products wait for HBM anyway (see kSplitProducts for the one exception).  Scores, sums and outputs are 32
// bits.  An e4m3 cache is widened to f16 (exact) on the way into the product; q' is scaled there by a power of two per head so
// that its largest value is between 2^14 and 2^15; a key's scale multiplies its score, and a value row's scale goes into the
// exponent of its probability, whose base for O is kept apart from the one for the sum.  Its warps and parts meet as means of
// value rows, never as sums of rows with their scales: finite value rows give a finite result (bf16 ones: see kUp).
#pragma once
#include <type_traits>
#include <utility>

#include "cache_rows.cuh"

namespace kf {

struct DecodeArgs {
    CacheView c;
    const void *q, *gamma, *cos, *sin;  // gamma, tables: may be null
    void* out;
    long long q_sb, q_sh, o_sb, o_sh;   // element strides
    const int* lengths;
    const void *new_k, *new_v, *gamma_k;  // the newest token's rows, not in the cache yet; null: they are
    long long nk_sb, nk_sh, nv_sb, nv_sh;
    float* ws;                          // decode_workspace_floats() floats
    unsigned int* arrived;              // a word per CTA, zero before and after the launch (see join_words)
    int B, Hkv, G, row_blocks;          // G query heads per KV head in row_blocks blocks
    int n_pos;
    float eps, scale_log2e;
    int* status;
};

// Items of up to this many units are not broken for CTAs that would be idle: joining costs about as much as four units (3
// units: 8.7 us whole, 9.7 broken).  Longer ones are, down to single units (128 units 17.8 -> 14.8 us, 16: 13.4 -> 11.4).
constexpr int kDecWhole = 4;  // (of 64 keys of 128; wider or longer units take that much longer)

template <int D, bool E8, int NT> struct DecodeCfg {
    static constexpr int kRows = 8 * NT;
    static constexpr bool kWide = D == 256 && NT == 2;                // more than eight heads of 256
    static constexpr int kWarps = kWide ? 8 : 4, kThreads = 32 * kWarps;
    static constexpr int kTiles = E8 && !kWide ? 2 : 1, kKeys = 16 * kTiles;  // blocks of 16 keys, keys of a warp's step
    static constexpr int kUnit = kKeys * kWarps;
    static constexpr int kRowBytes = D * (E8 ? 1 : 2);
    // What an item costs beside its units, in units of its keys: about 3 us of a CTA (looking up its rows, preparing its
    // queries, meeting of the warps), which hold a unit of 64 KB or two of 32.  32 ragged sequences of up to 1500 rows: 1 -> 36
    // us, 2 -> 28.7, 3 -> 27.7; wide heads 16 x 2047: 34.7, 32.8, 33.4; uniform batches do not care.
    static constexpr int kItemCost = kRowBytes == 512 ? 2 : 3;
    static constexpr int kSlotBytes = kKeys * kRowBytes;              // K or V rows of a step
    static constexpr int kScaleBytes = E8 ? kKeys : 0;                // and their scales
    static constexpr bool kQueryInRegs = !kWide;                      // else its fragments are read for every step
    static constexpr int kCtasPerSm = kWide ? 1 : E8 && D == 128 && NT == 1 ? 3 : 2;
    // An 8-bit cache is bound by the instructions that widen it as much as by HBM: steps of 32 keys share what a step costs
    // and have twice as many independent products (64 sequences of 4096 rows, G = 4: 118 -> 98 us, floor 83), and three CTAs
    // give the schedulers a third warp each (135 -> 116 us with steps of 16; four, at 128 registers: 124).
    // With more than eight heads of 256 O alone takes 128 registers and one CTA's queries 16 KB: eight warps share them.
    // The first pages of the next item are looked up when an item is entered: waiting for them at the border, twice where a
    // piece begins near an item's end, made the last CTAs late (16 sequences of 8192 rows, 8 heads: 21.5 -> 20.4 us; four of
    // 8192, 32/8 heads 31.1 -> 30.1).  The 8-bit and the wide kernels have no registers left for it (64 x 4096 rows 94.1 -> 95.7;
    // 48/2 heads of 256 132 -> 155).
    static constexpr bool kLookAhead = !E8 && !kWide;
    // slots of a warp's ring: as many as let that many CTAs onto an SM (about 100 KB each of two)
    static constexpr int kSlots = E8 ? (kWide || (D == 128 && NT == 2) ? 5 : 3) : D == 256 ? 3 : NT == 1 ? 6 : 5;
    // Copies of O in which the warps meet, one after the other in each (eight warps, 64 sequences of 1000 rows, 32/2 heads of
    // 256: 40 us with two, 37 with four; for four warps of an 8-bit cache four gained nothing, of a 16-bit one they do not fit).
    static constexpr int kCopies = kWide ? 4 : 2;
    // columns that meet at a time; a row of them in shared memory
    static constexpr int kMergeCols = D == 256 || E8 ? 64 : 128, kPad = kMergeCols + 4;
    static constexpr int kRingBytes = kWarps * kSlots * kSlotBytes;
    static constexpr int kScaleRingBytes = kWarps * kSlots * kScaleBytes;
    static constexpr int kQueryBytes = NT * (D / 16) * 32 * 16;       // {high, high, low, low} fragments of a lane
    static constexpr int kMergeBytes = kCopies * 8 * kPad * 4 + (2 * kWarps + 1) * kRows * 4;
    static constexpr int kNewBytes = 2 * kRowBytes;                   // a new token's K and V row
    static constexpr int kSmemBytes = kRingBytes + kQueryBytes + kMergeBytes + kScaleRingBytes + kNewBytes;
    static constexpr int kPartFloats = kRows * D + 2 * kRows;         // mean, and its weight, of a broken item's part
};

// Copies of cache rows into shared memory.  Each row is read once, so it is the first to leave L2 again: what is read over and
// over (the kernel's own instructions, weights, tables) stays.
__device__ __forceinline__ uint64_t evict_first_policy() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
// (without a policy: together with a source size it raised an illegal instruction on B200)
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool take) {
    const int n = take ? 16 : 0;  // (0: zeros, nothing is read)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int DST, int SRC> __device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0 + %3], [%1 + %4], 16, %2;" ::"r"(dst), "l"(src), "l"(policy),
                 "n"(DST), "n"(SRC) : "memory");
}
template <typename F, int... I> __device__ __forceinline__ void each_index(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
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
// Four e4m3 as two f16x2 (exact).
__device__ __forceinline__ void widen4(uint32_t x, uint32_t& lo, uint32_t& hi) {
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(lo), "=r"(hi) : "r"(x));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ int cached_rows(const DecodeArgs& a, int b) {
    return min(max(__ldg(a.lengths + b), 0), a.c.capacity);
}
template <int UNIT> __device__ __forceinline__ int units_of(int len) { return (len + UNIT - 1) / UNIT; }

// A place in the line of units: unit t of nt of KV head h of sequence b.
template <int UNIT, int COST> struct DecodeCursor {
    int b, h, t, nt, len;
    int left;  // of the line up to the end of the CTA's piece
    // to the next item, if the piece reaches it
    __device__ __forceinline__ void next_item(const DecodeArgs& a) {
        left -= COST;
        if (left <= 0) return;
        t = 0;
        if (++h < a.Hkv) return;
        h = 0;
        do len = cached_rows(a, ++b); while (len == 0 && b + 1 < a.B);
        nt = units_of<UNIT>(len);
    }
};

// An f16 product of a bf16 call has no second part: one number is off by 2^-12 of it at most, an eighth of what the output's
// own rounding may cost.  64 ragged sequences of up to 8192 rows: 114 us, with both parts 128; error against 64 bits 1.45e-3 of
// which the output's rounding makes 1.41e-3.  Scores spread by 1 to 32 (sequences of 4000 rows): 1.27e-3 .. 1.69e-3 with one
// part and with two, and from the rounding alone.
template <typename T, bool E8> constexpr bool kSplitProducts = !(E8 && std::is_same<T, __nv_bfloat16>::value);

// Two values, each as high + low of the products' type: high is rounded towards zero, so that low has the value's sign and
// together they hold twice the type's bits.  A low part that would be zero becomes the type's smallest number instead
// (kMin, far below what is kept): an infinity in the cache then meets two factors of one sign and stays that infinity.
template <typename M> struct Split;
template <> struct Split<__nv_bfloat16> {
    static constexpr float kMin = 0x1p-126f;
    __device__ static __forceinline__ uint32_t toward_zero(float lo, float hi) {
        uint32_t r;
        asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};
template <> struct Split<__half> {
    static constexpr float kMin = 0x1p-24f;
    __device__ static __forceinline__ uint32_t toward_zero(float lo, float hi) {
        uint32_t r;
        asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
};
// values of any sign (a zero stays zero in both parts)
template <typename M> __device__ __forceinline__ void split2(float x, float y, uint32_t& high, uint32_t& low) {
    high = Split<M>::toward_zero(x, y);
    const float2 h = Num<M>::unpack(high);
    auto rest = [](float v, float hv) {
        const float r = v - hv;
        return fabsf(r) < Split<M>::kMin && v != 0.f ? copysignf(Split<M>::kMin, v) : r;
    };
    low = Num<M>::pack(rest(x, h.x), rest(y, h.y));
}
// probabilities; FLOOR: against infinities in the cache (an 8-bit one has none)
template <typename M, bool FLOOR>
__device__ __forceinline__ void split2_probabilities(float x, float y, uint32_t& high, uint32_t& low) {
    if constexpr (FLOOR) {  // (x < kMin and not max(): a NaN stays one)
        x = x < Split<M>::kMin ? Split<M>::kMin : x;
        y = y < Split<M>::kMin ? Split<M>::kMin : y;
    }
    high = Split<M>::toward_zero(x, y);
    const float2 h = Num<M>::unpack(high);
    x -= h.x;
    y -= h.y;
    low = FLOOR ? Num<M>::pack(fmaxf(x, Split<M>::kMin), fmaxf(y, Split<M>::kMin)) : Num<M>::pack(x, y);
}

// The query rows that a warp prepares for an item (every WARPS-th), loaded ahead of time.
template <int D, typename T, int NT, int WARPS> struct QueryRows {
    using R = Row<D, 32>;
    static constexpr int kN = 8 * NT / WARPS;  // rows of a warp
    typename R::Words q[kN], cos, sin;
    template <typename Cursor> __device__ __forceinline__ void load(const DecodeArgs& a, const Cursor& at, int row0) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int r = row0 + warp + WARPS * i;
            if (r < a.G) {
                R::template load<false>(q[i], reinterpret_cast<const T*>(a.q) + at.b * a.q_sb + (at.h * a.G + r) * a.q_sh, lane);
            } else {
#pragma unroll
                for (int p = 0; p < R::kWords; ++p) q[i][0][p] = q[i][1][p] = 0u;
            }
        }
        if (a.cos != nullptr) {
            const long long row = static_cast<long long>(min(at.len, a.n_pos) - 1) * D;
            R::template load<false>(cos, reinterpret_cast<const T*>(a.cos) + row, lane);
            R::template load<false>(sin, reinterpret_cast<const T*>(a.sin) + row, lane);
        }
    }
    // Norm, rotation, and the fragments of the products into shared memory: lane l of a fragment holds row l/4, and of 16
    // columns 2t, 2t+1, 2t+8, 2t+9 (16-bit cache) or 4t .. 4t+3 (8-bit), t = l%4, as a K fragment of that step does.
    // back[row]: what the row's scores are to be multiplied with to undo the scaling of its values (8-bit cache).
    template <bool E8>
    __device__ __forceinline__ void prepare(const DecodeArgs& a, const typename R::Words& gamma, uint4* frag, float* back) const {
        using M = typename std::conditional<E8, __half, T>::type;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int r = warp + WARPS * i;
            R row;
            row.template unpack<T>(q[i]);
            if (a.gamma != nullptr) row.template norm<T>(gamma, a.eps);
            if (a.cos != nullptr) row.template rotate<T>(cos, sin);
            float up = 1.f;
            if constexpr (E8) {  // largest value to [2^14, 2^15) (an infinity or a NaN stays what it is)
                const uint32_t e = min(max(row.largest() >> 23, 15u), 254u);
                up = __uint_as_float((268u - e) << 23);                                     // 2^(141 - e)
                if (lane == 0) back[r] = a.scale_log2e * __uint_as_float((e - 14u) << 23);  // 2^(e - 141)
            }
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int p = 0; p < R::kWords; ++p) {
                    const int col = half * (D / 2) + lane * R::W + 2 * p, in = col % 16;
                    const int t = E8 ? in / 4 : in % 8 / 2, reg = E8 ? in % 4 / 2 : in / 8;
                    uint32_t* const dst = reinterpret_cast<uint32_t*>(frag + (r / 8 * (D / 16) + col / 16) * 32 + r % 8 * 4 + t);
                    const float x0 = row.x[half][2 * p] * up, x1 = row.x[half][2 * p + 1] * up;
                    if constexpr (kSplitProducts<T, E8>) split2<M>(x0, x1, dst[reg], dst[reg + 2]);
                    else dst[reg] = Num<M>::pack(x0, x1);
                }
        }
    }
};

// Where the broken items' parts lie in the workspace: for each CTA two (0: of an item that began in an earlier CTA, 1: of
// one that begins here).  Behind them are words for `arrived`, for launches that have none of the library's.
template <int D, bool E8, int NT> __host__ __device__ constexpr long long decode_part_at(int cta, int which) {
    return (2LL * cta + which) * DecodeCfg<D, E8, NT>::kPartFloats;
}
template <int D, bool E8, int NT> __host__ __device__ constexpr long long decode_workspace_floats(int ctas) {
    return decode_part_at<D, E8, NT>(ctas, 0) + ctas;
}

// Joining.  CTAs are numbered here among those of one block of query rows.  Item parts of CTAs first .. last (one that begins
// in `first`); groups of join_group() consecutive ones.  A CTA's word counts in three fields: parts that have arrived of the
// group whose first part is its part 0 (bits 0-7) or its part 1 (8-15), and joined groups of the item that begins in it
// (16-31).  Who completes a field takes it back to zero.
struct DecodeBroken {
    int first, last;  // its CTAs; first < 0: there is none
    int b, h;
};

// A part is the mean of its value rows and their weight, mantissa * 2^exponent: what a sum of probabilities against a base comes
// to, with the mantissa brought to [2^-8, 2^-7).  The weighted parts of a join, 64 at most, then add up to less than the largest
// value: it may be as large as 32 bits hold.  (0, infinity and NaN stay.)
__device__ __forceinline__ void part_weight(float* exponent, float* mantissa, float base, float sum) {
    const int e = static_cast<int>(__float_as_uint(sum) >> 23) - 119;
    const bool plain = sum > 0.f && sum < INFINITY;
    *exponent = plain ? base + static_cast<float>(e) : base;
    *mantissa = plain ? __uint_as_float((__float_as_uint(sum) & 0x7fffffu) | 119u << 23) : sum;
}

template <int D, typename T, bool E8, int NT> struct DecodeJoin {
    using C = DecodeCfg<D, E8, NT>;
    static constexpr int kRows = C::kRows;
    const DecodeArgs& a;
    float* room;     // shared memory: the ring
    int* s_flag;     // shared memory: 2
    int cta, row_block;

    __device__ __forceinline__ int row0() const { return row_block * kRows; }
    __device__ __forceinline__ int index(int of) const { return of * a.row_blocks + row_block; }  // in the grid
    __device__ __forceinline__ float* part(int of, bool begins) const {
        return a.ws + decode_part_at<D, E8, NT>(index(of), begins);
    }

    // parts that the ring holds side by side, of rows that exist
    __device__ __forceinline__ int part_floats() const { return min(kRows, a.G) * D + 2 * kRows; }
    // Parts that one CTA joins of an item of n: all, if its ring holds them, else about as many as there will be groups (32
    // parts of 4 KB: 7 us one ring full after the other, 5 in six groups of six).
    __device__ __forceinline__ int join_group(int n) const {
        return n <= min(64, C::kRingBytes / 4 / part_floats()) ? n : static_cast<int>(ceilf(sqrtf(static_cast<float>(n))));
    }

    static constexpr int kQuads = kRows * (D / 4) / C::kThreads;  // groups of four columns that a thread sums up, at most

    // One thread: count one more in the field; true for the CTA that completes `count`.  What the CTA has written before a
    // barrier in front of this is visible to whoever counts later, behind a barrier of theirs.  (acq_rel: with full fences
    // around a plain atomic the 16 sequences below take 28.1 instead of 26.6 us, the smallest broken calls 0.4 more.)
    __device__ __forceinline__ bool count_up(int of, int shift, int count) const {
        unsigned int before;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], %2;" : "=r"(before)
                     : "l"(a.arrived + index(of)), "r"(1u << shift) : "memory");
        const bool all = static_cast<int>(before >> shift & (shift == 16 ? 0xffffu : 0xffu)) == count - 1;
        if (all) atomicSub(a.arrived + index(of), static_cast<unsigned int>(count) << shift);
        return all;
    }
    // n parts, every `stride` CTAs from `from` on, to `out` (a part's place) or, if that is null, to the result's rows.  The
    // parts are copied into the ring, then a thread takes some columns of a row, four at a time.  (Little code: it is run once
    // a launch, and its own way from memory costs more than what it does: with eight parts at a time in registers 4 us.)
    __device__ __forceinline__ void sum(int first, int from, int stride, int n, float* out, int b, int h) const {
        const int size = part_floats(), rows = min(kRows, a.G - row0()), cap = C::kRingBytes / 4 / size;
        int have = 0;  // 1: the sum so far lies in front
#pragma unroll 1
        for (int i0 = 0; i0 < n;) {
            const int add = min(n - i0, cap - have), count = have + add;
            const int lane = threadIdx.x & 31;
#pragma unroll 1
            for (int i = threadIdx.x >> 5; i < add; i += C::kWarps) {
                const int of = from + (i0 + i) * stride;
                const float* const src = part(of, of == first) + lane * 4;
                const uint32_t dst = smem_u32(room + (have + i) * size) + lane * 16;
#pragma unroll
                for (int c = 0; c < kRows * (D / 4); c += 32)  // the rows that exist, then their weights
                    if (c < rows * (D / 4)) cp_async16(dst + c * 16, src + c * 4);
                if (lane < 2 * kRows / 4) cp_async16(dst + (size - 2 * kRows) * 4, src + kRows * D);
            }
            cp_async_commit();
            cp_async_wait<0>();
            __syncthreads();
            i0 += add;
            // a thread stays in one row, so that it takes the row's weights once
            const int shift = __clz(rows - 1) - __clz(C::kThreads) - 1;  // 2^shift threads to a row
            const int r = static_cast<int>(threadIdx.x) >> shift, c = threadIdx.x & ((1 << shift) - 1);
            float* const m = room + size - 2 * kRows + r;  // exponents of the first part's weights; mantissas kRows further
            float top = -INFINITY, total = 0.f;
            if (r < rows && c < D / 4) {
#pragma unroll 4
                for (int i = 0; i < count; ++i) top = fmaxf(top, m[i * size]);
                float4 z[kQuads];
#pragma unroll
                for (int k = 0; k < kQuads; ++k) z[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                float* const row = room + r * D + c * 4;
#pragma unroll 2
                for (int i = 0; i < count; ++i) {
                    const float mi = m[i * size], w = m[i * size + kRows] * (mi == -INFINITY ? 0.f : ex2(mi - top));
                    total += w;
#pragma unroll
                    for (int k = 0; k < kQuads; ++k) {
                        if (c + (k << shift) >= D / 4) break;
                        const float4 x = *reinterpret_cast<const float4*>(row + i * size + (k << shift) * 4);
                        z[k] = make_float4(fmaf(x.x, w, z[k].x), fmaf(x.y, w, z[k].y), fmaf(x.z, w, z[k].z), fmaf(x.w, w, z[k].w));
                    }
                }
                // (no weight at all: undefined, and as a part nothing)
                const float inv = total != 0.f ? 1.f / total : i0 >= n && out == nullptr ? NAN : 0.f;
#pragma unroll
                for (int k = 0; k < kQuads; ++k) {
                    const int at = (k << shift) * 4;
                    if (c * 4 + at >= D) break;
                    z[k] = make_float4(z[k].x * inv, z[k].y * inv, z[k].z * inv, z[k].w * inv);
                    if (i0 < n) {
                        *reinterpret_cast<float4*>(row + at) = z[k];  // (what only this thread has read)
                    } else if (out != nullptr) {
                        *reinterpret_cast<float4*>(out + r * D + c * 4 + at) = z[k];
                    } else {
                        T* const dst = reinterpret_cast<T*>(a.out) + b * a.o_sb + (h * a.G + row0() + r) * a.o_sh + c * 4 + at;
                        *reinterpret_cast<uint2*>(dst) =
                            make_uint2(Num<T>::pack(z[k].x, z[k].y), Num<T>::pack(z[k].z, z[k].w));
                    }
                }
            }
            if (i0 >= n && out == nullptr) break;
            // weights of the rows, once all have read the old ones
            __syncthreads();
            if (r < rows && c == 0) {
                float* const to = i0 < n ? m : out + kRows * D + r;
                part_weight(to, to + kRows, top, total);
            }
            have = 1;
            __syncthreads();
        }
        __syncthreads();  // (the ring is free again)
    }
    // One thread, behind a barrier behind the writing of this CTA's part of the item (`dead`: it never will be; only the
    // counts have to go on): count it.  True: the part completes its group.
    __device__ __forceinline__ bool part_done(const DecodeBroken& it) const {
        const int group = join_group(it.last - it.first + 1);
        const int from = it.first + (cta - it.first) / group * group;
        const int n = min(group, it.last - from + 1);
        return n == 1 || count_up(from, from == it.first ? 8 : 0, n);
    }
    // All threads, once, behind the counting: the joins that fall to this CTA (those whose s_flag is set).
    __device__ __forceinline__ void run(const DecodeBroken (&item)[2], bool dead) const {
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            if (s_flag[k] == 0) continue;
            const DecodeBroken it = k == 0 ? item[0] : item[1];
            const int group = join_group(it.last - it.first + 1), groups = (it.last - it.first) / group + 1;
            int from = it.first + (cta - it.first) / group * group, stride = 1, n = min(group, it.last - from + 1);
            bool final = groups == 1;
#pragma unroll 1
            for (;;) {
                float* const place = final ? nullptr : part(from, from == it.first);
                if (n > 1 && !dead) sum(it.first, from, stride, n, place, it.b, it.h);
                if (final) break;
                __syncthreads();
                if (threadIdx.x == 0) s_flag[k] = count_up(it.first, 16, groups);
                __syncthreads();
                if (s_flag[k] == 0) break;
                from = it.first;
                stride = group;
                n = groups;
                final = true;
            }
        }
    }
};

template <int D, typename T, bool E8, int NT>
__global__ void __launch_bounds__(DecodeCfg<D, E8, NT>::kThreads, DecodeCfg<D, E8, NT>::kCtasPerSm)
    decode_kernel(const DecodeArgs a) {
    using C = DecodeCfg<D, E8, NT>;
    using M = typename std::conditional<E8, __half, T>::type;  // type of the products' operands
    constexpr int kDT = D / 16, kRows = C::kRows;
    __shared__ int s_dead, s_flag[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int n_ctas = gridDim.x / a.row_blocks, cta = blockIdx.x / a.row_blocks, row_block = blockIdx.x - cta * a.row_blocks;
    const int row0 = row_block * kRows;
    if (tid == 0) s_dead = *reinterpret_cast<volatile int*>(a.status);  // (one reading for the whole CTA)

    // ---- this CTA's piece of the line of units; each warp finds it for itself
    // (in the line an item is its units behind kItemCost places that stand for its own cost)
    unsigned int u0, u1, piece;
    DecodeCursor<C::kUnit, C::kItemCost> cc;
    {
        const int per_lane = (a.B + 31) / 32, b_lo = lane * per_lane;
        unsigned int mine = 0, rows_at_all = 0;
#pragma unroll 8
        for (int b = b_lo; b < min(b_lo + per_lane, a.B); ++b) {
            const int n = __ldg(a.lengths + b);
            if (n > a.c.capacity) report(a.status, kStatusBadLength);
            if (a.cos != nullptr && n > a.n_pos) report(a.status, kStatusBadPosition);
            if (n > 0) mine += units_of<C::kUnit>(min(n, a.c.capacity)) + C::kItemCost;
            rows_at_all += n > 0;
        }
        unsigned int before = mine;  // inclusive sums
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const unsigned int x = __shfl_up_sync(0xffffffffu, before, d);
            if (lane >= d) before += x;
        }
        const unsigned int sum = __shfl_sync(0xffffffffu, before, 31), total = sum * a.Hkv;  // (the host has seen to it that this fits)
        const unsigned int average = sum / max(__reduce_add_sync(0xffffffffu, rows_at_all), 1u);
        const unsigned int least = average <= kDecWhole / (C::kTiles * (D / 128)) + C::kItemCost ? average : 1 + C::kItemCost;
        piece = max((total + n_ctas - 1) / n_ctas, max(least, 1u));
        u0 = piece * cta;
        u1 = min(u0 + piece, total);
        before -= mine;
        const unsigned int here = __ballot_sync(0xffffffffu, u0 < total && before * a.Hkv <= u0 && u0 < (before + mine) * a.Hkv);
        int b = b_lo;
        if (here >> lane & 1) {
            for (;;) {
                const int rows = cached_rows(a, b);
                const unsigned int n = rows > 0 ? units_of<C::kUnit>(rows) + C::kItemCost : 0;
                if (u0 < (before + n) * a.Hkv) break;
                before += n;
                ++b;
            }
        }
        const int src = here == 0 ? 0 : __ffs(here) - 1;
        cc.b = __shfl_sync(0xffffffffu, b, src);
        const unsigned int in_b = u0 - __shfl_sync(0xffffffffu, before, src) * a.Hkv;
        cc.left = 0;
        if (here != 0) {
            cc.len = cached_rows(a, cc.b);
            cc.nt = units_of<C::kUnit>(cc.len);
            cc.h = in_b / (cc.nt + C::kItemCost);
            cc.t = static_cast<int>(in_b - cc.h * (cc.nt + C::kItemCost)) - C::kItemCost;
            cc.left = u1 - u0;
            if (cc.t < 0) {  // in front of the item's first unit
                cc.left += cc.t;
                cc.t = 0;
            }
        }
    }
    auto empty_rows = [&] {  // sequences without rows have no units: their output is zero
        for (int b = blockIdx.x; b < a.B; b += gridDim.x)
            if (cached_rows(a, b) == 0)
                for (int i = tid; i < a.Hkv * a.G * (D / 8); i += C::kThreads)
                    reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + b * a.o_sb + (i / (D / 8)) * a.o_sh)[i % (D / 8)] =
                        make_uint4(0, 0, 0, 0);
    };
    if (cc.left <= 0) {  // (all warps of the CTA alike)
        __syncthreads();
        if (s_dead == 0) empty_rows();
        return;
    }
    // the broken items: the one that began before this piece (or fills it), and the one that begins in it and goes on
    DecodeBroken broken[2] = {{-1, 0, 0, 0}, {-1, 0, 0, 0}};
    auto cta_of = [&](unsigned int u) { return static_cast<int>(u / piece); };
    if (cc.t > 0) {
        const unsigned int from = u1 - cc.left - cc.t;  // the item's first unit
        broken[0] = {cta_of(from), cta_of(from + cc.nt - 1), cc.b, cc.h};
    }
    auto begins_and_goes_on = [&](int n) {  // n units of item cc are here
        if (cc.t == 0 && n < cc.nt)
            broken[1] = {cta, cta_of(u1 - cc.left + cc.nt - 1), cc.b, cc.h};
    };

    // ---- the warp's ring of slots: K rows, V rows, K rows ... of its steps (16-byte pieces xor-ed with the row so that
    // eight rows of a column block lie in different banks)
    extern __shared__ __align__(1024) unsigned char smem[];
    const uint32_t ring = smem_u32(smem) + warp * C::kSlots * C::kSlotBytes;
    unsigned char* const scales = smem + C::kSmemBytes - C::kScaleRingBytes + warp * C::kSlots * C::kScaleBytes;
    uint4* const frag = reinterpret_cast<uint4*>(smem + C::kRingBytes);
    float* const merge_o = reinterpret_cast<float*>(smem + C::kRingBytes + C::kQueryBytes);  // kCopies of [8][kPad]
    float* const merge_m = merge_o + C::kCopies * 8 * C::kPad;                               // [warps][rows]
    float* const merge_l = merge_m + C::kWarps * kRows;
    float* const back = merge_l + C::kWarps * kRows;                                         // [rows]
    unsigned char* const new_rows = smem + C::kSmemBytes - C::kScaleRingBytes - C::kNewBytes;  // K and V row of a new token

    QueryRows<D, T, NT, C::kWarps> rows;
    using R = Row<D, 32>;
    rows.load(a, cc, row0);
    typename R::Words gamma;
    if (a.gamma != nullptr) R::template load<false>(gamma, a.gamma, lane);

    auto pc = cc;
    constexpr int kLook = 32 / C::kTiles;        // units whose pages the lanes hold
    // lane i: page and row in it of the warp's i-th 16 keys of the units from table_at on
    int table_at = 0, my_page = 0, my_row = 0;
    int page[C::kTiles] = {}, page_row[C::kTiles] = {};  // of the unit that is being copied
    constexpr int kPieces = C::kRowBytes / 16, kRowsAtOnce = 32 / kPieces, kCopies = 16 / kRowsAtOnce;
    const int piece16 = lane % kPieces, r_lane = lane / kPieces;
    const uint32_t dst_lane = ring + r_lane * C::kRowBytes + ((piece16 ^ (r_lane & 7)) << 4);
    const uint64_t policy = evict_first_policy();
    // this lane's place in row 0 of page 0 of the item's head, and the scales of that row
    const unsigned char *k_src = nullptr, *v_src = nullptr, *ks_src = nullptr, *vs_src = nullptr;
    auto head_sources = [&] {
        k_src = a.c.k + wide(pc.h, a.c.k_sh) + wide(r_lane, a.c.k_ss) + piece16 * 16;
        v_src = a.c.v + wide(pc.h, a.c.v_sh) + wide(r_lane, a.c.v_ss) + piece16 * 16;
        if constexpr (E8) {
            ks_src = a.c.k_scale + wide(pc.h, a.c.ks_sh);
            vs_src = a.c.v_scale + wide(pc.h, a.c.vs_sh);
        }
    };
    // a step's rows of the pool to a slot; rows behind the sequence become zeros, whatever the page holds there
    auto copy_rows = [&](int slot, const unsigned char* pool, int sp, int ss, const unsigned char* scale, int scale_sp) {
        int n = pc.len - (pc.t * C::kUnit + warp * C::kKeys);
        if (n <= 0) return;
        n -= a.new_k != nullptr;  // (the last row is not in the cache yet)
#pragma unroll
        for (int tile = 0; tile < C::kTiles; ++tile) {
            const unsigned char* const src = pool + wide(page[tile], sp) + wide(page_row[tile], ss);
            const uint32_t base = dst_lane + slot * C::kSlotBytes + tile * 16 * C::kRowBytes;
            auto dst = [&](int i) {  // row r_lane + i * kRowsAtOnce (r_lane is below kRowsAtOnce, a power of two)
                return (base ^ ((i * kRowsAtOnce & 7) << 4)) + i * kRowsAtOnce * C::kRowBytes;
            };
            if (n >= 16 * (tile + 1) && ss == C::kRowBytes) {
                each_index([&](auto i) {
                    constexpr int kI = decltype(i)::value, kStep = kI * kRowsAtOnce * C::kRowBytes;
                    cp_async16<kStep, kStep>(base ^ ((kI * kRowsAtOnce & 7) << 4), src, policy);
                }, std::make_integer_sequence<int, kCopies>{});
            } else {
#pragma unroll 1
                for (int i = 0; i < kCopies; ++i) {
                    const bool take = r_lane + i * kRowsAtOnce < n - 16 * tile;
                    cp_async16_or_zero(dst(i), src + (take ? wide(i * kRowsAtOnce, ss) : 0), take);
                }
            }
            if constexpr (E8) {  // (all 16 scales: a page holds a multiple of 16 rows)
                if (lane == 0)
                    cp_async16<0, 0>(smem_u32(scales) + slot * C::kKeys + 16 * tile,
                                     scale + wide(page[tile], scale_sp) + page_row[tile], policy);
            }
        }
    };
    // this lane's page, and row in it, of the units of an item from `first` on; looked at when K rows are asked for
    auto page_of = [&](const auto& item, int first, int& row) {
        const int unit = first + lane / C::kTiles, key = unit * C::kUnit + warp * C::kKeys + lane % C::kTiles * 16;
        row = 0;
        if (unit >= item.nt || key >= item.len) return 0;
        const int i = key / a.c.page_size;
        row = key - i * a.c.page_size;
        return __ldg(a.c.pages + item.b * a.c.pages_sb + i);
    };
    auto look_up = [&] {
        table_at = pc.t;
        my_page = page_of(pc, pc.t, my_row);
    };
    int next_page = 0, next_row = 0;  // the first ones of the item after pc's
    auto look_ahead = [&] {
        auto next = pc;
        next.left -= next.nt - next.t;
        if (next.left > 0) next.next_item(a);
        if (next.left > 0) next_page = page_of(next, 0, next_row);
    };
    auto issue_k = [&](int slot) {
        if (pc.left > 0) {
#pragma unroll
            for (int tile = 0; tile < C::kTiles; ++tile) {
                page[tile] = __shfl_sync(0xffffffffu, my_page, (pc.t - table_at) * C::kTiles + tile);
                page_row[tile] = __shfl_sync(0xffffffffu, my_row, (pc.t - table_at) * C::kTiles + tile);
                if (static_cast<unsigned>(page[tile]) >= static_cast<unsigned>(a.c.n_pages)) {
                    if (lane == 0) report(a.status, kStatusBadPage);
                    page[tile] = 0;  // (what the call gives is not to be trusted then)
                }
            }
            copy_rows(slot, k_src, a.c.k_sp, a.c.k_ss, ks_src, a.c.ks_sp);
        }
        cp_async_commit();
    };
    auto issue_v = [&](int slot) {
        if (pc.left > 0) {
            copy_rows(slot, v_src, a.c.v_sp, a.c.v_ss, vs_src, a.c.vs_sp);
            ++pc.t;
            --pc.left;
            if (pc.t == pc.nt && pc.left > 0) {
                pc.next_item(a);
                if (pc.left > 0) {
                    head_sources();
                    if constexpr (C::kLookAhead) {
                        table_at = 0;
                        my_page = next_page;
                        my_row = next_row;
                        look_ahead();
                    } else {
                        look_up();
                    }
                }
            } else if (pc.t - table_at == kLook) {
                look_up();
            }
        }
        cp_async_commit();
    };
    head_sources();
    look_up();
    if constexpr (C::kLookAhead) look_ahead();
#pragma unroll 1
    for (int s = 0; s < C::kSlots - 1; s += 2) {
        issue_k(s);
        if (s + 1 < C::kSlots - 1) issue_v(s + 1);
    }
    // A step's two halves: wait for the slot, refill the one before it, which all lanes are done with.
    int slot = 0;
    auto arrive = [&](auto v) {  // v: true for the V half
        constexpr bool kIsV = decltype(v)::value;
        cp_async_wait<C::kSlots - 2>();
        __syncwarp();
        const int freed = slot == 0 ? C::kSlots - 1 : slot - 1;
        if constexpr ((C::kSlots % 2 == 1) != kIsV) issue_k(freed);
        else issue_v(freed);
    };
    auto leave = [&] { slot = slot + 1 == C::kSlots ? 0 : slot + 1; };

    const DecodeJoin<D, T, E8, NT> join{a, reinterpret_cast<float*>(smem), s_flag, cta, row_block};
    if (tid == 0) s_flag[0] = s_flag[1] = 0;
    rows.template prepare<E8>(a, gamma, frag, back);
    __syncthreads();
    if (s_dead != 0) {  // nothing is written; only the joins are counted on, other CTAs may complete them
        cp_async_wait<0>();
        while (cc.left > 0) {
            const int n = min(cc.nt - cc.t, cc.left);
            if (n <= 0) break;
            begins_and_goes_on(n);
            cc.t += n;
            cc.left -= n;
            if (cc.left > 0) cc.next_item(a);
        }
        if (tid == 0)
#pragma unroll 1
            for (int k = 0; k < 2; ++k) s_flag[k] = broken[k].first >= 0 && join.part_done(broken[k]);
        __syncthreads();
        join.run(broken, true);
        return;
    }
    empty_rows();

    // The new token's rows of an item, by the warp that has their step: into the cache and into new_rows.
    uint32_t new_ke = 0, new_ve = 0;  // scales' bytes
    auto prepare_new = [&] {
        const int pos = cc.len - 1, i = pos / a.c.page_size, row = pos - i * a.c.page_size;
        typename R::Words kw, vw, gk, c, s;
        const int pg = __ldg(a.c.pages + cc.b * a.c.pages_sb + i);
        R::template load<false>(kw, reinterpret_cast<const T*>(a.new_k) + cc.b * a.nk_sb + cc.h * a.nk_sh, lane);
        R::template load<false>(vw, reinterpret_cast<const T*>(a.new_v) + cc.b * a.nv_sb + cc.h * a.nv_sh, lane);
        if (a.gamma_k != nullptr) R::template load<false>(gk, a.gamma_k, lane);
        bool write = row_block == 0 && __ldg(a.lengths + cc.b) <= a.c.capacity;
        if (a.cos != nullptr) {
            write = write && pos < a.n_pos;
            const long long at = static_cast<long long>(min(pos, a.n_pos - 1)) * D;
            R::template load<false>(c, reinterpret_cast<const T*>(a.cos) + at, lane);
            R::template load<false>(s, reinterpret_cast<const T*>(a.sin) + at, lane);
        }
        // (reported by the copies of the step)
        if (static_cast<unsigned>(pg) >= static_cast<unsigned>(a.c.n_pages)) write = false;
        R k, v;
        k.template unpack<T>(kw);
        v.template unpack<T>(vw);
        if (a.gamma_k != nullptr) k.template norm<T>(gk, a.eps);
        if (a.cos != nullptr) k.template rotate<T>(c, s);
        auto to = [&](unsigned char* dst, unsigned char* pool) {
            return [=](int at, auto value) {
                *reinterpret_cast<decltype(value)*>(dst + at) = value;
                if (write) *reinterpret_cast<decltype(value)*>(pool + at) = value;
            };
        };
        const int p = write ? pg : 0;
        unsigned char* const k_to = a.c.k + wide(p, a.c.k_sp) + wide(cc.h, a.c.k_sh) + wide(row, a.c.k_ss);
        unsigned char* const v_to = a.c.v + wide(p, a.c.v_sp) + wide(cc.h, a.c.v_sh) + wide(row, a.c.v_ss);
        new_ke = k.template store<T, E8>(lane, to(new_rows, k_to));
        new_ve = v.template store<T, E8>(lane, to(new_rows + C::kRowBytes, v_to));
        if (E8 && write && lane == 0) {
            a.c.k_scale[wide(p, a.c.ks_sp) + wide(cc.h, a.c.ks_sh) + row] = static_cast<unsigned char>(new_ke);
            a.c.v_scale[wide(p, a.c.vs_sp) + wide(cc.h, a.c.vs_sh) + row] = static_cast<unsigned char>(new_ve);
        }
        __syncwarp();
    };
    // and from there behind the cached rows of the step in `slot`
    auto place_new = [&](int slot, int v) {
        const int r = (cc.len - 1) % C::kKeys;
        if (lane < kPieces)
            *reinterpret_cast<uint4*>(smem + (warp * C::kSlots + slot) * C::kSlotBytes + r * C::kRowBytes + ((lane ^ (r & 7)) << 4)) =
                *reinterpret_cast<const uint4*>(new_rows + v * C::kRowBytes + lane * 16);
        if (E8 && lane == 0) scales[slot * C::kKeys + r] = static_cast<unsigned char>(v ? new_ve : new_ke);
        __syncwarp();
    };

    // ldmatrix: the row (key) of the slot and the 16-byte piece that this lane names; piece + 2 j lies 32 j bytes further,
    // xor-ed below 128 bytes
    const int q8 = lane >> 3;
    const int k_row = (q8 & 1) * 8 + (lane & 7), k_piece = q8 >> 1;
    const int v_row = E8 ? k_row : (q8 >> 1) * 8 + (lane & 7), v_piece = E8 ? k_piece : (q8 & 1);
    const uint32_t k_lane = ring + k_row * C::kRowBytes + ((k_piece ^ (k_row & 7)) << 4);
    const uint32_t v_lane = ring + v_row * C::kRowBytes + ((v_piece ^ (v_row & 7)) << 4);
    auto step32 = [](uint32_t at, int j) { return (at ^ ((j & 3) << 5)) + (j >> 2) * 128; };
    // Probabilities are 2^(score - base + kUp), the base at most kSlack behind the largest score so far: up to 2^15 in f16,
    // whose smallest step is then 2^-35 of the largest probability, up to 2^-12 in bf16, so that a sum over 4096 of the
    // largest bf16 values is still finite (values below 2^-106 lose bits for it).
    constexpr bool kHalf = std::is_same<M, __half>::value;
    constexpr bool kSplit = kSplitProducts<T, E8>;
    constexpr float kSlack = kHalf ? 4.f : 8.f, kUp = kHalf ? 11.f : -20.f;

    while (cc.left > 0) {
        // ---- one item's part: units cc.t .. cc.t + n - 1
        const int n = min(cc.nt - cc.t, cc.left);
        if (n <= 0) break;
        const int h = cc.h;
        auto nc = cc;  // the item after this one: its query rows are on their way meanwhile
        nc.t += n;
        nc.left -= n;
        if (nc.left > 0) nc.next_item(a);
        if (nc.left > 0) rows.load(a, nc, row0);
        uint4 qf[C::kQueryInRegs ? NT : 1][C::kQueryInRegs ? kDT : 1];
        if constexpr (C::kQueryInRegs) {
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int j = 0; j < kDT; ++j) qf[u][j] = frag[(u * kDT + j) * 32 + lane];
        }
        float mul[NT][2];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
            mul[u][0] = E8 ? back[u * 8 + 2 * t4] : a.scale_log2e;
            mul[u][1] = E8 ? back[u * 8 + 2 * t4 + 1] : a.scale_log2e;
        }
        // m, mv: bases of the sum and of O (an 8-bit cache's value scales belong to the latter), -inf before the first key
        float o[NT][kDT][4], m[NT][2], mv[NT][2], l[NT][2];
        float off[NT][2], off_v[NT][2];  // kUp - base, what is added to a score
        float lim[NT][2], lim_v[NT][2];  // base + kSlack: a score above it moves the base
#pragma unroll
        for (int u = 0; u < NT; ++u) {
#pragma unroll
            for (int i = 0; i < kDT; ++i) o[u][i][0] = o[u][i][1] = o[u][i][2] = o[u][i][3] = 0.f;
            m[u][0] = m[u][1] = mv[u][0] = mv[u][1] = -INFINITY;
            off[u][0] = off[u][1] = off_v[u][0] = off_v[u][1] = 0.f;
            lim[u][0] = lim[u][1] = lim_v[u][0] = lim_v[u][1] = -INFINITY;
            l[u][0] = l[u][1] = 0.f;
        }
        // the new token's step is the last one with keys, in the item's last unit
        const bool has_new = a.new_k != nullptr && cc.t + n == cc.nt && warp == (cc.len - 1) % C::kUnit / C::kKeys;
        if (has_new) prepare_new();
        for (int i_unit = 0; i_unit < n; ++i_unit) {
            const int keys = cc.len - ((cc.t + i_unit) * C::kUnit + warp * C::kKeys);  // of the sequence, from this step's first on
            arrive(std::false_type{});
            // scores of keys g (0, 1), g + 8 (2, 3) of each 16 and heads 2 t4, 2 t4 + 1
            float x[NT][C::kTiles][4], w[NT][C::kTiles][4];
            if (has_new && i_unit == n - 1) place_new(slot, 0);
            if (keys > 0) {
                float s[NT][C::kTiles][2][4];  // high and low part of q': chains of products of their own
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int tile = 0; tile < C::kTiles; ++tile)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[u][tile][0][i] = s[u][tile][1][i] = 0.f;
                auto product = [&](int tile, int j, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                    for (int u = 0; u < NT; ++u) {
                        uint4 f;
                        if constexpr (C::kQueryInRegs) f = qf[u][j];
                        else f = frag[(u * kDT + j) * 32 + lane];
                        mma16816<M>(s[u][tile][0], a0, a1, a2, a3, f.x, f.y);
                        if constexpr (kSplit) mma16816<M>(s[u][tile][1], a0, a1, a2, a3, f.z, f.w);
                    }
                };
                float scale = 1.f;  // of key `lane` of the step (with steps of 16 keys, twice)
                if constexpr (E8) scale = scale_value(scales[slot * C::kKeys + lane % C::kKeys]);
                const uint32_t k_at = k_lane + slot * C::kSlotBytes;
#pragma unroll
                for (int j = 0; j < kDT; j += E8 ? 2 : 1)
#pragma unroll
                    for (int tile = 0; tile < C::kTiles; ++tile) {
                        uint32_t r[4];
                        ldmatrix4(r, step32(k_at, E8 ? j / 2 : j) + tile * 16 * C::kRowBytes);
                        if constexpr (E8) {
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                uint32_t a0, a1, a2, a3;
                                widen4(r[2 * y], a0, a2);
                                widen4(r[2 * y + 1], a1, a3);
                                product(tile, j + y, a0, a1, a2, a3);
                            }
                        } else {
                            product(tile, j, r[0], r[1], r[2], r[3]);
                        }
                    }
#pragma unroll
                for (int tile = 0; tile < C::kTiles; ++tile) {
                    float f0 = 1.f, f1 = 1.f;  // scales of the keys
                    if constexpr (E8) {
                        f0 = __shfl_sync(0xffffffffu, scale, 16 * tile + g);
                        f1 = __shfl_sync(0xffffffffu, scale, 16 * tile + g + 8);
                    }
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[u][tile][i] = (kSplit ? s[u][tile][0][i] + s[u][tile][1][i] : s[u][tile][0][i]) * mul[u][i & 1];
                            if constexpr (E8) x[u][tile][i] *= i < 2 ? f0 : f1;
                        }
                }
                if (keys < C::kKeys) {
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int i = 0; i < 4 * C::kTiles; ++i)
                            if (g + 8 * (i >> 1) >= keys) x[u][i / 4][i % 4] = -INFINITY;
                }
            }
            leave();
            arrive(std::true_type{});
            if (has_new && i_unit == n - 1) place_new(slot, 1);
            if (keys > 0) {
                bool above = false;
                if constexpr (E8) {
                    // exponent of value row `lane` of the step (2^23 + e as bits: e - 127 without a conversion)
                    const uint32_t e = scales[slot * C::kKeys + lane % C::kKeys];
                    const float exponent = e == 255 ? NAN : __uint_as_float(0x4b000000u | e) - 8388735.f;
#pragma unroll
                    for (int tile = 0; tile < C::kTiles; ++tile) {
                        const float ve0 = __shfl_sync(0xffffffffu, exponent, 16 * tile + g);
                        const float ve1 = __shfl_sync(0xffffffffu, exponent, 16 * tile + g + 8);
#pragma unroll
                        for (int u = 0; u < NT; ++u)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                w[u][tile][i] = x[u][tile][i] + (i < 2 ? ve0 : ve1);
                                above |= w[u][tile][i] > lim_v[u][i & 1];
                            }
                    }
                    if (keys < C::kKeys) {  // (scales behind the sequence are whatever the page holds)
#pragma unroll
                        for (int u = 0; u < NT; ++u)
#pragma unroll
                            for (int i = 0; i < 4 * C::kTiles; ++i)
                                if (g + 8 * (i >> 1) >= keys) w[u][i / 4][i % 4] = -INFINITY;
                    }
                }
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int i = 0; i < 4 * C::kTiles; ++i) above |= x[u][i / 4][i % 4] > lim[u][i & 1];
                if (__any_sync(0xffffffffu, above)) {  // move the bases (of the heads whose own scores ask for it) to the maxima
                    auto top = [](const float (&y)[C::kTiles][4], int c, float base) {
                        float z = fmaxf(y[0][c], y[0][c + 2]);
#pragma unroll
                        for (int tile = 1; tile < C::kTiles; ++tile) z = fmaxf(z, fmaxf(y[tile][c], y[tile][c + 2]));
                        z = fmaxf(z, __shfl_xor_sync(0xffffffffu, z, 4));
                        z = fmaxf(z, __shfl_xor_sync(0xffffffffu, z, 8));
                        z = fmaxf(z, __shfl_xor_sync(0xffffffffu, z, 16));
                        return z > base + kSlack ? z : base;
                    };
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float to = top(x[u], c, m[u][c]);
                            const float to_v = E8 ? top(w[u], c, mv[u][c]) : to;
                            l[u][c] *= m[u][c] == -INFINITY ? 0.f : ex2(m[u][c] - to);
                            const float f = mv[u][c] == -INFINITY ? 0.f : ex2(mv[u][c] - to_v);
#pragma unroll
                            for (int i = 0; i < kDT; ++i) {
                                o[u][i][c] *= f;
                                o[u][i][c + 2] *= f;
                            }
                            m[u][c] = to;
                            mv[u][c] = to_v;
                            off[u][c] = to == -INFINITY ? 0.f : kUp - to;
                            off_v[u][c] = to_v == -INFINITY ? 0.f : kUp - to_v;
                            lim[u][c] = to + kSlack;
                            lim_v[u][c] = to_v + kSlack;
                        }
                }
                uint32_t pb[NT][C::kTiles][4];  // high and low part of the probabilities of keys 0-7, 8-15
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int tile = 0; tile < C::kTiles; ++tile) {
                        float(&p)[4] = w[u][tile];
                        uint32_t(&b)[4] = pb[u][tile];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float y = ex2(x[u][tile][i] + off[u][i & 1]);
                            l[u][i & 1] += y;
                            p[i] = E8 ? ex2(p[i] + off_v[u][i & 1]) : y;
                        }
                        if constexpr (kSplit) {
                            split2_probabilities<M, !E8>(p[0], p[1], b[0], b[2]);
                            split2_probabilities<M, !E8>(p[2], p[3], b[1], b[3]);
                        } else {
                            b[0] = Num<M>::pack(p[0], p[1]);
                            b[1] = Num<M>::pack(p[2], p[3]);
                        }
#pragma unroll
                        for (int i = 0; i < (kSplit ? 4 : 2); ++i) b[i] = transpose8x8(b[i]);
                    }
                auto product = [&](int tile, int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                    for (int u = 0; u < NT; ++u) {
                        mma16816<M>(o[u][i], a0, a1, a2, a3, pb[u][tile][0], pb[u][tile][1]);
                        if constexpr (kSplit) mma16816<M>(o[u][i], a0, a1, a2, a3, pb[u][tile][2], pb[u][tile][3]);
                    }
                };
                const uint32_t v_at = v_lane + slot * C::kSlotBytes;
#pragma unroll
                for (int tile = 0; tile < C::kTiles; ++tile)
#pragma unroll
                    for (int i = 0; i < kDT; i += E8 ? 2 : 1) {
                        uint32_t r[4];
                        ldmatrix4_trans(r, step32(v_at, E8 ? i / 2 : i) + tile * 16 * C::kRowBytes);
                        if constexpr (E8) {
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                // bytes {key 2t col 2g, key 2t col 2g+1, key 2t+1 col 2g, key 2t+1 col 2g+1}
                                uint32_t a0, a1, a2, a3;
                                widen4(__byte_perm(r[2 * y], 0, 0x3120), a0, a1);
                                widen4(__byte_perm(r[2 * y + 1], 0, 0x3120), a2, a3);
                                product(tile, i + y, a0, a1, a2, a3);
                            }
                        } else {
                            product(tile, i, r[0], r[1], r[2], r[3]);
                        }
                    }
            }
            leave();
        }

        // ---- the warps' parts of the item together
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
        const bool whole = n == cc.nt;
        auto top_of = [&](int r) {  // base of row r over the warps
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < C::kWarps; ++w) top = fmaxf(top, merge_m[w * kRows + r]);
            return top;
        };
        auto sum_of = [&](int r, float top) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < C::kWarps; ++w) {
                const float lw = merge_l[w * kRows + r];
                sum += lw == 0.f ? 0.f : lw * ex2(merge_m[w * kRows + r] - (top == -INFINITY ? 0.f : top));
            }
            return sum;
        };
        // what makes means of sums; no weight at all: the whole item is undefined, a part counts for nothing
        auto inverse = [&](float sum) { return sum != 0.f ? 1.f / sum : whole ? NAN : 0.f; };
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = u * 8 + 2 * t4 + c;
                const float top = top_of(r), by = mv[u][c] - (top == -INFINITY ? 0.f : top);
                // To the common base.  That gives an 8-bit cache's values their scale back (up to 2^127), so they are divided by the
                // sum first: what is added up from then on is at most the largest value.  (In two halves, as the factor itself
                // may be more than 32 bits hold.)
                const float f = mv[u][c] == -INFINITY ? 0.f : ex2(E8 ? 0.5f * by : by);
                const float first = E8 ? f * inverse(sum_of(r, top)) : f;
#pragma unroll
                for (int i = 0; i < kDT; ++i)
#pragma unroll
                    for (int k = c; k < 4; k += 2) o[u][i][k] = E8 ? o[u][i][k] * first * f : o[u][i][k] * f;
            }
        begins_and_goes_on(n);
        float* const part = join.part(cta, cc.t == 0);
        float* const copy = merge_o + warp % C::kCopies * 8 * C::kPad;
        // eight rows and kMergeCols columns at a time: the last kCopies warps leave theirs, the ones before add theirs, all add the
        // copies
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int c0 = 0; c0 < D; c0 += C::kMergeCols) {
                auto each = [&](auto&& f) {  // f(place in a copy, value)
#pragma unroll
                    for (int i = 0; i < C::kMergeCols / 16; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            f((2 * t4 + (k & 1)) * C::kPad + 16 * i + (E8 ? 2 * g + (k >> 1) : g + 8 * (k >> 1)),
                              o[u][c0 / 16 + i][k]);
                };
                if (warp >= C::kWarps - C::kCopies) each([&](int at, float x) { copy[at] = x; });
                __syncthreads();
                // (all are done with the old ones)
                if (u == 0 && c0 == 0 && nc.left > 0) rows.template prepare<E8>(a, gamma, frag, back);
#pragma unroll 1
                for (int w = C::kWarps - 2 * C::kCopies; w >= 0; w -= C::kCopies) {
                    if (warp / C::kCopies * C::kCopies == w) each([&](int at, float x) { copy[at] += x; });
                    __syncthreads();
                }
                for (int i = tid; i < 8 * (C::kMergeCols / 4); i += C::kThreads) {
                    const int r8 = i / (C::kMergeCols / 4), d8 = (i % (C::kMergeCols / 4)) * 4, r = u * 8 + r8, d = c0 + d8;
                    if (row0 + r >= a.G) break;  // (rows go up with i)
                    float4 z = *reinterpret_cast<const float4*>(merge_o + r8 * C::kPad + d8);
#pragma unroll
                    for (int i = 1; i < C::kCopies; ++i) {
                        const float4 y = *reinterpret_cast<const float4*>(merge_o + (8 * i + r8) * C::kPad + d8);
                        z = make_float4(z.x + y.x, z.y + y.y, z.z + y.z, z.w + y.w);
                    }
                    const float top = top_of(r), sum = sum_of(r, top), inv = E8 ? 1.f : inverse(sum);
                    z = make_float4(z.x * inv, z.y * inv, z.z * inv, z.w * inv);
                    if (whole) {
                        T* const dst = reinterpret_cast<T*>(a.out) + cc.b * a.o_sb + (h * a.G + row0 + r) * a.o_sh + d;
                        *reinterpret_cast<uint2*>(dst) = make_uint2(Num<T>::pack(z.x, z.y), Num<T>::pack(z.z, z.w));
                    } else {
                        *reinterpret_cast<float4*>(part + r * D + d) = z;
                        if (d == 0) part_weight(part + kRows * D + r, part + kRows * D + kRows + r, top, sum);
                    }
                }
                __syncthreads();  // the copies are free
            }
        // A part counts as soon as it is written.  At the end of the pieces, which all CTAs reach at about the same time, a CTA
        // is then hardly ever the last one of two items (16 sequences of 8192 rows, 16 heads: 33.5 -> 29.5 us).
        if (!whole && tid == 0) s_flag[cc.t == 0] = join.part_done(cc.t == 0 ? broken[1] : broken[0]);
        cc = nc;
    }
    cp_async_wait<0>();  // (the ring serves the joins)
    __syncthreads();
    join.run(broken, false);
}

}  // namespace kf
