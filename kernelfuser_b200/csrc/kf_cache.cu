// C-ABI entry points of the serving operators (declared in include/kf_b200.h): rows into a paged key-value cache, out of
// it, and the attention of one new token over it.  Host-side argument checks and kernel launches only.
#include "../../include/kf_b200.h"
#include "host.cuh"
#include "cache_rows.cuh"
#include "decode_attn.cuh"

using namespace kf::host;

namespace {

constexpr int64_t kMaxRows = 1 << 30;  // of a sequence, and of a batch: indexes stay in 32 bits

int check_sizes(const char* what, int64_t n, int64_t most) {
    if (n < 1 || n > most) return fail(KF_EINVAL, "%s must be in [1, %lld] (got %lld)", what, (long long)most, (long long)n);
    return KF_OK;
}

// Element stride of a dimension of extent n: a positive multiple of `step` elements (16 bytes).  That of a single entry is
// never used.
bool step_ok(int64_t s, int64_t n, int64_t step) { return n == 1 || (s % step == 0 && s > 0); }

int cache_view(const kf_paged_cache& c, int64_t dtype, kf::CacheView* out) {
    if (dtype != KF_BF16 && dtype != KF_FP16) return fail(KF_EINVAL, "dtype must be KF_BF16 or KF_FP16");
    if (c.dtype != KF_E4M3 && c.dtype != dtype) return fail(KF_EINVAL, "the cache must hold the tensors' dtype or KF_E4M3");
    if (c.D != 128 && c.D != 256) return fail(KF_EINVAL, "head dim must be 128 or 256 (got %lld)", (long long)c.D);
    if (int r = check_sizes("n_pages", c.n_pages, kMaxRows)) return r;
    if (int r = check_sizes("max_pages", c.max_pages, kMaxRows)) return r;
    if (int r = check_sizes("Hkv", c.Hkv, 1 << 16)) return r;
    if (c.page_size < 16 || c.page_size > kMaxRows || c.page_size % 16)
        return fail(KF_EINVAL, "page_size must be a positive multiple of 16 (got %lld)", (long long)c.page_size);
    if (!c.k || !c.v || !c.pages) return fail(KF_EINVAL, "the cache's k, v and pages must not be NULL");
    if (!aligned16(c.k) || !aligned16(c.v)) return fail(KF_EALIGN, "pointers must be 16-byte aligned");
    const bool e8 = c.dtype == KF_E4M3;
    const int64_t step = e8 ? 16 : 8, size = e8 ? 1 : 2;
    const int64_t strides[6] = {c.k_stride_page, c.k_stride_head, c.k_stride_row,
                                c.v_stride_page, c.v_stride_head, c.v_stride_row};
    const int64_t extents[3] = {c.n_pages, c.Hkv, c.page_size};
    for (int i = 0; i < 6; ++i)
        if (!step_ok(strides[i], extents[i % 3], step))
            return fail(KF_EALIGN, "cache strides must be positive multiples of 16 bytes");
    if (c.k_stride_row < c.D || c.v_stride_row < c.D) return fail(KF_EINVAL, "row stride must be at least D");
    if (e8) {
        if (!c.k_scale || !c.v_scale) return fail(KF_EINVAL, "an e4m3 cache needs k_scale and v_scale");
        if (!aligned16(c.k_scale) || !aligned16(c.v_scale)) return fail(KF_EALIGN, "pointers must be 16-byte aligned");
        const int64_t s[4] = {c.k_scale_stride_page, c.k_scale_stride_head, c.v_scale_stride_page, c.v_scale_stride_head};
        for (int i = 0; i < 4; ++i)
            if (!step_ok(s[i], extents[i % 2], 16))
                return fail(KF_EALIGN, "scale strides must be positive multiples of 16");
    }
    if (c.pages_stride < 0) return fail(KF_EINVAL, "pages_stride must not be negative");
    kf::CacheView& v = *out;
    v.k = static_cast<unsigned char*>(c.k);
    v.v = static_cast<unsigned char*>(c.v);
    v.k_scale = static_cast<unsigned char*>(c.k_scale);
    v.v_scale = static_cast<unsigned char*>(c.v_scale);
    // in bytes; below 2^31 each (that of a single entry may be anything: it is never used)
    const int64_t from[10] = {c.k_stride_page * size, c.k_stride_head * size, c.k_stride_row * size, c.v_stride_page * size,
                              c.v_stride_head * size, c.v_stride_row * size, c.k_scale_stride_page, c.k_scale_stride_head,
                              c.v_scale_stride_page, c.v_scale_stride_head};
    int* const to[10] = {&v.k_sp, &v.k_sh, &v.k_ss, &v.v_sp, &v.v_sh, &v.v_ss, &v.ks_sp, &v.ks_sh, &v.vs_sp, &v.vs_sh};
    for (int i = 0; i < 10; ++i) {
        const bool one = extents[i < 6 ? i % 3 : i % 2] == 1, used = !one && (i < 6 || e8);
        if (used && from[i] > 0x7fffffff) return fail(KF_EINVAL, "cache strides must be below 2^31 bytes");
        *to[i] = used ? (int)from[i] : 0;
    }
    v.pages = c.pages;
    v.pages_sb = c.pages_stride;
    v.n_pages = static_cast<int>(c.n_pages);
    v.page_size = static_cast<int>(c.page_size);
    v.max_pages = static_cast<int>(c.max_pages);
    const int64_t rows = c.max_pages * c.page_size;
    v.capacity = static_cast<int>(rows < kMaxRows ? rows : kMaxRows);
    return KF_OK;
}

int check_rows(const char* what, const void* p, int64_t B, int64_t H, int64_t S, int64_t D, int64_t sb, int64_t sh,
               int64_t ss) {
    if (!p) return fail(KF_EINVAL, "%s must not be NULL", what);
    if (!aligned16(p)) return fail(KF_EALIGN, "pointers must be 16-byte aligned");
    if (!step_ok(sb, B, 8) || !step_ok(sh, H, 8) || !step_ok(ss, S, 8))
        return fail(KF_EALIGN, "strides must be positive multiples of 8 elements");
    if (S > 1 && ss < D) return fail(KF_EINVAL, "row stride must be at least D");
    return KF_OK;
}

int check_tables(const void* gamma, const void* cos_table, const void* sin_table, int64_t n_positions) {
    if ((cos_table == nullptr) != (sin_table == nullptr)) return fail(KF_EINVAL, "provide both rotary tables or neither");
    if (!aligned16(gamma) || !aligned16(cos_table) || !aligned16(sin_table))
        return fail(KF_EALIGN, "pointers must be 16-byte aligned");
    if (cos_table) return check_sizes("n_positions", n_positions, 0x7fffffff);
    return KF_OK;
}

int launched(const char* what, cudaError_t e) {
    return e == cudaSuccess ? KF_OK : fail(KF_ECUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
}

template <int D, typename T, bool E8> int launch_append(const kf::AppendArgs& a, cudaStream_t st) {
    constexpr int kTasks = kf::kRowsThreads / (D / 16);
    const long long gx = (static_cast<long long>(a.B) * a.S + kTasks - 1) / kTasks;
    kf::AppendArgs args = a;
    // One head to a group of lanes while that is what spreads the rows over the SMs, several (the tables are then read once
    // for them, and as many rows are in flight) once there are two CTAs an SM that way.
    args.heads_per_group = gx * ((a.H + kf::kAppendHeads - 1) / kf::kAppendHeads) >= sm_count() ? kf::kAppendHeads : 1;
    const unsigned gy = (unsigned)((a.H + args.heads_per_group - 1) / args.heads_per_group);
    if (gy > 65535) return fail(KF_EINVAL, "too many heads");
    return launched("append_rows", launch_kernel(kf::append_rows_kernel<D, T, E8>, dim3((unsigned)gx, gy, 2),
                                                 dim3(kf::kRowsThreads), 0, st, args));
}

template <int D, typename T, bool E8> int launch_read(const kf::ReadArgs& a, cudaStream_t st) {
    constexpr int kRows = kf::read_block<D>() * kf::kReadBlocks;
    const unsigned gx = (unsigned)((a.S + kRows - 1) / kRows);
    const long long bh = static_cast<long long>(a.B) * a.H;
    return launched("read_rows", launch_kernel(kf::read_rows_kernel<D, T, E8>, dim3(gx, (unsigned)(bh < 65535 ? bh : 65535)),
                                               dim3(kf::kRowsThreads), 0, st, a));
}

// Words in which the CTAs of a decode launch count what has arrived for a join: a row of them per launch, zero between
// launches (in the library image; the CTA that completes a count takes it back).  Each stream has a row, and each captured launch.
constexpr int kMaxCtas = 512, kJoinSlots = 1024, kJoinGraphSlots = 4096;
__device__ unsigned int g_arrived[kJoinSlots + kJoinGraphSlots][kMaxCtas];
StreamSlots<kJoinSlots> g_join_slots;
GraphSlots<kJoinGraphSlots> g_join_graph_slots;

// NULL: every row is taken.
int join_words(cudaStream_t st, unsigned int** out) {
    static SymbolCache cache;
    void* p = nullptr;
    unsigned long long context = 0;
    cudaError_t e = symbol_address(cache, g_arrived, &p, &context);
    if (e != cudaSuccess) return fail(KF_ECUDA, "cudaGetSymbolAddress(join words) failed: %s", cudaGetErrorString(e));
    int slot = -1;
    if (int r = launch_slot<g_join_slots, g_join_graph_slots>(st, context, &slot)) return r;
    *out = slot < 0 ? nullptr : static_cast<unsigned int*>(p) + static_cast<size_t>(slot) * kMaxCtas;
    return KF_OK;
}

template <int D, bool E8, int NT> int decode_ctas() {
    const int n = sm_count() * kf::DecodeCfg<D, E8, NT>::kCtasPerSm;
    return n < kMaxCtas ? n : kMaxCtas;
}

template <int D, typename T, bool E8, int NT> int launch_decode_nt(const kf::DecodeArgs& a, cudaStream_t st) {
    constexpr auto kern = kf::decode_kernel<D, T, E8, NT>;
    constexpr int smem = kf::DecodeCfg<D, E8, NT>::kSmemBytes;
    cudaError_t e = allow_smem<kern>(smem);
    if (e != cudaSuccess) return fail(KF_ECUDA, "cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
    kf::DecodeArgs args = a;
    args.row_blocks = (a.G + 8 * NT - 1) / (8 * NT);
    // a CTA for each block of query rows of every piece of the line; no more pieces than the batch can have
    const long long items = static_cast<long long>(a.B) * a.Hkv, unit = kf::DecodeCfg<D, E8, NT>::kUnit;
    const long long per_item = (a.c.capacity + unit - 1) / unit;
    const long long most = items * (per_item + kf::DecodeCfg<D, E8, NT>::kItemCost);
    if (most > 0x7fffffffLL)
        return fail(KF_EINVAL, "the batch is too large: its page table can hold more than 2^31 pieces of 64 keys");
    const long long fit = decode_ctas<D, E8, NT>(), room = fit / args.row_blocks > 0 ? fit / args.row_blocks : 1;
    const long long pieces = items * per_item < room ? items * per_item : room;
    const unsigned grid = (unsigned)(pieces * args.row_blocks);
    if (pieces > 1) {
        if (int r = join_words(st, &args.arrived)) return r;
        if (args.arrived == nullptr) {  // then words in the workspace, cleared first
            args.arrived = reinterpret_cast<unsigned int*>(a.ws + kf::decode_part_at<D, E8, NT>((int)fit, 0));
            e = cudaMemsetAsync(args.arrived, 0, sizeof(unsigned int) * grid, st);
            if (e != cudaSuccess) return fail(KF_ECUDA, "cudaMemsetAsync failed: %s", cudaGetErrorString(e));
        }
    }
    return launched("decode_attention",
                    launch_kernel(kern, dim3(grid), dim3(kf::DecodeCfg<D, E8, NT>::kThreads), smem, st, args));
}

template <int D, typename T, bool E8> int launch_decode(const kf::DecodeArgs& a, cudaStream_t st) {
    return a.G <= 8 ? launch_decode_nt<D, T, E8, 1>(a, st) : launch_decode_nt<D, T, E8, 2>(a, st);
}

// f<D, T, E8>() for the sizes and types of a call
template <typename F> int by_type(int64_t D, int64_t dtype, bool e8, F&& f) {
    auto for_d = [&](auto d) {
        constexpr int kD = decltype(d)::value;
        if (dtype == KF_BF16)
            return e8 ? f.template operator()<kD, __nv_bfloat16, true>() : f.template operator()<kD, __nv_bfloat16, false>();
        return e8 ? f.template operator()<kD, __half, true>() : f.template operator()<kD, __half, false>();
    };
    return D == 128 ? for_d(std::integral_constant<int, 128>{}) : for_d(std::integral_constant<int, 256>{});
}
struct Append {
    const kf::AppendArgs& a;
    cudaStream_t st;
    template <int D, typename T, bool E8> int operator()() const { return launch_append<D, T, E8>(a, st); }
};
struct Read {
    const kf::ReadArgs& a;
    cudaStream_t st;
    template <int D, typename T, bool E8> int operator()() const { return launch_read<D, T, E8>(a, st); }
};
struct Decode {
    const kf::DecodeArgs& a;
    cudaStream_t st;
    template <int D, typename T, bool E8> int operator()() const { return launch_decode<D, T, E8>(a, st); }
};
struct Workspace {
    bool wide;
    template <int D, typename T, bool E8> int operator()() const {
        return wide ? (int)(4 * kf::decode_workspace_floats<D, E8, 2>(decode_ctas<D, E8, 2>()))
                    : (int)(4 * kf::decode_workspace_floats<D, E8, 1>(decode_ctas<D, E8, 1>()));
    }
};

}  // namespace

extern "C" {

int kf_append_rows(const kf_append_params* p, void* stream) {
    if (!p) return fail(KF_EINVAL, "params must not be NULL");
    kf::AppendArgs a{};
    if (int r = cache_view(p->cache, p->dtype, &a.c)) return r;
    if (int r = check_sizes("B", p->B, kMaxRows)) return r;
    if (int r = check_sizes("S", p->S, kMaxRows)) return r;
    if (p->B * p->S > kMaxRows) return fail(KF_EINVAL, "too many rows");
    const int64_t H = p->cache.Hkv, D = p->cache.D;
    if (int r = check_rows("k", p->k, p->B, H, p->S, D, p->k_stride_b, p->k_stride_h, p->k_stride_s)) return r;
    if (int r = check_rows("v", p->v, p->B, H, p->S, D, p->v_stride_b, p->v_stride_h, p->v_stride_s)) return r;
    if (int r = check_tables(p->gamma, p->cos_table, p->sin_table, p->n_positions)) return r;
    if (!p->start || !p->status) return fail(KF_EINVAL, "start and status must not be NULL");
    if (!(p->eps > 0)) return fail(KF_EINVAL, "eps must be positive");
    if (int r = check_device()) return r;
    a.k = p->k; a.v = p->v; a.gamma = p->gamma; a.cos = p->cos_table; a.sin = p->sin_table;
    a.k_sb = p->k_stride_b; a.k_sh = p->k_stride_h; a.k_ss = p->k_stride_s;
    a.v_sb = p->v_stride_b; a.v_sh = p->v_stride_h; a.v_ss = p->v_stride_s;
    a.start = p->start; a.counts = p->counts;
    a.B = (int)p->B; a.H = (int)H; a.S = (int)p->S; a.n_pos = (int)p->n_positions;
    a.eps = (float)p->eps;
    a.status = p->status;
    return by_type(D, p->dtype, p->cache.dtype == KF_E4M3, Append{a, static_cast<cudaStream_t>(stream)});
}

int kf_read_rows(const kf_read_params* p, void* stream) {
    if (!p) return fail(KF_EINVAL, "params must not be NULL");
    kf::ReadArgs a{};
    if (int r = cache_view(p->cache, p->dtype, &a.c)) return r;
    if (int r = check_sizes("B", p->B, kMaxRows)) return r;
    if (int r = check_sizes("S", p->S, kMaxRows)) return r;
    const int64_t H = p->cache.Hkv, D = p->cache.D;
    if (int r = check_rows("k", p->k, p->B, H, p->S, D, p->k_stride_b, p->k_stride_h, p->k_stride_s)) return r;
    if (int r = check_rows("v", p->v, p->B, H, p->S, D, p->v_stride_b, p->v_stride_h, p->v_stride_s)) return r;
    if (!p->lengths || !p->status) return fail(KF_EINVAL, "lengths and status must not be NULL");
    if (int r = check_device()) return r;
    a.k = p->k; a.v = p->v;
    a.k_sb = p->k_stride_b; a.k_sh = p->k_stride_h; a.k_ss = p->k_stride_s;
    a.v_sb = p->v_stride_b; a.v_sh = p->v_stride_h; a.v_ss = p->v_stride_s;
    a.lengths = p->lengths;
    a.B = (int)p->B; a.H = (int)H; a.S = (int)p->S;
    a.status = p->status;
    return by_type(D, p->dtype, p->cache.dtype == KF_E4M3, Read{a, static_cast<cudaStream_t>(stream)});
}

size_t kf_decode_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t cache_dtype) {
    if (B < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || (D != 128 && D != 256)) return 0;
    return (size_t)by_type(D, KF_BF16, cache_dtype == KF_E4M3, Workspace{Hq / Hkv > 8});
}

int kf_decode_attention(const kf_decode_params* p, void* stream) {
    if (!p) return fail(KF_EINVAL, "params must not be NULL");
    kf::DecodeArgs a{};
    if (int r = cache_view(p->cache, p->dtype, &a.c)) return r;
    const int64_t Hkv = p->cache.Hkv, D = p->cache.D;
    if (int r = check_sizes("B", p->B, 1 << 20)) return r;
    if (p->Hq < 1 || p->Hq > (1 << 16) || p->Hq % Hkv)
        return fail(KF_EINVAL, "Hq (%lld) must be a positive multiple of Hkv (%lld)", (long long)p->Hq, (long long)Hkv);
    if (p->B * p->Hq > kMaxRows) return fail(KF_EINVAL, "too many query rows");
    if (int r = check_rows("q", p->q, p->B, p->Hq, 1, D, p->q_stride_b, p->q_stride_h, 0)) return r;
    if (int r = check_rows("out", p->out, p->B, p->Hq, 1, D, p->o_stride_b, p->o_stride_h, 0)) return r;
    if (int r = check_tables(p->gamma_q, p->cos_table, p->sin_table, p->n_positions)) return r;
    if ((p->new_k == nullptr) != (p->new_v == nullptr)) return fail(KF_EINVAL, "provide both new rows or neither");
    if (!p->lengths || !p->status || !p->workspace) return fail(KF_EINVAL, "lengths, status and workspace must not be NULL");
    if (!aligned16(p->workspace)) return fail(KF_EALIGN, "pointers must be 16-byte aligned");
    if (!(p->eps > 0)) return fail(KF_EINVAL, "eps must be positive");
    if (!(p->scale > 0) || !(p->scale < 1e30)) return fail(KF_EINVAL, "scale must be positive and finite");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p->new_k) {
        if (int r = check_rows("new_k", p->new_k, p->B, Hkv, 1, D, p->k_stride_b, p->k_stride_h, 0)) return r;
        if (int r = check_rows("new_v", p->new_v, p->B, Hkv, 1, D, p->v_stride_b, p->v_stride_h, 0)) return r;
        if (!aligned16(p->gamma_k)) return fail(KF_EALIGN, "pointers must be 16-byte aligned");
    }
    if (int r = check_device()) return r;
    a.new_k = p->new_k; a.new_v = p->new_v; a.gamma_k = p->gamma_k;
    a.nk_sb = p->k_stride_b; a.nk_sh = p->k_stride_h; a.nv_sb = p->v_stride_b; a.nv_sh = p->v_stride_h;
    a.q = p->q; a.gamma = p->gamma_q; a.cos = p->cos_table; a.sin = p->sin_table;
    a.out = p->out;
    a.q_sb = p->q_stride_b; a.q_sh = p->q_stride_h; a.o_sb = p->o_stride_b; a.o_sh = p->o_stride_h;
    a.lengths = p->lengths;
    a.ws = static_cast<float*>(p->workspace);
    a.B = (int)p->B; a.Hkv = (int)Hkv; a.G = (int)(p->Hq / Hkv);
    a.n_pos = (int)p->n_positions;
    a.eps = (float)p->eps;
    a.scale_log2e = (float)(p->scale * 1.4426950408889634);
    a.status = p->status;
    return by_type(D, p->dtype, p->cache.dtype == KF_E4M3, Decode{a, st});
}

}  // extern "C"
