// C ABI of the paged KV cache: tables, pre-processing with append, decode.  Argument checks, launch plans, launches.
#include "../../include/arc_sdpa.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "arc_internal.hpp"
#include "decode_paged_sm100.cuh"
#include "paged_sm100.cuh"

using namespace arc;

// Strides of a pool of pages: rows must hold a token's heads, pages their rows.
static int check_pool(int64_t stride_page, int64_t stride_t, int page_size, int num_pages, int64_t row) {
    if (stride_page < 0 || stride_t < 0 || (stride_page & 7) || (stride_t & 7)) return ARC_ERR_ALIGNMENT;
    if (stride_t < row || (num_pages > 1 && stride_page < (page_size - 1) * stride_t + row)) return ARC_ERR_BAD_SHAPE;
    return ARC_OK;
}

static int check_pages(int page_size, int num_pages) {
    if (page_size < 16 || page_size % 16 != 0 || num_pages < 1) return ARC_ERR_BAD_SHAPE;
    if ((int64_t)page_size * num_pages > 0x7fffffffLL) return ARC_ERR_TOO_LARGE;  // (slots are 32 bits wide)
    return ARC_OK;
}

extern "C" int arc_paged_tables(const arc_paged_tables_params* p, void* stream) {
    if (!p) return ARC_ERR_NULL_POINTER;
    if (p->batch <= 0 || p->num_tokens < 0 || p->table_width < 1 || p->free_count < 0 || p->table_stride < p->table_width ||
        p->page_size < 16 || p->page_size % 16 != 0)
        return ARC_ERR_BAD_SHAPE;
    if (p->batch > TABLES_MAX_BATCH || p->num_tokens > 1 << 30) return ARC_ERR_TOO_LARGE;  // (tokens are counted in 32 bits, a grid at a time)
    if (!p->new_len || !p->block_table || (p->free_count > 0 && !p->free_pages) || (p->num_tokens > 0 && (!p->slots || !p->positions)) ||
        !p->token_begin || !p->kv_len || !p->pages_used)
        return ARC_ERR_NULL_POINTER;
    const void* all[] = {p->new_len, p->past_len, p->block_table, p->free_pages, p->free_begin, p->slots, p->positions, p->token_begin, p->kv_len, p->pages_used};
    for (const void* a : all)
        if (reinterpret_cast<uintptr_t>(a) & 3u) return ARC_ERR_ALIGNMENT;
    HostState hs;
    const int rc = host_state(&hs);
    if (rc != ARC_OK) return rc;
    PagedTablesParams kp{};
    kp.new_len = p->new_len;
    kp.past_len = p->past_len;
    kp.table = p->block_table;
    kp.free_pages = p->free_pages;
    kp.free_begin = p->free_begin;
    kp.slots = p->slots;
    kp.positions = p->positions;
    kp.token_begin = p->token_begin;
    kp.kv_len = p->kv_len;
    kp.pages_used = p->pages_used;
    kp.fault = hs.fault;
    kp.batch = p->batch;
    kp.num_tokens = p->num_tokens;
    kp.page = p->page_size;
    kp.width = p->table_width;
    kp.free_count = p->free_count;
    kp.table_stride = p->table_stride;
    const int blocks = std::max(1, std::min(hs.sm_count * 2, (p->num_tokens + TABLES_THREADS - 1) / TABLES_THREADS));
    ARC_CUDA(launch_dependent(paged_tables_kernel, dim3((unsigned)blocks), dim3(TABLES_THREADS), 0, static_cast<cudaStream_t>(stream), 1, kp));
    count_launch();
    return ARC_OK;
}

extern "C" int arc_qkv_prepare_paged(const arc_qkv_prepare_paged_params* p, void* stream) {
    if (!p) return ARC_ERR_NULL_POINTER;
    if (p->hd != 128 && p->hd != 256 && p->hd != 512) return ARC_ERR_UNSUPPORTED_HEAD_DIM;
    if (p->tokens < 0 || (p->q && p->nq < 1) || (p->k && p->nkv < 1)) return ARC_ERR_BAD_SHAPE;
    if (p->rotary_dim < 0 || p->rotary_dim > p->hd || p->rotary_dim % 16 != 0) return ARC_ERR_BAD_SHAPE;
    if (!std::isfinite(p->eps) || p->eps < 0.f || !std::isfinite(p->mscale)) return ARC_ERR_BAD_SHAPE;
    if (p->tokens == 0) return ARC_OK;  // (ahead of the pointers: an empty tensor has none)
    if (p->v && !p->k) return ARC_ERR_NULL_POINTER;
    if ((p->q && !p->q_out) || (p->k && !p->k_out && !p->k_pages) || (p->v && !p->v_out && !p->v_pages)) return ARC_ERR_NULL_POINTER;
    if ((p->rotary_dim > 0 && !p->inv_freq) || !p->positions) return ARC_ERR_NULL_POINTER;
    const bool pages = (p->k && p->k_pages) || (p->v && p->v_pages);
    if (pages && !p->slots) return ARC_ERR_NULL_POINTER;
    if (!p->q && !p->k) return ARC_ERR_NULL_POINTER;
    const void* all[] = {p->q, p->k, p->v, p->q_out, p->k_out, p->v_out, p->k_pages, p->v_pages, p->q_weight, p->k_weight};
    for (const void* a : all)
        if (!aligned16(a)) return ARC_ERR_ALIGNMENT;
    if ((reinterpret_cast<uintptr_t>(p->inv_freq) & 7u) || (reinterpret_cast<uintptr_t>(p->slots) & 3u) || (reinterpret_cast<uintptr_t>(p->positions) & 3u))
        return ARC_ERR_ALIGNMENT;
    const int64_t qrow = (int64_t)p->nq * p->hd, row = (int64_t)p->nkv * p->hd;
    int rc;
    const auto tokens_apart = [](bool used, int64_t stride, int64_t least) {
        if (!used) return ARC_OK;
        if (stride < 0 || (stride & 7)) return ARC_ERR_ALIGNMENT;
        return stride < least ? ARC_ERR_BAD_SHAPE : ARC_OK;
    };
    if ((rc = tokens_apart(p->q, p->q_stride, qrow)) != ARC_OK || (rc = tokens_apart(p->q, p->q_out_stride, qrow)) != ARC_OK ||
        (rc = tokens_apart(p->k, p->k_stride, row)) != ARC_OK || (rc = tokens_apart(p->v, p->v_stride, row)) != ARC_OK ||
        (rc = tokens_apart(p->k && p->k_out, p->k_out_stride, row)) != ARC_OK || (rc = tokens_apart(p->v && p->v_out, p->v_out_stride, row)) != ARC_OK)
        return rc;
    if (pages) {
        if ((rc = check_pages(p->page_size, p->num_pages)) != ARC_OK) return rc;
        if (p->k_pages && (rc = check_pool(p->k_stride_page, p->k_stride_t, p->page_size, p->num_pages, row)) != ARC_OK) return rc;
        if (p->v && p->v_pages && (rc = check_pool(p->v_stride_page, p->v_stride_t, p->page_size, p->num_pages, row)) != ARC_OK) return rc;
    }
    HostState hs;
    if ((rc = host_state(&hs)) != ARC_OK) return rc;

    QkvPagedParams kp{};
    const auto u16 = [](const void* x) { return static_cast<uint16_t*>(const_cast<void*>(x)); };
    kp.k0 = p->q ? p->nq : 0;
    kp.v0 = kp.k0 + (p->k ? p->nkv : 0);
    kp.rows = kp.v0 + (p->v ? p->nkv : 0);
    if (p->q) {
        kp.q = u16(p->q), kp.q_stride = p->q_stride;
        kp.q_dst = u16(p->q_out), kp.q_dst_stride = p->q_out_stride;
    }
    if (p->k) {
        kp.k = u16(p->k), kp.k_stride = p->k_stride;
        kp.pool_k = p->k_pages != nullptr;
        kp.k_dst = u16(kp.pool_k ? p->k_pages : p->k_out);
        kp.k_page_stride = p->k_stride_page, kp.k_row_stride = kp.pool_k ? p->k_stride_t : p->k_out_stride;
        if (kp.pool_k) kp.k_also = u16(p->k_out), kp.k_also_stride = p->k_out_stride;
    }
    if (p->v) {
        kp.v = u16(p->v), kp.v_stride = p->v_stride;
        kp.pool_v = p->v_pages != nullptr;
        kp.v_dst = u16(kp.pool_v ? p->v_pages : p->v_out);
        kp.v_page_stride = p->v_stride_page, kp.v_row_stride = kp.pool_v ? p->v_stride_t : p->v_out_stride;
        if (kp.pool_v) kp.v_also = u16(p->v_out), kp.v_also_stride = p->v_out_stride;
    }
    const int rows = kp.rows;
    kp.slots = pages ? p->slots : nullptr;
    kp.positions = p->positions;
    kp.inv_freq = p->inv_freq;
    kp.weight[0] = static_cast<const uint16_t*>(p->q_weight);
    kp.weight[1] = static_cast<const uint16_t*>(p->k_weight);
    kp.fault = hs.fault;
    static std::atomic<uint32_t> launches{0};
    kp.own_fault = FAULT_BAD_KV_RANGE | launches.fetch_add(1, std::memory_order_relaxed) << FAULT_LAUNCH_SHIFT;
    kp.tokens = p->tokens;
    kp.page = pages ? p->page_size : 1;
    kp.num_rows = pages ? p->page_size * p->num_pages : 0;
    kp.half = p->rotary_dim / 2;
    kp.norm_qk = p->norm_qk != 0;
    kp.norm_v = p->norm_v != 0;
    kp.eps = p->eps;
    kp.mscale = p->mscale;
    // Equal shares of all passes: a pass a warp while one CTA per SM has them all, then three and more (each CTA has its start to pay
    // for: 128 tokens of 64 rows of 128, 2048 passes, 4.4 us as one each, 3.9 as two), on at most three CTAs per SM.
    const int passes = (rows + 512 / p->hd - 1) / (512 / p->hd);
    const long long total = (long long)p->tokens * passes, one_each = (long long)hs.sm_count * PREP_WARPS;
    if (total > 0x7fffffffLL) return ARC_ERR_TOO_LARGE;
    const long long warps = total <= one_each ? total : std::min(3 * one_each, std::max(one_each, total / 3));
    const unsigned ctas = (unsigned)((warps + PREP_WARPS - 1) / PREP_WARPS);
    const int share = (int)(total / ((long long)ctas * PREP_WARPS)), longer = (int)(total % ((long long)ctas * PREP_WARPS));
    const bool common = kp.norm_qk && !kp.norm_v && kp.pool_k && kp.pool_v && !kp.k_also && !kp.v_also;
    auto launch = [&](auto hd_tag) {
        constexpr int H = decltype(hd_tag)::value;
        const auto kernel = common ? (p->interleaved ? qkv_prepare_paged_kernel<H, true, true> : qkv_prepare_paged_kernel<H, false, true>)
                                   : (p->interleaved ? qkv_prepare_paged_kernel<H, true, false> : qkv_prepare_paged_kernel<H, false, false>);
        return launch_dependent(kernel, dim3(ctas), dim3(32 * PREP_WARPS), 0,
                                static_cast<cudaStream_t>(stream), 1, kp, passes, share, longer);
    };
    ARC_CUDA(p->hd == 128 ? launch(std::integral_constant<int, 128>{}) : p->hd == 256 ? launch(std::integral_constant<int, 256>{}) : launch(std::integral_constant<int, 512>{}));
    count_launch();
    return ARC_OK;
}

// ---------------------------------------------------------------------------
// Decode
// ---------------------------------------------------------------------------
struct DecodePagedPlan {
    int nkv_cta = 1, groups = 1, subs = 1, slices = 1, stages = 2, ncta = 1, smem_bytes = 0;
    long long parts = 0;
    size_t ws_bytes = 0;
    bool cluster = false;  // one launch: `ncta` CTAs of a cluster per sequence and group of heads
};

// Slices of 16 keys that a token at the end of `len` keys sees at most.
static long long most_slices_seen(const arc_sdpa_decode_paged_params* p, int64_t len) {
    if (p->window >= len) return (len + 15) / 16;
    return std::min<long long>((len + 15) / 16, ((int64_t)p->window + 30) / 16 + ((int64_t)p->sinks + 15) / 16);
}

// Stages of 16-key slices of `heads` KV heads, `slices` each; extra: bytes behind them.  False: not even two fit.
static bool size_paged_cta(int hd, int heads, int slices, int extra, int smem_optin, DecodePagedPlan* plan) {
    const int stage = 64 * slices * heads * hd, fixed = 1024 + 4 * 16 + extra;
    plan->nkv_cta = heads;
    plan->slices = slices;
    plan->stages = std::min(4, (smem_optin - kDecodeStaticSmem - fixed) / stage);
    plan->smem_bytes = plan->stages * stage + fixed;
    return plan->stages >= 2;
}

static int paged_slices(int hd, int heads, int subs) { return std::max(1, std::min(64 * 1024 / (64 * heads * hd), 8 / (heads * subs))); }

// One launch or two?  Clusters take 4.8 us and the longer of two times: of a CTA of the longest sequence, taken to stream 65 / 70 / 85 GB/s with
// one / two / four and more KV heads of 128 and 91 with heads of 256 (measured rates: decode_paged_sm100.cuh; one of 1200 keys
// among 19 of 16, a head each 14.0 us where this says 14.2; among 59, two heads each 18.9 and 22.4; of 900, heads of 256 16.5 and 15.1), and of
// all keys at 6.5 TB/s.  Shares read those at the same rate, whatever the lengths, but cost 7 us, up to 3 more that parts of a few slices do not hide, and 0.03 for each sequence (the
// second launch, the records, shares that two sequences divide).  (us, shares and clusters, all sequences as long: one token of 24/4
// heads of 256 over 513 keys 7.2 and 6.1, of 28/4 of 128 over 4100 10.6 and 9.2; 16 over 1028 15.5 and 11.1; 48 26.9 and 22.2; 100
// 43.2 and 39.2; 128 of 16/2 over 4100 94 and 83.)  Lengths on the device are not known here, only what a table row can name and what
// a window leaves of it.  Behind a window that is shorter than that, streams tend to its length; otherwise one sequence may be as
// long as the table says and work alone in its cluster, so the form is taken where that costs at most 24 us or 1.3 times what
// shares do.
static bool worth_cluster(const arc_sdpa_decode_paged_params* p, int heads, int size) {
    const int64_t longest = p->kv_len ? (int64_t)p->table_width * p->page_size : p->kv_len_uniform;
    const double keys = 16.0 * (double)most_slices_seen(p, longest), key = 4.0 * p->nkv * p->hd;  // bytes of one
    const double rate = p->hd == 256 ? 91e3 : heads == 1 ? 65e3 : heads < 4 ? 70e3 : 85e3;       // bytes a us
    const double alone = 4.8 + keys * key * heads / p->nkv / size / rate;
    const auto shares = [&](double k) { return 7.0 + 3.0 * std::min(1.0, k * key / 8e6) + 0.03 * p->batch + k * key / 6.5e6; };
    if (p->kv_len && p->batch > 1 && p->window >= longest) return alone <= std::max(24.0, 1.3 * shares(keys));
    return std::max(alone, 4.8 + keys * p->batch * key / 6.5e6) <= shares(keys * p->batch);
}

static void plan_paged_cluster(const arc_sdpa_decode_paged_params* p, const HostState& hs, DecodePagedPlan* plan) {
    if (p->num_ctas != 0 || p->batch > 1024) return;
    // The smallest group of heads, and then the largest cluster, that are all resident at once.
    int heads = 0, size = 0;
    for (int c = 1; c <= plan->nkv_cta && !heads; ++c)
        if (p->nkv % c == 0 && (long long)p->batch * (p->nkv / c) <= hs.decode_clusters[1]) heads = c;
    for (int n = 8; heads && n >= 1 && !size; --n)
        if ((long long)p->batch * (p->nkv / heads) <= hs.decode_clusters[n]) size = n;
    if (!size) return;
    if (!worth_cluster(p, heads, size)) return;
    DecodePagedPlan one = *plan;
    const int rows = heads * (p->nq / p->nkv);
    int finishers = 1;
    while (finishers * 2 <= size) finishers *= 2;
    const int extra = 64 + 8 * ((rows + 1) & ~1) * 8 + size * rows * (p->hd / finishers) * 4 + rows * 32;
    if (!size_paged_cta(p->hd, heads, paged_slices(p->hd, heads, plan->subs), extra, hs.smem_optin, &one)) return;
    one.cluster = true;
    one.groups = p->nkv / heads;
    one.ncta = size;
    one.ws_bytes = 0;
    *plan = one;
}

static int plan_decode_paged(const arc_sdpa_decode_paged_params* p, const HostState& hs, DecodePagedPlan* plan) {
    if (!p) return ARC_ERR_NULL_POINTER;
    if (p->batch <= 0 || p->nq <= 0 || p->nkv <= 0 || p->nq % p->nkv != 0 || p->table_width < 1 || p->table_stride < p->table_width)
        return ARC_ERR_BAD_SHAPE;
    if (p->batch > DECODE_MAX_BATCH) return ARC_ERR_TOO_LARGE;
    if (p->hd != 128 && p->hd != 256) return ARC_ERR_UNSUPPORTED_HEAD_DIM;
    if (!(p->scale > 0.f) || !std::isfinite(p->scale)) return ARC_ERR_BAD_SHAPE;
    if (p->window < 1 || p->sinks < 0 || p->num_ctas < 0) return ARC_ERR_BAD_SHAPE;
    int rc = check_pages(p->page_size, p->num_pages);
    if (rc != ARC_OK) return rc;
    if (!p->kv_len && (p->kv_len_uniform < 0 || p->kv_len_uniform > (int64_t)p->table_width * p->page_size)) return ARC_ERR_BAD_SHAPE;
    const int G = p->nq / p->nkv;
    if (G > 16) return ARC_ERR_UNSUPPORTED_GQA;
    plan->subs = G > 8 ? 2 : 1;
    // KV heads of a CTA: the largest divisor of nkv whose rows are at most 2 KB; slices of a stage: 64 KB of K and V, eight warps.
    int heads = 1;
    for (int c = 1; c <= p->nkv && c <= 1024 / p->hd && c * plan->subs <= 8; ++c)
        if (p->nkv % c == 0) heads = c;
    if (!size_paged_cta(p->hd, heads, paged_slices(p->hd, heads, plan->subs), (p->batch + 2) * 8, hs.smem_optin, plan)) return ARC_ERR_TOO_LARGE;
    plan->groups = p->nkv / plan->nkv_cta;
    plan->ncta = std::min(1024, std::max(1, p->num_ctas > 0 ? p->num_ctas : hs.sm_count / plan->groups));
    plan->parts = ((long long)plan->ncta + p->batch) * plan->slices;
    plan->ws_bytes = (size_t)plan->parts * p->nq * ((size_t)p->hd + 1) * sizeof(float);
    plan_paged_cluster(p, hs, plan);
    return ARC_OK;
}

// A pool of pages as (64 columns, row, 64-column chunk, KV head, page); box: 16 rows of `heads` heads.
static int make_pool_map(CUtensorMap* tm, const void* base, int hd, int nkv, int heads, int page, int num_pages, int64_t stride_t, int64_t stride_page) {
    const cuuint64_t dims[5] = {64u, (cuuint64_t)page, (cuuint64_t)hd / 64u, (cuuint64_t)nkv, (cuuint64_t)num_pages};
    const cuuint64_t last = (cuuint64_t)(num_pages > 1 ? stride_page : stride_t * page);
    const cuuint64_t strides[4] = {(cuuint64_t)stride_t * 2u, 128u, (cuuint64_t)hd * 2u, last * 2u};
    const cuuint32_t box[5] = {64u, 16u, (cuuint32_t)hd / 64u, (cuuint32_t)heads, 1u};
    return encode_bf16_map(tm, base, 5, dims, strides, box, " (pages)");
}

// Dynamic shared memory beyond 48 KB, once per device: a call of its own for every launch took 0.6 us.
static int allow_shared_memory(const HostState& hs) {
    static std::atomic<bool> done[kMaxDevices];
    if (done[hs.device].load(std::memory_order_acquire)) return ARC_OK;
    const int most = hs.smem_optin - kDecodeStaticSmem;
    ARC_CUDA(opt_in_smem(sdpa_decode_paged_kernel<128>, most));
    ARC_CUDA(opt_in_smem(sdpa_decode_paged_kernel<256>, most));
    ARC_CUDA(opt_in_smem(sdpa_decode_paged_cluster_kernel<128>, most));
    ARC_CUDA(opt_in_smem(sdpa_decode_paged_cluster_kernel<256>, most));
    done[hs.device].store(true, std::memory_order_release);
    return ARC_OK;
}

template <int HD>
static int launch_decode_paged(const arc_sdpa_decode_paged_params* p, const DecodePagedPlan& plan, const HostState& hs, cudaStream_t stream) {
    CUtensorMap tk, tv;
    int rc;
    if ((rc = allow_shared_memory(hs)) != ARC_OK) return rc;
    if ((rc = make_pool_map(&tk, p->k_pages, HD, p->nkv, plan.nkv_cta, p->page_size, p->num_pages, p->k_stride_t, p->k_stride_page)) != ARC_OK) return rc;
    if ((rc = make_pool_map(&tv, p->v_pages, HD, p->nkv, plan.nkv_cta, p->page_size, p->num_pages, p->v_stride_t, p->v_stride_page)) != ARC_OK) return rc;
    DecodePagedParams kp{};
    kp.q = static_cast<const uint16_t*>(p->q);
    kp.table = p->block_table;
    kp.kv_len = p->kv_len;
    kp.part_o = static_cast<float*>(p->workspace);
    kp.part_lse = kp.part_o + (size_t)plan.parts * p->nq * HD;
    kp.fault = hs.fault;
    kp.batch = p->batch;
    kp.nq = p->nq;
    kp.nkv = p->nkv;
    kp.kv_len_uniform = p->kv_len_uniform;
    kp.page = p->page_size;
    kp.num_pages = p->num_pages;
    kp.max_len = (int)std::min<int64_t>((int64_t)p->table_width * p->page_size, 0x7fffffffLL - 16);
    kp.window = p->window;
    kp.sinks = p->sinks;
    kp.q_stride_b = p->q_stride_b;
    kp.table_stride = p->table_stride;
    kp.scale_log2 = p->scale * 1.4426950408889634f;
    kp.nkv_cta = plan.nkv_cta;
    kp.subs = plan.subs;
    kp.slices = plan.slices;
    kp.stages = plan.stages;
    kp.ncta = plan.ncta;
    const unsigned threads = 32u * (unsigned)(plan.nkv_cta * plan.subs * plan.slices + 1);
    if (plan.cluster) {
        kp.gate = static_cast<const uint16_t*>(p->gate);
        kp.out = static_cast<uint16_t*>(p->out);
        kp.out_f32 = p->out_f32;
        kp.out_lse = p->out_lse;
        kp.o_stride_b = p->o_stride_b;
        ARC_CUDA(launch_dependent(sdpa_decode_paged_cluster_kernel<HD>, dim3((unsigned)plan.ncta, (unsigned)plan.groups, (unsigned)p->batch), dim3(threads),
                                  (size_t)plan.smem_bytes, stream, plan.ncta, tk, tv, kp));
        count_launch();
        return ARC_OK;
    }
    ARC_CUDA(launch_dependent(sdpa_decode_paged_kernel<HD>, dim3((unsigned)plan.ncta, (unsigned)plan.groups), dim3(threads),
                              (size_t)plan.smem_bytes, stream, 1, tk, tv, kp));
    count_launch();

    DecodeMergeParams mp{};
    mp.part_o = kp.part_o;
    mp.part_lse = kp.part_lse;
    mp.kv_len = p->kv_len;
    mp.gate = static_cast<const uint16_t*>(p->gate);
    mp.out = static_cast<uint16_t*>(p->out);
    mp.out_f32 = p->out_f32;
    mp.out_lse = p->out_lse;
    mp.batch = p->batch;
    mp.nq = p->nq;
    mp.kv_len_uniform = p->kv_len_uniform;
    mp.ncta = plan.ncta;
    mp.slices = plan.slices;
    mp.o_stride_b = p->o_stride_b;
    mp.fault = hs.fault;
    mp.window = p->window;
    mp.sinks = p->sinks;
    // 64 columns a block while that leaves at most one block per SM (arc_sdpa.cu); else as many rows a block as leave one for each.
    const long long rows = (long long)p->nq * p->batch;
    const auto blocks = [&](int n) { return (long long)(p->nq + n - 1) / n * p->batch; };
    const auto merge = [&](auto kernel, int n) {
        return launch_dependent(kernel, dim3((unsigned)((p->nq + n - 1) / n), (unsigned)p->batch), dim3(256), 0, stream, 1, mp);
    };
    if (rows * (HD / 64) <= hs.sm_count)
        ARC_CUDA(launch_dependent(sdpa_decode_merge_kernel<HD, false, 64, true>, dim3((unsigned)p->nq, (unsigned)p->batch, HD / 64), dim3(MERGE_THREADS), 0, stream, 1, mp));
    else if (blocks(8) >= hs.sm_count) ARC_CUDA(merge(sdpa_decode_paged_merge_kernel<HD, 8>, 8));
    else if (blocks(4) >= hs.sm_count) ARC_CUDA(merge(sdpa_decode_paged_merge_kernel<HD, 4>, 4));
    else if (blocks(2) >= hs.sm_count) ARC_CUDA(merge(sdpa_decode_paged_merge_kernel<HD, 2>, 2));
    else ARC_CUDA(merge(sdpa_decode_paged_merge_kernel<HD, 1>, 1));
    count_launch();
    return ARC_OK;
}

extern "C" size_t arc_sdpa_decode_paged_workspace_bytes(const arc_sdpa_decode_paged_params* p) {
    HostState hs;
    DecodePagedPlan plan;
    if (host_state(&hs) != ARC_OK || plan_decode_paged(p, hs, &plan) != ARC_OK) return 0;
    return plan.ws_bytes;
}

extern "C" int arc_sdpa_decode_paged(const arc_sdpa_decode_paged_params* p, void* stream) {
    if (!p || !p->q || !p->k_pages || !p->v_pages || !p->block_table || (!p->out && !p->out_f32) || (p->gate && !p->out)) return ARC_ERR_NULL_POINTER;
    // What needs no device is refused without one.
    DecodePagedPlan plan;
    int rc = plan_decode_paged(p, HostState{nullptr, 148, 232448, 0, {}}, &plan);
    if (rc != ARC_OK) return rc;
    if (!aligned16(p->q) || !aligned16(p->k_pages) || !aligned16(p->v_pages) || !aligned16(p->out) || !aligned16(p->gate) || !aligned16(p->out_f32) ||
        ((reinterpret_cast<uintptr_t>(p->block_table) | reinterpret_cast<uintptr_t>(p->kv_len) | reinterpret_cast<uintptr_t>(p->out_lse)) & 3u) ||
        (p->q_stride_b & 7) || (p->o_stride_b & 7))
        return ARC_ERR_ALIGNMENT;
    const int64_t qrow = (int64_t)p->nq * p->hd;
    if (p->batch > 1 && (p->q_stride_b < qrow || (p->out && p->o_stride_b < qrow))) return ARC_ERR_BAD_SHAPE;
    if ((rc = check_pool(p->k_stride_page, p->k_stride_t, p->page_size, p->num_pages, (int64_t)p->nkv * p->hd)) != ARC_OK ||
        (rc = check_pool(p->v_stride_page, p->v_stride_t, p->page_size, p->num_pages, (int64_t)p->nkv * p->hd)) != ARC_OK)
        return rc;
    HostState hs;
    if ((rc = host_state(&hs)) != ARC_OK || (rc = plan_decode_paged(p, hs, &plan)) != ARC_OK) return rc;
    if (plan.ws_bytes && (!p->workspace || p->workspace_bytes < plan.ws_bytes)) return ARC_ERR_WORKSPACE_TOO_SMALL;
    if (plan.ws_bytes && !aligned16(p->workspace)) return ARC_ERR_ALIGNMENT;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return p->hd == 128 ? launch_decode_paged<128>(p, plan, hs, st) : launch_decode_paged<256>(p, plan, hs, st);
}
