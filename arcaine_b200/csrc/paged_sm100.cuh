// What a paged KV cache needs in front of its attention: block tables and slot maps from the requests' lengths, and the norms,
// rotation and append of a step's projected rows.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"
#include "qkv_prepare_sm100.cuh"

namespace arc {

constexpr int TABLES_MAX_BATCH = 2048;
constexpr int TABLES_THREADS = 256;

struct PagedTablesParams {
    const int* new_len;
    const int* past_len;
    int* table;
    const int* free_pages;
    const int* free_begin;
    int* slots;
    int* positions;
    int* token_begin;
    int* kv_len;
    int* pages_used;
    uint32_t* fault;
    int batch, num_tokens, page, width, free_count;
    long long table_stride;
};

// begin[b] = sum of new lengths in front of request b; taken[b] = pages the requests in front take: ceil((past + new) / page) -
// ceil(past / page) each.  Token i belongs to the last request with begin[b] <= i.  A page that the step opens has its first
// row from a token of the step, so the thread with that token writes the table's entry: no second walk over pages.
//
// Every CTA scans all requests (16 KB at most, out of L2) and takes its share of the tokens, so there is one launch and no
// wait between CTAs.  Bound by its chain of latencies (lengths, scan, search, table): 8 requests of a token 3.1 us, 509 with 5093
// tokens 3.7, 64 prompts of 85266 tokens 4.4, for 0.7 MB at most.
__global__ void __launch_bounds__(TABLES_THREADS) paged_tables_kernel(const PagedTablesParams p) {
    constexpr int PER = TABLES_MAX_BATCH / TABLES_THREADS;
    __shared__ int s_begin[TABLES_MAX_BATCH + 1], s_taken[TABLES_MAX_BATCH], s_past[TABLES_MAX_BATCH];
    __shared__ long long s_warp[2][TABLES_THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dependency_wait();
    grid_launch_dependents();
    bool bad = threadIdx.x == 0 && *reinterpret_cast<volatile uint32_t*>(p.fault) != 0u;
    const int list0 = p.free_begin ? *p.free_begin : 0;

    // This thread's requests: `per` in a row.
    const int per = (p.batch + TABLES_THREADS - 1) / TABLES_THREADS, b0 = threadIdx.x * per;
    int past[PER], fresh[PER], pages[PER];
    long long sum_new = 0, sum_pages = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        past[i] = fresh[i] = pages[i] = 0;
        if (i >= per || b0 + i >= p.batch) continue;
        past[i] = p.past_len ? p.past_len[b0 + i] : 0;
        fresh[i] = p.new_len[b0 + i];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (i >= per || b0 + i >= p.batch) continue;
        const long long most = min((long long)p.width * p.page, 0x7fffffffll);  // (positions and lengths are 32 bits wide)
        if (past[i] < 0 || fresh[i] < 0 || (long long)past[i] + fresh[i] > most) {
            report_fault(p.fault, FAULT_BAD_KV_RANGE, (uint32_t)(b0 + i));
            bad = true;
            past[i] = fresh[i] = 0;
        }
        pages[i] = (int)(((long long)past[i] + fresh[i] + p.page - 1) / p.page - ((long long)past[i] + p.page - 1) / p.page);
        sum_new += fresh[i];
        sum_pages += pages[i];
    }
    long long at_new = sum_new, at_pages = sum_pages;  // inclusive within the warp, then exclusive in the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, at_new, o), c = __shfl_up_sync(0xffffffffu, at_pages, o);
        if (lane >= o) at_new += a, at_pages += c;
    }
    if (lane == 31) s_warp[0][warp] = at_new, s_warp[1][warp] = at_pages;
    __syncthreads();
    long long total_new = 0, total_pages = 0;
    at_new -= sum_new, at_pages -= sum_pages;
#pragma unroll
    for (int w = 0; w < TABLES_THREADS / 32; ++w) {
        if (w == warp) at_new += total_new, at_pages += total_pages;
        total_new += s_warp[0][w], total_pages += s_warp[1][w];
    }
    if (total_new > p.num_tokens) {
        if (threadIdx.x == 0) report_fault(p.fault, FAULT_BAD_KV_RANGE, (uint32_t)p.batch);
        bad = true;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (i >= per || b0 + i >= p.batch) continue;
        s_begin[b0 + i] = (int)at_new, s_taken[b0 + i] = (int)at_pages, s_past[b0 + i] = past[i];
        at_new += fresh[i], at_pages += pages[i];
    }
    if (__syncthreads_or(bad)) return;  // nothing is written
    if (blockIdx.x == 0) {
        for (int b = threadIdx.x; b < p.batch; b += TABLES_THREADS) {
            const int end = b + 1 < p.batch ? s_begin[b + 1] : (int)total_new;
            p.token_begin[b] = s_begin[b];
            p.kv_len[b] = s_past[b] + end - s_begin[b];
        }
        if (threadIdx.x == 0) {
            p.token_begin[p.batch] = (int)total_new;
            *p.pages_used = (int)total_pages;
        }
    }
    for (int i = blockIdx.x * TABLES_THREADS + threadIdx.x; i < p.num_tokens; i += gridDim.x * TABLES_THREADS) {
        int slot = -1, pos = -1;
        if (i < (int)total_new) {
            int lo = 0, hi = p.batch;  // the last request that begins at or before i is in [lo, hi)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_begin[mid] <= i) lo = mid;
                else hi = mid;
            }
            const int held = (int)(((long long)s_past[lo] + p.page - 1) / p.page);
            pos = s_past[lo] + i - s_begin[lo];
            const int column = pos / p.page, row = pos - column * p.page;
            int* entry = p.table + lo * p.table_stride + column;
            int page;
            if (column < held) {
                page = *entry;
            } else {
                const long long at = (long long)list0 + s_taken[lo] + column - held;
                page = at >= 0 && at < p.free_count ? p.free_pages[at] : -1;
                if (row == 0) *entry = page;
            }
            const long long place = (long long)page * p.page + row;
            if (page >= 0 && place <= 0x7fffffffLL) slot = (int)place;
        }
        p.slots[i] = slot;
        p.positions[i] = pos;
    }
}

struct QkvPagedParams {
    const uint16_t *q, *k, *v;    // projected rows: (tokens, heads, hd); nullptr: none
    uint16_t *q_dst, *k_dst, *v_dst;  // rows of Q; of K and V the pools where there are any (PAGES_K, PAGES_V), else rows
    uint16_t *k_also, *v_also;    // rows of K and V besides the pools, or nullptr
    const int* slots;
    const int* positions;
    const double* inv_freq;
    const uint16_t* weight[2];
    uint32_t* fault;
    int tokens, page, num_rows;  // num_rows: of a pool
    int k0, v0, rows;            // a token's first K row, first V row, all its rows
    int half;                    // rotary_dim / 2
    int norm_qk, norm_v, pool_k, pool_v;  // pool_*: k_dst / v_dst is a pool
    long long q_stride, k_stride, v_stride, q_dst_stride, k_also_stride, v_also_stride;
    long long k_page_stride, v_page_stride, k_row_stride, v_row_stride;  // row stride: between two rows of a page, or two tokens
    float eps, mscale;
    uint32_t own_fault;          // what this launch reports a bad slot as (FAULT_LAUNCH_SHIFT)
};

// A pass is 512 / HD rows of a token by a warp.  All tokens' passes are laid end to end and cut into equal parts, one per warp, which may
// begin and end inside a token (whole tokens in turn left a tenth of the last round idle).  A lane holds two 16-byte pieces of a row
// such that no rotation pair leaves it, and a load's pieces lie side by side.  Half layout, r = rotary_dim / 16: pieces l and l + r for
// the lanes l < r, which have the pairs 8 l to 8 l + 7, and l + r and l + HD / 16 for the others.  Interleaved: pieces l and
// l + HD / 16, each with its own four pairs.  Norm and rotation stay in fp32 and are rounded once.
//
// Angles: turns = position * inv_freq / 2 pi in 64 bits (three roundings: 3 * 2^-53 of them, 1.2e-7 turns at position 2^31 and one
// radian each), less the nearest whole number; what is left, at most half a turn, is rounded to fp32 (2^-26 turns) and goes to
// sincospif.  (In fp32 the angle of position 500000 would be off by 0.03 rad.)  Once a token and pair, not a head.
//
// Bound by HBM, reads and writes mixed; a pass's rows are asked for one ahead, over the end of a token, too, and with them the
// next token's position and slot.  (16384 tokens of 32/16 heads of 128, 537 MB: 149 us asked for when needed, two CTAs an SM; 100 a
// pass ahead on three; 94.8, 5.67 TB/s, in equal parts.  1024 tokens 12.9 -> 9.8, one of them 3.1.)
// passes: of a token; share: passes of a warp, one more for the first `longer` of them.  COMMON: Q and K rows normed, V rows copied, K and V to pools only (267
// warp instructions a pass, 297 with the other forms' branches: 4096 tokens 34.1 -> 32.3 us, one 3.39 -> 3.22).
template <int HD, bool INTERLEAVED, bool COMMON>
__global__ void __launch_bounds__(32 * PREP_WARPS, 3) qkv_prepare_paged_kernel(const QkvPagedParams p, const int passes, const int share, const int longer) {
    constexpr int LPR = HD / 16;   // lanes per row
    constexpr int RPW = 512 / HD;  // rows per pass
    __shared__ __align__(16) float s_cos[PREP_WARPS][HD / 2], s_sin[PREP_WARPS][HD / 2];
    __shared__ __align__(16) float s_w[2][HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane / LPR, li = lane % LPR;
    const int turning = p.half >> 3;  // half layout: lanes of a row that rotate
    const bool second = !INTERLEAVED && li >= turning;  // (that do not)
    const int c0 = (second ? li + turning : li) * 8;    // this lane's columns: [c0, c0 + 8) and `apart` on
    const int apart = INTERLEAVED ? HD / 2 : second ? HD / 2 - turning * 8 : turning * 8;
    const int pair0 = INTERLEAVED ? li * 4 : li * 8, pair1 = INTERLEAVED ? pair0 + HD / 4 : pair0 + 4;  // four pairs each
    const bool norm_qk = COMMON || p.norm_qk, norm_v = !COMMON && p.norm_v, pool_k = COMMON || p.pool_k, pool_v = COMMON || p.pool_v, slots = COMMON || p.slots;
    grid_dependency_wait();
    grid_launch_dependents();
    for (int i = threadIdx.x; i < 2 * HD; i += blockDim.x) {
        const uint16_t* w = p.weight[i / HD];
        s_w[i / HD][i % HD] = w ? bf16_bits_to_f32(w[i % HD]) : 1.0f;
    }
    const int w = blockIdx.x * PREP_WARPS + warp;
    int left = share + (w < longer ? 1 : 0);  // passes of this warp to be worked on
    const int at = w * share + min(w, longer);

    // The walk of the loads, a pass ahead of the work: token ft, rows from fr to f_end; f_left passes to be asked for.
    int ft = at / passes, fr = (at - ft * passes) * RPW, f_left = left, f_pos = -1, f_slot = -1;
    const uint16_t *fq = nullptr, *fk = nullptr, *fv = nullptr;
    auto begin_loads = [&]() {
        f_pos = p.positions[ft];
        f_slot = slots ? p.slots[ft] : 0;
        fq = p.q + ft * p.q_stride + c0;
        fk = p.k + ft * p.k_stride + c0 - p.k0 * HD;
        fv = p.v + ft * p.v_stride + c0 - p.v0 * HD;
    };
    uint4 na = make_uint4(0u, 0u, 0u, 0u), nb = na;
    auto fetch = [&]() {
        const int r = fr + sub;
        if (r < p.rows) {
            const uint16_t* src = (r < p.k0 ? fq : r < p.v0 ? fk : fv) + r * HD;
            na = *reinterpret_cast<const uint4*>(src);
            nb = *reinterpret_cast<const uint4*>(src + apart);
        }
        fr += RPW;
        --f_left;
    };
    int t = ft, r0 = fr;
    if (left > 0) {
        begin_loads();
        fetch();
    }
    // A status is set: no work.  One of this launch's own, a bad slot that another CTA has met already, keeps nobody from the other tokens:
    // CTAs start when there is room for them, beside other streams' kernels long after the first.
    // (A status stays as it is while kernels run, so that all threads find the same one.)
    const auto status = [&] { return *reinterpret_cast<volatile uint32_t*>(p.fault); };
    if (__syncthreads_or(threadIdx.x == 0 && status() != 0u) && status() != p.own_fault) return;

    for (; left > 0; ++t, r0 = 0) {
        const int pos = f_pos;
        int slot = f_slot;
        if (slots && (slot >= p.num_rows || slot < -1)) {
            if (lane == 0 && pos >= 0) report_fault(p.fault, p.own_fault, (uint32_t)t);
            slot = -1;
        }
        const bool live = pos >= 0, stored = live && slot >= 0;  // (padding; rows that are not appended)
        if (live && r0 < p.v0 && p.half > 0) {
            __syncwarp();
            for (int f = lane; f < p.half; f += 32) {
                const double turns = (double)pos * p.inv_freq[f] * 0.15915494309189533577;
                float s, c;
                sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
                s_cos[warp][f] = c * p.mscale;
                s_sin[warp][f] = s * p.mscale;
            }
            __syncwarp();
        }
        const int page = stored && slots ? slot / p.page : 0, row = slots ? slot - page * p.page : t;
        uint16_t* dq = p.q_dst + t * p.q_dst_stride + c0;
        uint16_t* dk = p.k_dst + (pool_k ? page * p.k_page_stride + row * p.k_row_stride : t * p.k_row_stride) + c0 - p.k0 * HD;
        uint16_t* dv = p.v_dst + (pool_v ? page * p.v_page_stride + row * p.v_row_stride : t * p.v_row_stride) + c0 - p.v0 * HD;
        for (; left > 0 && r0 < p.rows; r0 += RPW, --left) {
            uint4 ra = na, rb = nb;
            if (f_left > 0) {
                if (fr >= p.rows) {  // the next token's first rows follow at once
                    ++ft, fr = 0;
                    begin_loads();
                }
                fetch();
            }
            const int r = r0 + sub;
            const bool is_v = r >= p.v0;
            if (r0 >= p.v0 ? norm_v : (norm_qk || norm_v || p.half)) {  // (what only V rows share with the pass is copied below)
                float a[8], b[8];
                unpack8(ra, a);
                unpack8(rb, b);
                if (norm_qk || norm_v) {
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    const float inv = (is_v ? norm_v : norm_qk) ? rsqrtf(ss / static_cast<float>(HD) + p.eps) : 1.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) a[e] *= inv, b[e] *= inv;
                    if (r0 < p.v0 && norm_qk && !is_v) {
                        const float* w = s_w[r < p.k0 ? 0 : 1] + c0;
#pragma unroll
                        for (int e = 0; e < 8; e += 4) {
                            const float4 x = *reinterpret_cast<const float4*>(w + e), y = *reinterpret_cast<const float4*>(w + apart + e);
                            a[e] *= x.x, a[e + 1] *= x.y, a[e + 2] *= x.z, a[e + 3] *= x.w;
                            b[e] *= y.x, b[e + 1] *= y.y, b[e + 2] *= y.z, b[e + 3] *= y.w;
                        }
                    }
                }
                if (pair0 < p.half && !is_v) {
                    float c[8], s[8];  // (interleaved: of pair1 on whatever is there, where those do not rotate)
                    auto angles = [&](const float* from, float* to, int pair) {
                        const float4 x = *reinterpret_cast<const float4*>(from + pair);
                        to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
                    };
                    angles(s_cos[warp], c, pair0), angles(s_cos[warp], c + 4, pair1);
                    angles(s_sin[warp], s, pair0), angles(s_sin[warp], s + 4, pair1);
                    auto turn = [&](float& x, float& y, int f) {
                        const float x0 = x, y0 = y;
                        x = x0 * c[f] - y0 * s[f];
                        y = x0 * s[f] + y0 * c[f];
                    };
                    if constexpr (INTERLEAVED) {
#pragma unroll
                        for (int f = 0; f < 4; ++f) turn(a[2 * f], a[2 * f + 1], f);
                        if (pair1 < p.half) {
#pragma unroll
                            for (int f = 0; f < 4; ++f) turn(b[2 * f], b[2 * f + 1], f + 4);
                        }
                    } else {
#pragma unroll
                        for (int f = 0; f < 8; ++f) turn(a[f], b[f], f);
                    }
                }
                if (!is_v || norm_v) {
                    ra = pack8(a);
                    rb = pack8(b);
                }
            }
            if (r >= p.rows || !live) continue;
            const bool is_q = r < p.k0;
            if (is_q || stored || !(is_v ? pool_v : pool_k)) {
                uint16_t* dst = (is_q ? dq : is_v ? dv : dk) + r * HD;
                *reinterpret_cast<uint4*>(dst) = ra;
                *reinterpret_cast<uint4*>(dst + apart) = rb;
            }
            if (!COMMON && !is_q && (p.k_also || p.v_also)) {
                uint16_t* also = is_v ? p.v_also : p.k_also;
                if (also) {
                    also += t * (is_v ? p.v_also_stride : p.k_also_stride) + (r - (is_v ? p.v0 : p.k0)) * HD + c0;
                    *reinterpret_cast<uint4*>(also) = ra;
                    *reinterpret_cast<uint4*>(also + apart) = rb;
                }
            }
        }
    }
}

}  // namespace arc
