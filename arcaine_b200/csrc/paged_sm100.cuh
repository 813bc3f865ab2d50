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
// wait between CTAs.  Bound by its chain of latencies (lengths, scan, search, table), a few us whatever the step.
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
        const long long most = (long long)p.width * p.page;
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
    const uint16_t* src[3];  // projected rows of Q, K, V: (tokens, heads, hd)
    uint16_t* out[3];        // rows for the caller, or nullptr
    uint16_t* pages[3];      // the pools of K and V, or nullptr
    const int* slots;
    const int* positions;
    const double* inv_freq;
    const uint16_t* weight[2];
    uint32_t* fault;
    int tokens, page, num_rows;  // num_rows: of a pool
    int end[3];                  // first row of a token behind its Q / K / V rows
    int half;                    // rotary_dim / 2
    int norm_qk, norm_v;
    long long src_stride[3], out_stride[3], page_stride[3], row_stride[3];
    float eps, mscale;
};

// A warp takes a token, or a part of its rows where tokens are few, 512 / HD rows a pass: a lane holds two 16-byte pieces of a row
// such that no rotation pair leaves it.  With r = rotary_dim / 16 lanes that rotate, those are pieces (l, l + r) for l < r and
// (2 l, 2 l + 1) for the others in the half layout, (2 l, 2 l + 1) for all in the interleaved one; either way lane l < r has the
// pairs 8 l to 8 l + 7.  Norm and rotation stay in fp32 and are rounded once.
//
// Angles: turns = position * inv_freq / 2 pi in 64 bits, less the nearest whole number; what is left, at most half a turn, is exact
// in fp32 and goes to sincospif.  (In fp32 the angle of position 500000 would be off by 0.03 rad.)  Once a token and pair, not a head.
template <int HD, bool INTERLEAVED>
__global__ void __launch_bounds__(32 * PREP_WARPS, 2) qkv_prepare_paged_kernel(const QkvPagedParams p, const int chunk, const int chunks) {
    constexpr int LPR = HD / 16;   // lanes per row
    constexpr int RPW = 512 / HD;  // rows per pass
    __shared__ __align__(16) float s_cos[PREP_WARPS][HD / 2], s_sin[PREP_WARPS][HD / 2];
    __shared__ __align__(16) float s_w[2][HD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int sub = lane / LPR, li = lane % LPR;
    const int turning = p.half >> 3;  // lanes of a row that rotate
    const bool split = !INTERLEAVED && li < turning;
    const int c0 = (split ? li : 2 * li) * 8, c1 = (split ? li + turning : 2 * li + 1) * 8;  // this lane's columns
    grid_dependency_wait();
    grid_launch_dependents();
    for (int i = threadIdx.x; i < 2 * HD; i += blockDim.x) {
        const uint16_t* w = p.weight[i / HD];
        s_w[i / HD][i % HD] = w ? bf16_bits_to_f32(w[i % HD]) : 1.0f;
    }
    const bool aborted = __syncthreads_or(threadIdx.x == 0 && *reinterpret_cast<volatile uint32_t*>(p.fault) != 0u);
    if (aborted) return;  // a status is set: no work
    const int units = p.tokens * chunks;  // the host keeps this below 2^31
    for (int u = blockIdx.x * PREP_WARPS + warp; u < units; u += gridDim.x * PREP_WARPS) {
        const int t = u / chunks, r_begin = (u - t * chunks) * chunk * RPW, r_end = min(p.end[2], r_begin + chunk * RPW);
        const int pos = p.positions[t];
        if (pos < 0) continue;  // padding
        int slot = p.slots ? p.slots[t] : -1;
        if (slot >= p.num_rows || slot < -1) {
            if (p.slots && lane == 0) report_fault(p.fault, FAULT_BAD_KV_RANGE, (uint32_t)t);
            slot = -1;
        }
        const int page = slot < 0 ? 0 : slot / p.page, row = slot - page * p.page;
        if (r_begin < p.end[1] && p.half > 0) {
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
        for (int r0 = r_begin; r0 < r_end; r0 += RPW) {
            const int r = r0 + sub;
            const bool there = r < r_end;
            const int part = r < p.end[0] ? 0 : r < p.end[1] ? 1 : 2, head = r - (part ? p.end[part - 1] : 0);
            uint4 ra = make_uint4(0u, 0u, 0u, 0u), rb = ra;
            if (there) {
                const uint16_t* src = p.src[part] + t * p.src_stride[part] + (long long)head * HD;
                ra = *reinterpret_cast<const uint4*>(src + c0);
                rb = *reinterpret_cast<const uint4*>(src + c1);
            }
            if (part == 2 ? p.norm_v : (p.norm_qk || p.half)) {
                float a[8], b[8];
                unpack8(ra, a);
                unpack8(rb, b);
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + b[e] * b[e];
                // (a row's lanes agree on its part)
                const uint32_t row_lanes = LPR == 32 ? 0xffffffffu : ((1u << LPR) - 1u) << (sub * LPR);
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(row_lanes, ss, o);
                if (part == 2 || p.norm_qk) {
                    const float inv = rsqrtf(ss / static_cast<float>(HD) + p.eps);
#pragma unroll
                    for (int e = 0; e < 8; ++e) a[e] *= inv, b[e] *= inv;
                    if (part < 2) {
                        const float *wa = s_w[part] + c0, *wb = s_w[part] + c1;
#pragma unroll
                        for (int e = 0; e < 8; ++e) a[e] *= wa[e], b[e] *= wb[e];
                    }
                }
                if (part < 2 && li < turning) {
                    const float *cs = s_cos[warp] + li * 8, *sn = s_sin[warp] + li * 8;
                    auto turn = [&](float& x, float& y, int f) {
                        const float x0 = x, y0 = y;
                        x = x0 * cs[f] - y0 * sn[f];
                        y = x0 * sn[f] + y0 * cs[f];
                    };
#pragma unroll
                    for (int f = 0; f < 8; ++f) {
                        if constexpr (INTERLEAVED) turn(f < 4 ? a[2 * f] : b[2 * f - 8], f < 4 ? a[2 * f + 1] : b[2 * f - 7], f);
                        else turn(a[f], b[f], f);
                    }
                }
                ra = pack8(a);
                rb = pack8(b);
            }
            if (!there) continue;
            if (p.out[part]) {
                uint16_t* dst = p.out[part] + t * p.out_stride[part] + (long long)head * HD;
                *reinterpret_cast<uint4*>(dst + c0) = ra;
                *reinterpret_cast<uint4*>(dst + c1) = rb;
            }
            if (p.pages[part] && slot >= 0) {
                uint16_t* dst = p.pages[part] + page * p.page_stride[part] + row * p.row_stride[part] + (long long)head * HD;
                *reinterpret_cast<uint4*>(dst + c0) = ra;
                *reinterpret_cast<uint4*>(dst + c1) = rb;
            }
        }
    }
}

}  // namespace arc
