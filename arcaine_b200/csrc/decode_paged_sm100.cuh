// Split-KV decode over a paged cache: one new query token per sequence, its keys in pages that a block table names, all
// of them or behind a window the last ones and the first (sinks).
//
// The arithmetic is decode_sm100.cuh's: o = sum_j exp(q k_j scale - m) v_j / sum_j exp(q k_j scale - m), online per 16-key slice, with the
// GQA group as the N dimension of the warp MMAs, so K and V are read once.  The unit of everything is the slice: pages are
// multiples of 16 rows, so a slice never leaves its page, and a TMA box of (64 columns, 16 rows, chunks, KV heads) brings
// all heads of a CTA of one slice at once, 4 to 32 KB, wherever the page is (the map's fifth dimension).  The slices
// that a sequence's token sees (SeenKeys) are laid end to end over the batch and cut into equal shares, one per CTA, so
// neither the lengths nor what a window leaves of them have to be alike.  The producer's lanes look up a page each, a
// step ahead of the copies.  Shares, records and their merge are those of decode_sm100.cuh, counted in slices.
//
// Bound by HBM where there is much to read: 64 sequences of 1 K to 32 K keys, 24/4 heads of 256, 3.07 GB, 455 us (6.75 TB/s, of a copy's
// 6.54); 48 streams of 300 to 65536 keys behind a window of 1024 with 4 sinks, 28/4 of 128, 88 MB, 21.9 (13.5 at the copy rate).
// Where there is little, by a chain of latencies: one token of 24/4 heads of 256 over 513 keys 6.2.  A CTA on its own streams what its copies
// let it.  One by shares, the others idle: with 1 / 2 / 4 / 8 heads of 128 a copy (4 to 32 KB) 56 / 71 / 78 / 88 GB/s, with 1 / 2 / 4 of
// 256 78 / 84 / 94.  That of one long sequence in clusters of one, beside short ones: 61 with a head of 128, 83 with two, 77 with one of 256.
#pragma once
#include "decode_sm100.cuh"

namespace arc {

struct DecodePagedParams {
    const uint16_t* q;
    const int* table;
    const int* kv_len;
    float* part_o;    // [(cta + sequence) * slices + slice][nq][HD]
    float* part_lse;  // [(cta + sequence) * slices + slice][nq]
    uint32_t* fault;
    int batch, nq, nkv, kv_len_uniform;
    int page, num_pages, max_len;  // max_len: keys a table row can name
    int window, sinks;
    long long q_stride_b, table_stride;
    float scale_log2;
    int nkv_cta;  // KV heads of a CTA (grid.y = nkv / nkv_cta)
    int subs;     // warps that divide a KV head's query heads, eight each
    int slices;   // 16-key slices of a stage; consumer warps = nkv_cta * subs * slices
    int stages;
    int ncta;     // grid.x
    // One launch (sdpa_decode_paged_cluster_kernel): the results
    const uint16_t* gate;
    uint16_t* out;
    float* out_f32;
    float* out_lse;
    long long o_stride_b;
};

// What a consumer warp holds of up to eight query heads of a KV head: Q^T fragments (B operand, hd x 8 heads), running maximum (log2
// domain) and sum, O^T.  Larger groups go to two warps, which read the same keys out of shared memory.  (Sixteen heads in one warp are
// 192 registers at head dim 256, and spilled: us, 64 sequences of 4100 keys of 16/1 heads 84.6 -> 53.6, one of 513 11.5 -> 7.3.  At head
// dim 128 200 of 300 27.7 -> 22.6, one of 513 5.9 -> 5.5, but 64 of 4100 27.0 -> 31.1: eight warps then have four slices a step.)
template <int HD>
struct GroupState {
    uint32_t q[HD / 16][2];
    float m[2], l[2], o[HD / 16][4];

    __device__ __forceinline__ void load(const uint16_t* heads, int G) {  // heads: the first of the G query heads
        const int lane = threadIdx.x & 31, n = lane >> 2;
        const bool valid = n < G;
        const uint16_t* src = heads + (valid ? n : 0) * HD + (lane & 3) * 2;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
            q[kk][0] = valid ? *reinterpret_cast<const uint32_t*>(src + kk * 16) : 0u;
            q[kk][1] = valid ? *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8) : 0u;
        }
        m[0] = m[1] = -CUDART_INF_F;
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) o[mt][0] = o[mt][1] = o[mt][2] = o[mt][3] = 0.f;
    }

    // Sum of head (lane & 3) * 2 + u over the key rows.
    __device__ __forceinline__ float sum(int u) const {
        float ls = l[u];
        ls += __shfl_xor_sync(0xffffffffu, ls, 4);
        ls += __shfl_xor_sync(0xffffffffu, ls, 8);
        ls += __shfl_xor_sync(0xffffffffu, ls, 16);
        return ls;
    }
};

constexpr int SLICE_CHUNK = 16 * 128;  // 64 columns of a slice in shared memory: 16 rows x 128 bytes

// One slice: sK, sV its head's rows in shared memory ([64-column chunk][row], 128-byte swizzle), bit k of vis: key k is seen.
template <int HD>
__device__ __forceinline__ void attend_slice(GroupState<HD>& g, uint32_t sK, uint32_t sV, uint32_t vis, float sl) {
    constexpr int CHUNK = SLICE_CHUNK;
    const int lane = threadIdx.x & 31, g4 = lane >> 2;  // g4: accumulator row group
    // Swizzled addressing: 16-byte unit u of row r sits at unit u ^ (r & 7).
    const int key_k = lane & 15, key_v = (lane & 7) + (lane >> 4) * 8;
    const uint32_t a_k = sK + key_k * 128, a_v = sV + key_v * 128;
    const int xk = key_k & 7, hk = lane >> 4;
    const int xv = key_v & 7, hv = (lane >> 3) & 1;
    if (vis != 0xffffu) {
        // Rows nobody sees may hold anything (never-written cache, another user's NaN): their V becomes zero, so
        // that 0 * x stays 0; their scores are replaced below.
        for (int u = lane; u < 16 * (HD / 8); u += 32) {
            const int key = u / (HD / 8), c = u % (HD / 8);
            if ((vis >> key) & 1u) continue;
            const uint32_t a = sV + (c >> 3) * CHUNK + key * 128 + (c & 7) * 16;  // (whole rows: their units' order does not matter)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(a), "r"(0u) : "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
    }
    // Fragments are fetched AHEAD at a time and a batch before their MMAs (decode_sm100.cuh).
    constexpr int AHEAD = 4, BATCHES = HD / 16 / AHEAD, CHAINS = 4;  // CHAINS: independent sums of S
    uint32_t fr[2][AHEAD][4];
    auto fetch_k = [&](int bt) {
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const int kk = bt * AHEAD + e;
            ldmatrix_x4(fr[bt & 1][e], a_k + (kk >> 2) * CHUNK + ((((kk & 3) * 2 + hk) ^ xk) << 4));
        }
    };
    auto fetch_v = [&](int bt) {
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const int mt = bt * AHEAD + e;
            ldmatrix_x4_trans(fr[bt & 1][e], a_v + (mt >> 2) * CHUNK + ((((mt & 3) * 2 + hv) ^ xv) << 4));
        }
    };
    float acc[CHAINS][4];
#pragma unroll
    for (int c = 0; c < CHAINS; ++c) acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
    fetch_k(0);
#pragma unroll
    for (int bt = 0; bt < BATCHES; ++bt) {
        if (bt + 1 < BATCHES) fetch_k(bt + 1);
        else fetch_v(0);  // (an even number of batches: into the other half)
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) {
            const int kk = bt * AHEAD + e;
            mma_bf16_16816(acc[kk % CHAINS], fr[bt & 1][e], g.q[kk][0], g.q[kk][1]);
        }
    }
    static_assert(BATCHES % 2 == 0, "the first batch of V goes where the last one of K is not");
    const bool v_lo = (vis >> g4) & 1u, v_hi = (vis >> (g4 + 8)) & 1u;
    float x[4], pr[4], alpha[2];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float s = ((acc[0][e] + acc[1][e]) + (acc[2][e] + acc[3][e])) * sl;
        x[e] = ((e < 2) ? v_lo : v_hi) ? s : -CUDART_INF_F;
    }
    bool any_rescale = false;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        float mx = fmaxf(x[u], x[u + 2]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float m_new = fmaxf(g.m[u], mx);
        const float m_eff = (m_new == -CUDART_INF_F) ? 0.f : m_new;
        alpha[u] = (m_new == -CUDART_INF_F) ? 1.f : fast_exp2(g.m[u] - m_new);
        pr[u] = fast_exp2(x[u] - m_eff);
        pr[u + 2] = fast_exp2(x[u + 2] - m_eff);
        g.l[u] = g.l[u] * alpha[u] + pr[u] + pr[u + 2];
        g.m[u] = m_new;
        any_rescale |= alpha[u] != 1.f;
    }
    // (Probabilities as bf16 for the second MMA, 2^-8 of each at most; their sums as they are.)
    const uint32_t pb[2] = {movmatrix_trans(pack_bf16x2(pr[0], pr[1])), movmatrix_trans(pack_bf16x2(pr[2], pr[3]))};
    if (__any_sync(0xffffffffu, any_rescale)) {
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            g.o[mt][0] *= alpha[0];
            g.o[mt][1] *= alpha[1];
            g.o[mt][2] *= alpha[0];
            g.o[mt][3] *= alpha[1];
        }
    }
#pragma unroll
    for (int bt = 0; bt < BATCHES; ++bt) {
        if (bt + 1 < BATCHES) fetch_v(bt + 1);
#pragma unroll
        for (int e = 0; e < AHEAD; ++e) mma_bf16_16816(g.o[bt * AHEAD + e], fr[bt & 1][e], pb[0], pb[1]);
    }
}

// The ring of stages in a CTA's shared memory: [stage][K, V][slice][head][64-column chunk][row].
struct PagedRing {
    uint8_t* base;
    uint64_t *full, *empty;
    int stages, tile_bytes, slice_bytes;  // tile: K or V of a stage; slice: K or V of one
    __device__ __forceinline__ uint8_t* slice(int stage, int v, int i) const { return base + (size_t)(2 * stage + v) * tile_bytes + i * slice_bytes; }
};

// The producer warp's side of a step of n slices; lane i has page and first row of slice i.  The stage is free.  (Whole warp, an elected lane
// issuing: a lane per copy took 120 clk for each, and a step of eight slices of one head of 128, 16 copies, 1950 clk.)
__device__ __forceinline__ void ask_slices(const PagedRing& r, const CUtensorMap& tm_k, const CUtensorMap& tm_v, const DecodePagedParams& p, int st, int n, int page,
                                           int row, int head0, int b) {
    const int lane = threadIdx.x & 31;
    if (lane < n && (page < 0 || page >= p.num_pages)) {
        report_fault(p.fault, FAULT_BAD_KV_RANGE, (uint32_t)b);
        page = p.num_pages;  // (behind the last: reads as zero)
    }
    if (lane == 0) mbar_arrive_expect_tx(&r.full[st], (uint32_t)(2 * n * r.slice_bytes));
    __syncwarp();
    for (int i = 0; i < n; ++i) {
        const int pg = __shfl_sync(0xffffffffu, page, i), rw = __shfl_sync(0xffffffffu, row, i);
        tma_load_5d_warp(r.slice(st, 0, i), &tm_k, &r.full[st], 0, rw, 0, head0, pg);
        tma_load_5d_warp(r.slice(st, 1, i), &tm_v, &r.full[st], 0, rw, 0, head0, pg);
    }
}

// Every copy issued has landed before the CTA retires (it: steps so far).
__device__ __forceinline__ void drain(const PagedRing& r, int it) {
    if ((threadIdx.x & 31) != 0) return;
    for (int back = 1; back <= r.stages && back <= it; ++back) {
        const int j = it - back;
        mbar_wait(&r.full[j % r.stages], (j / r.stages) & 1);
    }
}

// Folds the records of a CTA's consumer warps, of which `slices` have the same G heads (set, of `sets`: this warp's heads, slice: its place among them), through the
// shared memory at `smem`, which nothing else uses any more.  weigh(n, s, mx, z, wt) gets maximum and sum over the slices of the set's
// head n and this lane's slice's weight relative to the maximum, in eight lanes per row (s: slice, from `slices` on none), and
// returns what the slice's values are multiplied by; store(n, d, sum) gets columns d to d + 3.  All of it runs once per call, from
// instructions fetched cold, so loops are rolled and the weights worked out once.  (A row at a time, normalised records with
// log-sum-exps: one token of 28/4 heads of 128 over 513 keys 9.3 us, of which the fold was 2.8.)
template <int HD, typename W, typename S>
__device__ __forceinline__ void fold_warps(const GroupState<HD>& group, uint8_t* smem, int sets, int slices, int set, int slice, int G, W&& weigh, S&& store) {
    constexpr int RS = HD + 4;  // floats from one head's row of a warp's record to the next
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, q4 = lane & 3, ncw = sets * slices;
    float* rec = reinterpret_cast<float*>(smem);                                   // [warp][8 heads][RS]
    float2* rec_ml = reinterpret_cast<float2*>(rec + (size_t)ncw * 8 * RS);  // [warp][8]
    float* rec_w = reinterpret_cast<float*>(rec_ml + ncw * 8);
    static_assert(2 * 8 * (RS + 3) <= 2 * 16 * HD, "records, sums and weights of two warps in a KV head's slice of K and V of two stages");
    consumer_sync(ncw);  // every warp is through with the stages; no copy is in flight any more
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const float ls = group.sum(u);
        const int n = warp * 8 + q4 * 2 + u;
        if (g4 == 0) rec_ml[n] = make_float2(group.m[u], ls);
        float* dst = rec + (size_t)n * RS + g4;
#pragma unroll
        for (int mt = 0; mt < HD / 16; ++mt) {
            dst[mt * 16] = group.o[mt][u];
            dst[mt * 16 + 8] = group.o[mt][u + 2];
        }
    }
    consumer_sync(ncw);
#pragma unroll 1
    for (int n0 = slice * 4; n0 < G; n0 += slices * 4) {  // four heads a turn, a lane per slice
        const int n = n0 + (lane >> 3), s = lane & 7, at = (s * sets + set) * 8 + n;
        const bool some = n < G && s < slices;
        const float2 ml = some ? rec_ml[at] : make_float2(-CUDART_INF_F, 0.f);
        float mx = ml.x;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (mx == -CUDART_INF_F) mx = 0.f;  // (nothing seen, or nothing that is a number)
        const float wt = ml.y != ml.y ? ml.y : fast_exp2(ml.x - mx);
        float z = ml.x == -CUDART_INF_F ? ml.y : wt * ml.y;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        const float f = weigh(n, s, mx, z, wt);
        if (some) rec_w[at] = f;
    }
    consumer_sync(ncw);
#pragma unroll 1
    for (int i = slice; i < G * (HD / 128); i += slices) {  // half a row (head dim 256) a turn
        const int n = i / (HD / 128), d = i % (HD / 128) * 128 + lane * 4;
        const float* src = rec + (size_t)(set * 8 + n) * RS + d;
        const float* wts = rec_w + set * 8 + n;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int s = 0; s < slices; ++s) {
            const float wt = *wts;
            const float4 v = *reinterpret_cast<const float4*>(src);
            acc.x = fmaf(wt, v.x, acc.x), acc.y = fmaf(wt, v.y, acc.y), acc.z = fmaf(wt, v.z, acc.z), acc.w = fmaf(wt, v.w, acc.w);
            src += (size_t)sets * 8 * RS, wts += sets * 8;
        }
        store(n, d, acc);
    }
}

// Equal shares: CTA x takes slices [x * per, (x + 1) * per) of all; grid.y: groups of KV heads.
template <int HD>
__global__ void __launch_bounds__(288, 1)
    sdpa_decode_paged_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                             const DecodePagedParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int HEAD = HD / 64 * SLICE_CHUNK;

    const int sets = p.nkv_cta * p.subs, ncw = sets * p.slices;  // sets of query heads, consumer warps
    PagedRing ring;
    ring.slice_bytes = p.nkv_cta * HEAD;
    ring.tile_bytes = p.slices * ring.slice_bytes;
    ring.base = smem;
    ring.stages = p.stages;
    ring.full = reinterpret_cast<uint64_t*>(smem + (size_t)p.stages * 2 * ring.tile_bytes);
    ring.empty = ring.full + p.stages;
    long long* cum = reinterpret_cast<long long*>(ring.empty + p.stages);  // slices in front of each sequence

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head0 = blockIdx.y * p.nkv_cta;
    const int G = p.nq / p.nkv;
    if (threadIdx.x == 32) {
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_v);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&ring.full[s], 1);
            mbar_init(&ring.empty[s], ncw);
        }
        fence_mbar_init();
    }
    // Up to here nothing depends on the kernels in front; everything below may.
    grid_dependency_wait();
    grid_launch_dependents();  // (the merge kernel waits for this grid before it reads the records)
    bool bad = threadIdx.x == 0 && *reinterpret_cast<volatile uint32_t*>(p.fault) != 0u;
    auto length = [&](int b) { return p.kv_len ? p.kv_len[b] : p.kv_len_uniform; };
    if (warp == 0)
        build_len_prefix(p.batch, cum, [&](int b) {
            const int len = length(b);
            if (len > p.max_len) {
                report_fault(p.fault, FAULT_BAD_KV_RANGE, (uint32_t)b);
                bad = true;
            }
            return seen_of(len, p.window, p.sinks).n;
        });
    if (__syncthreads_or(bad)) return;
    const long long total = cum[p.batch], per = share_size(total, p.ncta, p.slices);
    const long long g0 = (long long)blockIdx.x * per, g1 = min(total, g0 + per);
    if (g0 >= g1) return;
    int b = 0;
    for (int b0 = 0; b0 < p.batch - 1; b0 += 32) {  // sequences that end at or before the share's first slice
        const int n = __popc(__ballot_sync(0xffffffffu, b0 + lane < p.batch - 1 && cum[b0 + lane + 1] <= g0));
        b += n;
        if (n < 32) break;
    }
    if (warp == ncw) {
        // ------------------------------------------------------------------ producer
        // A step is up to `slices` slices of one sequence.
        const int i = lane;
        struct Step {
            int n, page, row;  // slices; page and first row of this lane's slice
        };
        int seq = -1;
        SeenKeys seen{};
        long long g = g0;
        auto next_step = [&]() {
            Step s{0, 0, 0};
            if (g >= g1) return s;
            while (cum[b + 1] <= g) ++b;
            if (seq != b) seen = seen_of(length(b), p.window, p.sinks), seq = b;
            s.n = (int)min((long long)p.slices, min(g1, cum[b + 1]) - g);
            if (i < s.n) {
                const int key = seen.slice((int)(g - cum[b]) + i) * 16, column = key / p.page;
                s.row = key - column * p.page;
                s.page = p.table[b * p.table_stride + column];
            }
            g += s.n;
            return s;
        };
        Step next = next_step();
        int it = 0;
        for (; next.n > 0; ++it) {
            const Step s = next;
            const int of = b;
            next = next_step();  // (its pages are on their way while this step's stage is waited for)
            const int st = it % p.stages;
            if (it >= p.stages && !mbar_wait_warp(&ring.empty[st], ((it / p.stages) - 1) & 1)) {
                if (lane == 0) report_fault(p.fault, FAULT_WAIT_EMPTY, it);
                break;
            }
            ask_slices(ring, tm_k, tm_v, p, st, s.n, s.page, s.row, head0, of);
        }
        drain(ring, it);
    } else if (warp < ncw) {
        // ------------------------------------------------------------------ consumers: a KV head, a slice of every step
        const int set = warp % sets, slice = warp / sets, hl = set / p.subs, sub = set - hl * p.subs;
        const int own = min(8, G - 8 * sub), own0 = (head0 + hl) * G + 8 * sub;  // this warp's query heads
        const int g4 = lane >> 2, q4 = lane & 3;  // accumulator row group, column pair
        int it = 0;
        bool ok = true;
        long long g = g0;
        GroupState<HD> group;
        while (ok && g < g1) {
            while (cum[b + 1] <= g) ++b;
            const long long seg_end = min(g1, cum[b + 1]);
            const SeenKeys seen = seen_of(length(b), p.window, p.sinks);
            const int first = (int)(g - cum[b]), seg = (int)(seg_end - g);
            group.load(p.q + b * p.q_stride_b + (long long)own0 * HD, own);
            for (int k0 = 0; k0 < seg; k0 += p.slices, ++it) {
                const int st = it % p.stages;
                if (!mbar_wait_warp(&ring.full[st], (it / p.stages) & 1)) {
                    if (lane == 0) report_fault(p.fault, FAULT_WAIT_FULL, it);
                    ok = false;
                    break;
                }
                if (k0 + slice < seg)
                    attend_slice<HD>(group, smem_u32(ring.slice(st, 0, slice)) + hl * HEAD, smem_u32(ring.slice(st, 1, slice)) + hl * HEAD,
                                         seen.keys_of(seen.slice(first + k0 + slice)), p.scale_log2);
                __syncwarp();
                if (lane == 0) mbar_arrive(&ring.empty[st]);
            }

            // Partial records: normalised out + natural-log lse.  Of the share's last segment (for most CTAs the only one) one, in
            // slice 0's place; of a sequence that ends inside the share one per slice.  (With one slice a step there is nothing to
            // fold: through shared memory all the same, a call took 1.4 us more.)
            const long long part = ((long long)blockIdx.x + b) * p.slices;
            if (p.slices > 1 && seg_end == g1) {  // CTA-uniform
                if (!ok) break;
                const long long row0 = part * p.nq + own0;
                fold_warps<HD>(group, smem, sets, p.slices, set, slice, own,
                    [&](int n, int s, float mx, float z, float wt) {
                        if (n < own && s == 0) p.part_lse[row0 + n] = z == 0.f ? -CUDART_INF_F : (mx + fast_log2(z)) * 0.6931471805599453f;
                        return z == 0.f ? 0.f : __fdividef(wt, z);
                    },
                    [&](int n, int d, float4 v) { *reinterpret_cast<float4*>(p.part_o + (row0 + n) * HD + d) = v; });
            } else if (ok) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float ls = group.sum(u);
                    const float inv = ls == 0.f ? 0.f : 1.f / ls;  // (what is no number goes on to the result)
                    const int n = q4 * 2 + u;
                    if (n >= own) continue;
                    const long long row = (part + slice) * p.nq + own0 + n;
                    if (g4 == 0) p.part_lse[row] = ls == 0.f ? -CUDART_INF_F : (group.m[u] + fast_log2(ls)) * 0.6931471805599453f;
                    float* dst = p.part_o + row * HD + g4;
#pragma unroll
                    for (int mt = 0; mt < HD / 16; ++mt) {
                        dst[mt * 16] = group.o[mt][u] * inv;
                        dst[mt * 16 + 8] = group.o[mt][u + 2] * inv;
                    }
                }
            }
            g = seg_end;
        }
        // A warp that gave up a wait does not fold: it meets the others at the fold's three barriers.
        if (!ok && p.slices > 1)
            for (int i = 0; i < 3; ++i) consumer_sync(ncw);
    }
}

// One launch: a cluster of p.ncta CTAs (at most eight) owns a sequence (grid.z) and a group of KV heads (grid.y), its CTAs equal parts of the slices.
// Each folds its warps' records and sends them, as they are, to the CTAs that finish the columns (the largest power of two of
// the cluster's), which weight, gate and store them: no records in global memory, no merge.  The sends are st.async, counted by
// an mbarrier of the CTA they go to, as in decode_sm100.cuh, whose comments have what was measured against a barrier of the
// cluster.
template <int HD>
__global__ void __launch_bounds__(288, 1)
    sdpa_decode_paged_cluster_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                                     const DecodePagedParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int HEAD = HD / 64 * SLICE_CHUNK;

    const int sets = p.nkv_cta * p.subs, ncw = sets * p.slices;  // sets of query heads, consumer warps
    PagedRing ring;
    ring.slice_bytes = p.nkv_cta * HEAD;
    ring.tile_bytes = p.slices * ring.slice_bytes;
    ring.base = smem;
    ring.stages = p.stages;
    ring.full = reinterpret_cast<uint64_t*>(smem + (size_t)p.stages * 2 * ring.tile_bytes);
    ring.empty = ring.full + p.stages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.z, rank = blockIdx.x, head0 = blockIdx.y * p.nkv_cta;
    const int G = p.nq / p.nkv, rows = p.nkv_cta * G, rows2 = (rows + 1) & ~1;
    const bool alone = p.ncta == 1;  // (st.async is for clusters: plain stores then)
    // The CTAs that finish `dc` columns of all rows each; per CTA of the cluster they get [row][column], in front of them [CTA][row]
    // maximum (log2 domain) and sum, and whether all of its waits ended well.
    const int dc_log2 = (HD == 256 ? 8 : 7) - (31 - __clz(p.ncta)), dc = 1 << dc_log2, finishers = HD >> dc_log2;
    uint64_t* gathered = ring.empty + p.stages;
    int* gave_up = reinterpret_cast<int*>(gathered + 1);
    float* cflag = reinterpret_cast<float*>(gathered + 2);     // [8]
    float2* cml = reinterpret_cast<float2*>(cflag + 8);         // [8][rows2]
    float* crec = reinterpret_cast<float*>(cml + 8 * rows2);    // [CTA][rows][dc]
    float* cweight = crec + (size_t)p.ncta * rows * dc;         // [rows][8]
    if (threadIdx.x == 32) {
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_v);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&ring.full[s], 1);
            mbar_init(&ring.empty[s], ncw);
        }
        mbar_init(gathered, 1);
        *gave_up = 0;
        fence_mbar_init();
        mbar_arrive_expect_tx(gathered, (uint32_t)(p.ncta * (4 + rows * (8 + dc * 4))));
    }
    cluster_sync_all();  // every CTA runs: its shared memory may be written
    // Up to here nothing depends on the kernels in front; everything below may.
    grid_dependency_wait();
    grid_launch_dependents();
    const uint32_t fault = threadIdx.x == 0 ? *reinterpret_cast<volatile uint32_t*>(p.fault) : 0u;
    const int len = p.kv_len ? p.kv_len[b] : p.kv_len_uniform;
    // The first steps of the CTAs come in order, so that without a window a CTA's first pages, which do not depend on the length, are
    // looked up beside it; what is left behind them is divided evenly.
    int page = 0, row = 0;  // producer: of this lane's slice of the next step
    auto look_up = [&](int slice) {
        const int column = slice * 16 / p.page;
        row = slice * 16 - column * p.page;
        page = p.table[b * p.table_stride + column];
    };
    const bool early = p.window >= p.max_len;
    if (early && warp == ncw && lane < p.slices && (rank * p.slices + lane) * 16 < p.max_len) look_up(rank * p.slices + lane);
    if (len > p.max_len) {  // (the same in all of the cluster's CTAs)
        if (threadIdx.x == 0) report_fault(p.fault, FAULT_BAD_KV_RANGE, (uint32_t)b);
        return;
    }
    const SeenKeys seen = seen_of(len, p.window, p.sinks);
    const int steps_all = (seen.n + p.slices - 1) / p.slices, rest = max(0, steps_all - p.ncta);
    const int more0 = p.ncta + rest * rank / p.ncta, steps = rank < steps_all ? 1 + p.ncta + rest * (rank + 1) / p.ncta - more0 : 0;
    auto first_of = [&](int step) { return (step == 0 ? rank : more0 + step - 1) * p.slices; };  // first slice of this CTA's step

    if (warp == ncw) {
        // ------------------------------------------------------------------ producer
        auto look_up_step = [&](int step) {
            const int at = first_of(step) + lane;
            if (step < steps && lane < p.slices && at < seen.n) look_up(seen.slice(at));
        };
        if (!early) look_up_step(0);
        int it = 0;
        for (; it < steps; ++it) {
            const int own_page = page, own_row = row, n = min(p.slices, seen.n - first_of(it));
            look_up_step(it + 1);
            const int st = it % p.stages;
            if (it >= p.stages && !mbar_wait_warp(&ring.empty[st], ((it / p.stages) - 1) & 1)) {
                if (lane == 0) report_fault(p.fault, FAULT_WAIT_EMPTY, it);
                break;
            }
            ask_slices(ring, tm_k, tm_v, p, st, n, own_page, own_row, head0, b);
        }
        drain(ring, it);
    } else if (warp < ncw) {
        // ------------------------------------------------------------------ consumers
        const int set = warp % sets, slice = warp / sets, hl = set / p.subs, sub = set - hl * p.subs;
        const int own = min(8, G - 8 * sub), own0 = hl * G + 8 * sub;  // this warp's query heads of the CTA's
        GroupState<HD> group;
        group.load(p.q + b * p.q_stride_b + (long long)(head0 * G + own0) * HD, own);
        bool ok = true;
        for (int it = 0; it < steps; ++it) {
            const int st = it % p.stages, at = first_of(it) + slice;
            if (!mbar_wait_warp(&ring.full[st], (it / p.stages) & 1)) {
                if (lane == 0) report_fault(p.fault, FAULT_WAIT_FULL, it);
                ok = false;
                break;
            }
            if (at < seen.n)
                attend_slice<HD>(group, smem_u32(ring.slice(st, 0, slice)) + hl * HEAD, smem_u32(ring.slice(st, 1, slice)) + hl * HEAD,
                                     seen.keys_of(seen.slice(at)), p.scale_log2);
            __syncwarp();
            if (lane == 0) mbar_arrive(&ring.empty[st]);
        }
        if (lane == 0 && (!ok || fault != 0u)) *reinterpret_cast<volatile int*>(gave_up) = 1;  // (no result is written)
        const uint32_t bar = smem_u32(gathered);
        fold_warps<HD>(group, smem, sets, p.slices, set, slice, own,
            [&](int n, int s, float mx, float z, float wt) {
                if (n < own && s < finishers) {
                    float2* to = cml + rank * rows2 + own0 + n;
                    if (alone) *to = make_float2(mx, z);
                    else st_async_f32x2(map_to_cta(smem_u32(to), s), make_float2(mx, z), map_to_cta(bar, s));
                }
                // (2^-6, taken back with the CTAs' weights: up to 64 records are added up before their sum of weights is divided by, and
                // values that a record of its own can hold must not run over in between.)
                return wt * 0.015625f;
            },
            [&](int n, int d, float4 v) {
                float* at = crec + (size_t)(rank * rows + own0 + n) * dc + (d & (dc - 1));
                const int to = d >> dc_log2;
                if (alone) *reinterpret_cast<float4*>(at) = v;
                else st_async_f32x4(map_to_cta(smem_u32(at), to), v, map_to_cta(bar, to));
            });
        if (warp == 0 && lane < finishers) {  // (behind the fold's barriers: every warp has said whether it gave up)
            const float good = *reinterpret_cast<volatile int*>(gave_up) ? 0.f : 1.f;
            if (alone) cflag[0] = good;
            else st_async_f32(map_to_cta(smem_u32(cflag + rank), lane), good, map_to_cta(bar, lane));
        }
    }
    // This CTA's columns, two a thread, once every record is in its own shared memory.  (Nothing is sent to a CTA that finishes none, and
    // what this one has sent is waited for by those it went to: no barrier of the cluster here.)
    if (!alone && (rank << dc_log2) >= HD) return;
    const int items = rows * (dc / 2);
    auto offset_of = [&](int item) {
        return (long long)b * p.o_stride_b + (long long)(head0 * G + (item >> (dc_log2 - 1))) * HD + rank * dc + (item & (dc / 2 - 1)) * 2;
    };
    uint32_t gw = p.gate && (int)threadIdx.x < items ? *reinterpret_cast<const uint32_t*>(p.gate + offset_of(threadIdx.x)) : 0u;
    __syncwarp();
    // Whether the records came is settled for the whole CTA before any warp goes on: each warp waits by its own clock.
    const bool came = alone || mbar_wait_cluster(gathered, 0);
    if (!__syncthreads_and(came)) {
        if (!came && lane == 0) report_fault(p.fault, FAULT_WAIT_FULL, 0x10000u);
        cluster_sync_all();  // (what is still under way here arrives before the other CTAs have gone)
        return;
    }
    const bool fine = __all_sync(0xffffffffu, (lane & 7) >= p.ncta || cflag[lane & 7] != 0.f);  // (the same in every warp)
    // The CTAs' weights of a row: eight lanes.
#pragma unroll 1
    for (int n0 = warp * 4; n0 < rows; n0 += (ncw + 1) * 4) {
        const int n = n0 + (lane >> 3), c = lane & 7;
        const float2 ml = n < rows && c < p.ncta ? cml[c * rows2 + n] : make_float2(-CUDART_INF_F, 0.f);
        float mx = ml.y == 0.f ? -CUDART_INF_F : ml.x;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float wt = ml.y == 0.f ? 0.f : fast_exp2(ml.x - mx);
        float z = wt * ml.y;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        if (n < rows) {
            cweight[n * 8 + c] = z == 0.f ? 0.f : __fdividef(wt * 64.f, z);
            if (p.out_lse && fine && rank == 0 && c == 0)
                p.out_lse[(long long)b * p.nq + head0 * G + n] = z == 0.f ? -CUDART_INF_F : fmaf(mx, 0.6931471805599453f, logf(z));
        }
    }
    __syncthreads();
    if (!fine) return;
#pragma unroll 1
    for (int item = threadIdx.x; item < items; item += blockDim.x) {
        const int n = item >> (dc_log2 - 1), d = (item & (dc / 2 - 1)) * 2;
        const long long eoff = offset_of(item);
        if (p.gate && item != (int)threadIdx.x) gw = *reinterpret_cast<const uint32_t*>(p.gate + eoff);
        float a0 = 0.f, a1 = 0.f;
#pragma unroll 2
        for (int c = 0; c < p.ncta; ++c) {
            const float wt = cweight[n * 8 + c];
            const float2 v = *reinterpret_cast<const float2*>(crec + (size_t)(c * rows + n) * dc + d);
            a0 = fmaf(wt, v.x, a0);
            a1 = fmaf(wt, v.y, a1);
        }
        const long long row = (long long)b * p.nq + head0 * G + n;
        if (p.out_f32) *reinterpret_cast<float2*>(p.out_f32 + row * HD + rank * dc + d) = make_float2(a0, a1);
        if (p.out) {
            if (p.gate) a0 = gated<true>(a0, (uint16_t)(gw & 0xffffu)), a1 = gated<true>(a1, (uint16_t)(gw >> 16));
            *reinterpret_cast<uint32_t*>(p.out + eoff) = pack_bf16x2(a0, a1);
        }
    }
}

// Merge of the records: a block takes ROWS query heads of a sequence, 8 / ROWS warps each.  What it costs is a chain of trips (the wait, the
// log-sum-exps and values) and the blocks that stand in line for it, so where there are rows enough a warp takes one on its
// own, and 64 registers let a block wait beside each decode CTA.  (48 sequences of 28 heads: 11.5 us as a block per row, which
// is 4.5 waves of them.)  Rows of few sequences go by sdpa_decode_merge_kernel, whose blocks divide the columns, too.
template <int HD, int ROWS>
__global__ void __launch_bounds__(256, ROWS == 1 ? 2 : 4) sdpa_decode_paged_merge_kernel(const DecodeMergeParams p) {
    constexpr int TEAM = 8 / ROWS, VPL = HD / 32, U = HD == 256 ? 2 : 4;  // warps of a row; values of a lane; records a warp has in flight
    __shared__ float s_acc[TEAM > 1 ? 8 * HD : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x * ROWS + warp / TEAM, b = blockIdx.y, member = warp % TEAM;
    // (The decode kernel released this one behind its own wait for the kernels in front: the lengths are final.)
    long long k_begin = 0, total = 0, k_len = 0;
    for (int i = lane; i < p.batch; i += 32) {
        const int n = seen_of(p.kv_len ? p.kv_len[i] : p.kv_len_uniform, p.window, p.sinks).n;
        total += n;
        if (i < b) k_begin += n;
        if (i == b) k_len = n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, o);
        k_begin += __shfl_xor_sync(0xffffffffu, k_begin, o);
        k_len += __shfl_xor_sync(0xffffffffu, k_len, o);
    }
    const bool live = h < p.nq;
    const long long eoff = (long long)b * p.o_stride_b + (long long)h * HD + lane * VPL;
    if (p.gate && live) prefetch_l2(p.gate + eoff);
    const long long per = share_size(total, p.ncta, p.slices), k_end = k_begin + k_len;
    const bool small = total < (1ll << 30);
    const int c_first = small ? (int)((uint32_t)k_begin / (uint32_t)per) : (int)(k_begin / per);
    const int c_last = k_len == 0 ? c_first : small ? (int)((uint32_t)(k_end - 1) / (uint32_t)per) : (int)((k_end - 1) / per);
    // The shares in front of the last one end with this sequence and have one record of it; the last one has one for each slice if
    // it goes on behind it.
    const int n_full = c_last - c_first;
    const int n_rec = k_len == 0 || !live ? 0 : n_full + (k_end == min(total, (c_last + 1) * per) ? 1 : p.slices);
    const long long part0 = ((long long)c_first + b) * p.slices;
    auto rec_of = [&](int j) { return part0 + (j < n_full ? (long long)j * p.slices : (long long)n_full * p.slices + (j - n_full)); };
    grid_dependency_wait();  // from here on the records are read
    grid_launch_dependents();
    const bool fault = *reinterpret_cast<volatile uint32_t*>(p.fault) != 0u;
    const float* lses = p.part_lse + h;
    float wu[U], acc[VPL];
    float4 ov[U][VPL / 4];
    auto load = [&](int j0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * TEAM;
            wu[u] = -CUDART_INF_F;
            if (j < n_rec) {
                const long long rec = rec_of(j);
                wu[u] = lses[rec * p.nq];
                const float* src = p.part_o + (rec * p.nq + h) * HD + lane * VPL;
#pragma unroll
                for (int i = 0; i < VPL / 4; ++i) ov[u][i] = *reinterpret_cast<const float4*>(src + 4 * i);
            }
        }
    };
    load(member);
    float mx = -CUDART_INF_F, z = 0.f;
    for (int j = lane; j < n_rec; j += 32) mx = fmaxf(mx, lses[rec_of(j) * p.nq]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (mx == -CUDART_INF_F) mx = 0.f;  // (no records, or none that are numbers)
    for (int j = lane; j < n_rec; j += 32) z += __expf(lses[rec_of(j) * p.nq] - mx);  // (L1 has them)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] = 0.f;
    for (int j0 = member; j0 < n_rec; j0 += TEAM * U) {
        if (j0 != member) load(j0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (wu[u] == -CUDART_INF_F) continue;  // an empty slice's record may hold anything
            const float w = __expf(wu[u] - mx);
#pragma unroll
            for (int i = 0; i < VPL / 4; ++i) {
                acc[4 * i] = fmaf(w, ov[u][i].x, acc[4 * i]), acc[4 * i + 1] = fmaf(w, ov[u][i].y, acc[4 * i + 1]);
                acc[4 * i + 2] = fmaf(w, ov[u][i].z, acc[4 * i + 2]), acc[4 * i + 3] = fmaf(w, ov[u][i].w, acc[4 * i + 3]);
            }
        }
    }
    if constexpr (TEAM > 1) {
#pragma unroll
        for (int i = 0; i < VPL / 4; ++i)
            *reinterpret_cast<float4*>(s_acc + warp * HD + lane * VPL + 4 * i) = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
        __syncthreads();
        if (member != 0) return;
#pragma unroll
        for (int t = 1; t < TEAM; ++t)
#pragma unroll
            for (int i = 0; i < VPL; ++i) acc[i] += s_acc[(warp + t) * HD + lane * VPL + i];
    }
    if (fault || !live) return;  // a status is set: no result
    const float inv = z == 0.f ? 0.f : 1.f / z;
    const long long row = (long long)b * p.nq + h;
    if (p.out_lse && lane == 0) p.out_lse[row] = z == 0.f ? -CUDART_INF_F : mx + __logf(z);
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] *= inv;
    if (p.out_f32) {
#pragma unroll
        for (int i = 0; i < VPL / 4; ++i)
            *reinterpret_cast<float4*>(p.out_f32 + row * HD + lane * VPL + 4 * i) = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
    }
    if (p.out) {
        uint32_t o[VPL / 2];
#pragma unroll
        for (int i = 0; i < VPL / 2; ++i) {
            if (p.gate) {
                const uint32_t gw = *reinterpret_cast<const uint32_t*>(p.gate + eoff + 2 * i);
                acc[2 * i] = gated<true>(acc[2 * i], (uint16_t)(gw & 0xffffu)), acc[2 * i + 1] = gated<true>(acc[2 * i + 1], (uint16_t)(gw >> 16));
            }
            o[i] = pack_bf16x2(acc[2 * i], acc[2 * i + 1]);
        }
        if constexpr (VPL == 8) *reinterpret_cast<uint4*>(p.out + eoff) = make_uint4(o[0], o[1], o[2], o[3]);
        else *reinterpret_cast<uint2*>(p.out + eoff) = make_uint2(o[0], o[1]);
    }
}

}  // namespace arc
