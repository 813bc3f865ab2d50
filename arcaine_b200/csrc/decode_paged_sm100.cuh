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
    int slices;   // 16-key slices of a stage; consumer warps = nkv_cta * slices
    int stages;
    int ncta;     // grid.x
};

template <int HD, int NT>
__global__ void __launch_bounds__(288, 1)
    sdpa_decode_paged_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                             const DecodePagedParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int CHUNK = 16 * 128;  // 64 columns of a slice: 16 rows x 128 bytes
    constexpr int HEAD = HD / 64 * CHUNK;

    const int ncw = p.nkv_cta * p.slices;  // consumer warps
    const int slice_bytes = p.nkv_cta * HEAD;  // of K or of V
    const int tile_bytes = p.slices * slice_bytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)p.stages * 2 * tile_bytes);
    uint64_t* empty = full + p.stages;
    long long* cum = reinterpret_cast<long long*>(empty + p.stages);  // slices in front of each sequence

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head0 = blockIdx.y * p.nkv_cta;
    const int G = p.nq / p.nkv;
    if (threadIdx.x == 32) {
        prefetch_tensormap(&tm_k);
        prefetch_tensormap(&tm_v);
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], ncw);
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
    constexpr int RS = HD + 4;  // floats from one head's row of a warp's record to the next

    if (warp == ncw) {
        // ------------------------------------------------------------------ producer
        // A step is up to `slices` slices of one sequence.  Lane i looks after K of slice i of it, lane 16 + i after V.
        const int i = lane & 15;
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
            if (it >= p.stages && !mbar_wait_warp(&empty[st], ((it / p.stages) - 1) & 1)) {
                if (lane == 0) report_fault(p.fault, FAULT_WAIT_EMPTY, it);
                break;
            }
            int page = s.page;
            if (i < s.n && (page < 0 || page >= p.num_pages)) {
                report_fault(p.fault, FAULT_BAD_KV_RANGE, (uint32_t)of);
                page = p.num_pages;  // (behind the last: reads as zero)
            }
            if (lane == 0) mbar_arrive_expect_tx(&full[st], (uint32_t)(2 * s.n * slice_bytes));
            __syncwarp();
            if (i < s.n) {
                const bool is_v = lane >= 16;
                tma_load_5d(smem + (size_t)(2 * st + is_v) * tile_bytes + i * slice_bytes, is_v ? &tm_v : &tm_k, &full[st], 0, s.row, 0, head0, page);
            }
            __syncwarp();
        }
        // Every copy issued above has landed before the CTA retires.
        if (lane == 0) {
            for (int back = 1; back <= p.stages && back <= it; ++back) {
                const int j = it - back;
                mbar_wait(&full[j % p.stages], (j / p.stages) & 1);
            }
        }
    } else if (warp < ncw) {
        // ------------------------------------------------------------------ consumers: a KV head, a slice of every step
        const int hl = warp % p.nkv_cta, slice = warp / p.nkv_cta, kvh = head0 + hl;
        const int g4 = lane >> 2;  // accumulator row group
        const int q4 = lane & 3;   // accumulator column pair
        const float sl = p.scale_log2;
        int it = 0;
        bool ok = true, folded = false;  // folded: this warp has been through the two barriers of the in-CTA fold
        long long g = g0;
        while (ok && g < g1) {
            while (cum[b + 1] <= g) ++b;
            const long long seg_end = min(g1, cum[b + 1]);
            const SeenKeys seen = seen_of(length(b), p.window, p.sinks);
            const int first = (int)(g - cum[b]), seg = (int)(seg_end - g);

            // Q^T fragments (B operand, hd x 8 heads) for this head's GQA group.
            uint32_t qf[NT][HD / 16][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int n = nt * 8 + g4;
                const bool valid = n < G;
                const uint16_t* qp = p.q + b * p.q_stride_b + ((long long)kvh * G + (valid ? n : 0)) * HD + q4 * 2;
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    qf[nt][kk][0] = valid ? *reinterpret_cast<const uint32_t*>(qp + kk * 16) : 0u;
                    qf[nt][kk][1] = valid ? *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 8) : 0u;
                }
            }
            float m[NT][2], l[NT][2];
            float o[NT][HD / 16][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                m[nt][0] = m[nt][1] = -CUDART_INF_F;
                l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
                for (int mt = 0; mt < HD / 16; ++mt) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.f;
            }

            for (int k0 = 0; k0 < seg; k0 += p.slices, ++it) {
                const int st = it % p.stages;
                if (!mbar_wait_warp(&full[st], (it / p.stages) & 1)) {
                    if (lane == 0) report_fault(p.fault, FAULT_WAIT_FULL, it);
                    ok = false;
                    break;
                }
                if (k0 + slice < seg) {
                    const uint32_t vis = seen.keys_of(seen.slice(first + k0 + slice));
                    // Swizzled addressing: 16-byte unit u of row r sits at unit u ^ (r & 7).
                    const uint32_t sK = smem_u32(smem + (size_t)2 * st * tile_bytes) + slice * slice_bytes + hl * HEAD;
                    const uint32_t sV = sK + tile_bytes;
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
                    constexpr int AHEAD = HD * NT > 256 ? 2 : 4, BATCHES = HD / 16 / AHEAD;
                    constexpr int CHAINS = NT == 1 ? 4 : 2;  // independent sums of S
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
                    float acc[NT][CHAINS][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int hh = 0; hh < CHAINS; ++hh) acc[nt][hh][0] = acc[nt][hh][1] = acc[nt][hh][2] = acc[nt][hh][3] = 0.f;
                    fetch_k(0);
#pragma unroll
                    for (int bt = 0; bt < BATCHES; ++bt) {
                        if (bt + 1 < BATCHES) fetch_k(bt + 1);
                        else if (NT == 1) fetch_v(0);  // (an even number of batches: into the other half)
#pragma unroll
                        for (int e = 0; e < AHEAD; ++e) {
                            const int kk = bt * AHEAD + e;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(acc[nt][kk % CHAINS], fr[bt & 1][e], qf[nt][kk][0], qf[nt][kk][1]);
                        }
                    }
                    static_assert(BATCHES % 2 == 0, "the first batch of V goes where the last one of K is not");
                    const bool v_lo = (vis >> g4) & 1u, v_hi = (vis >> (g4 + 8)) & 1u;
                    uint32_t pb[NT][2];
                    bool any_rescale = false;
                    float alpha[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float x[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float s = acc[nt][0][e] + acc[nt][1][e];
                            if constexpr (CHAINS == 4) s += acc[nt][2][e] + acc[nt][3][e];
                            s *= sl;
                            x[e] = ((e < 2) ? v_lo : v_hi) ? s : -CUDART_INF_F;
                        }
                        float pr[4];
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            float mx = fmaxf(x[u], x[u + 2]);
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                            const float m_new = fmaxf(m[nt][u], mx);
                            const float m_eff = (m_new == -CUDART_INF_F) ? 0.f : m_new;
                            alpha[nt][u] = (m_new == -CUDART_INF_F) ? 1.f : fast_exp2(m[nt][u] - m_new);
                            pr[u] = fast_exp2(x[u] - m_eff);
                            pr[u + 2] = fast_exp2(x[u + 2] - m_eff);
                            l[nt][u] = l[nt][u] * alpha[nt][u] + pr[u] + pr[u + 2];
                            m[nt][u] = m_new;
                            any_rescale |= alpha[nt][u] != 1.f;
                        }
                        pb[nt][0] = movmatrix_trans(pack_bf16x2(pr[0], pr[1]));
                        pb[nt][1] = movmatrix_trans(pack_bf16x2(pr[2], pr[3]));
                    }
                    if (__any_sync(0xffffffffu, any_rescale)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int mt = 0; mt < HD / 16; ++mt) {
                                o[nt][mt][0] *= alpha[nt][0];
                                o[nt][mt][1] *= alpha[nt][1];
                                o[nt][mt][2] *= alpha[nt][0];
                                o[nt][mt][3] *= alpha[nt][1];
                            }
                    }
                    if (NT > 1) fetch_v(0);
#pragma unroll
                    for (int bt = 0; bt < BATCHES; ++bt) {
                        if (bt + 1 < BATCHES) fetch_v(bt + 1);
#pragma unroll
                        for (int e = 0; e < AHEAD; ++e)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_bf16_16816(o[nt][bt * AHEAD + e], fr[bt & 1][e], pb[nt][0], pb[nt][1]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[st]);
            }

            // Partial record of this (CTA, sequence, slice): normalised out + natural-log lse.  Those of the share's last segment are
            // folded here first, into the record of slice 0 (decode_sm100.cuh).
            const bool fold_here = p.slices > 1 && seg_end == g1;  // CTA-uniform
            float* rec = reinterpret_cast<float*>(smem);               // [warp][NT * 8 heads][RS]
            float* rec_lse = rec + (size_t)ncw * NT * 8 * RS;          // [warp][NT * 8]
            if (fold_here) {
                consumer_sync(ncw);  // every warp is through with the stages; no copy is in flight any more
                folded = true;
            }
            if (ok) {
                const long long part = ((long long)blockIdx.x + b) * p.slices + slice;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float inv[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float ls = l[nt][u];
                        ls += __shfl_xor_sync(0xffffffffu, ls, 4);
                        ls += __shfl_xor_sync(0xffffffffu, ls, 8);
                        ls += __shfl_xor_sync(0xffffffffu, ls, 16);
                        inv[u] = ls == 0.f ? 0.f : 1.f / ls;  // (what is no number goes on to the result)
                        const int n = nt * 8 + q4 * 2 + u;
                        const float lse = ls == 0.f ? -CUDART_INF_F : (m[nt][u] + fast_log2(ls)) * 0.6931471805599453f;
                        if (g4 == 0) {
                            if (fold_here) rec_lse[warp * NT * 8 + n] = lse;
                            else if (n < G) p.part_lse[part * p.nq + (long long)kvh * G + n] = lse;
                        }
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int n = nt * 8 + q4 * 2 + u;
                        if (fold_here || n < G) {
                            float* dst = fold_here ? rec + ((size_t)warp * NT * 8 + n) * RS
                                                   : p.part_o + (part * p.nq + (long long)kvh * G + n) * HD;
#pragma unroll
                            for (int mt = 0; mt < HD / 16; ++mt) {
                                dst[mt * 16 + g4] = o[nt][mt][u] * inv[u];
                                dst[mt * 16 + g4 + 8] = o[nt][mt][u + 2] * inv[u];
                            }
                        }
                    }
                }
            }
            if (fold_here) {
                consumer_sync(ncw);  // all records of the CTA are in shared memory
                const long long row0 = ((long long)blockIdx.x + b) * p.slices * p.nq + (long long)kvh * G;
                for (int n = slice; n < G; n += p.slices) {
                    const float li = lane < p.slices ? rec_lse[(lane * p.nkv_cta + hl) * NT * 8 + n] : -CUDART_INF_F;
                    float mx = li;
#pragma unroll
                    for (int e = 4; e > 0; e >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, e));
                    mx = __shfl_sync(0xffffffffu, mx, 0);
                    if (mx == -CUDART_INF_F) mx = 0.f;  // (all empty, or no numbers)
                    float z = __expf(li - mx);
                    const float e0 = z;
#pragma unroll
                    for (int e = 4; e > 0; e >>= 1) z += __shfl_xor_sync(0xffffffffu, z, e);
                    z = __shfl_sync(0xffffffffu, z, 0);
                    const float weight = z == 0.f ? 0.f : e0 / z;
                    float4 acc[HD / 128];
#pragma unroll
                    for (int j = 0; j < HD / 128; ++j) acc[j] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int s = 0; s < p.slices; ++s) {
                        const float wt = __shfl_sync(0xffffffffu, weight, s);
                        const float* src = rec + ((size_t)(s * p.nkv_cta + hl) * NT * 8 + n) * RS + lane * 4;
#pragma unroll
                        for (int j = 0; j < HD / 128; ++j) {  // (an empty slice's record holds zeros)
                            const float4 ov = *reinterpret_cast<const float4*>(src + 128 * j);
                            acc[j].x = fmaf(wt, ov.x, acc[j].x);
                            acc[j].y = fmaf(wt, ov.y, acc[j].y);
                            acc[j].z = fmaf(wt, ov.z, acc[j].z);
                            acc[j].w = fmaf(wt, ov.w, acc[j].w);
                        }
                    }
                    const float rec_l = z == 0.f ? -CUDART_INF_F : mx + __logf(z);
#pragma unroll
                    for (int j = 0; j < HD / 128; ++j) *reinterpret_cast<float4*>(p.part_o + (row0 + n) * HD + lane * 4 + 128 * j) = acc[j];
                    if (lane == 0) p.part_lse[row0 + n] = rec_l;
                }
            }
            g = seg_end;
        }
        // A warp that gave up a wait never reached the fold: it still meets the others at both barriers.
        if (!folded && p.slices > 1) {
            consumer_sync(ncw);
            consumer_sync(ncw);
        }
    }
}

}  // namespace arc
