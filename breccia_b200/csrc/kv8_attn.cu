// Attention over 8-bit pages (value = code * 2^e, one exponent per page, kv head and side; brc_pool_create_kv8), for one
// or several tokens per sequence.
//
//   out[i,h] = sigmoid(gate) * sum_c softmax_c(scale * q.k_c) v_c,   c < len - (T - 1 - i)
//
// What bounds it: one token of 8 heads per kv head does 32 FLOP per cached byte, far under the 260 a B200's tensor cores
// have per byte of HBM, so the cache stream is the floor - if converting it keeps up: 24 bytes per SM and clock have to
// become binary16 operands.  Hence:
//   - the codes go to the tensor cores as the exact binary16 numbers they are (cvt of e4m3 pairs; byte permute and one
//     subtraction for int8), never scaled: K's scale multiplies the finished dot product, V's joins the exponent of
//     the probability, so scales cost one multiply per 16 cells and row instead of one per value;
//   - mma.sync m16n8k16 with the CACHE as the 16-row operand and the query rows as the 8-column one.  tcgen05 would pad 8
//     rows to 64 or 128 and want the converted operand written back to shared memory, twice the bytes the codes
//     themselves cost; the warp-level form takes it from the registers the conversion leaves it in.  Its rate is
//     not the limit: 32 of them per page and head against 350 clocks of HBM time;
//   - fragments are cut so that a thread's sixteen consecutive bytes are one 16-byte shared-memory read: the sum over
//     head_dim may run in any order, so K's columns are dealt out 16 bytes to a thread, and V's columns likewise become
//     the output rows; the 128-byte swizzle of the TMA box keeps every such read free of bank conflicts;
//   - all (sequence, kv-head group, pass) units form one list of page-units cut into equal shares, one persistent CTA per
//     SM; one warp streams the pages with TMA into a ring, eight consume.  A unit cut by a share boundary leaves partial
//     results in the caller's workspace, and a second kernel, launched with its prologue overlapped (programmatic
//     dependent launch), merges them.  No counters and no flags: nothing survives a call, so calls with workspaces of
//     their own may overlap.
//
// Two running maxima per row: m of the scores s (for the sum of probabilities), and M of s + e_v, the exponent at which a
// cell's V codes enter the result.  Weights are 2^(s + e_v - M + 15): at most 2^15, so binary16 keeps cells down to 2^-39 of
// the heaviest one, and a page whose V scale dwarfs the others' neither overflows nor silences them.
#include <algorithm>
#include <atomic>

#include "brc_internal.h"
#include "kv8.cuh"

namespace {

constexpr uint32_t WARPS = 8, CONSUMERS = WARPS * 32, THREADS = CONSUMERS + 32;
constexpr uint32_t PASS_ROWS = 32;       // query rows (tokens x heads of a kv head) that share one stream of the cache
constexpr uint32_t MIN_SHARE = 4;        // page-units a CTA takes at least
constexpr uint32_t SMEM_LIMIT = 232448;  // 227 KiB
constexpr uint32_t MAX_STAGES = 24;
constexpr uint32_t SCRATCH_ROW = 132;    // floats between rows of the merge buffer: 128 and a shift of one 16-byte group
constexpr float NONE = -1e30f;           // running maximum before any cell

struct AttnParams {
    const void *q;
    void *out;
    const float *gate;
    const uint32_t *block_tables, *seq_lens, *cu_q;
    const uint8_t *k_layer, *v_layer;
    uint64_t *prefix;        // workspace: pages before each sequence
    float *ml;               // [slot][row of a unit][m, M, l, -]
    float *acc;              // [slot][row of a unit][head_dim]
    uint32_t *status;
    uint64_t page_bytes;
    uint32_t q_dtype, out_dtype, gate_head_stride;
    uint32_t table_stride, n_seqs, max_seq_len, max_q, n_pages, page0;   // page0: layer * n_pages
    uint32_t n_head, n_kv, group, kvb, row_groups;                        // row_groups: warps that split a pass's rows
    uint32_t pass_rows, passes, units_per_seq, n_stages;
    float scale_log2;
};

struct Smem {   // byte offsets behind the ring
    uint32_t stage_bytes, q, q_lo, scratch, stat, row_fac, row_vis, bars, sched, total;
};

__host__ __device__ inline Smem smem_layout(uint32_t hd, uint32_t kvb, uint32_t pass_rows, bool prec, uint32_t n_stages) {
    Smem s;
    s.stage_bytes = kvb * 2u * 16u * hd;
    uint32_t at = n_stages * s.stage_bytes;
    s.q = at;
    at += kvb * pass_rows * hd * 2u;
    s.q_lo = at;
    if (prec) at += kvb * pass_rows * hd * 2u;
    s.scratch = at;
    at += WARPS * 8u * SCRATCH_ROW * 4u;
    s.stat = at;
    at += WARPS * 16u * 4u * 4u;   // [warp][row of two tiles][m, M, l, -]
    s.row_fac = at;
    at += kvb * pass_rows * 4u;
    s.row_vis = at;
    at += pass_rows * 4u;
    s.bars = at;
    at += 2u * MAX_STAGES * 8u;
    s.sched = at;
    at += 257u * 8u + 64u;
    s.total = at;
    return s;
}

__device__ __forceinline__ uint32_t tokens_of(const AttnParams &p, uint32_t s) { return p.cu_q ? p.cu_q[s + 1] - p.cu_q[s] : p.max_q; }
__device__ __forceinline__ uint32_t cells_of(const AttnParams &p, uint32_t s) { return min(p.seq_lens[s], p.max_seq_len); }
__device__ __forceinline__ uint32_t pages_of(const AttnParams &p, uint32_t s) {
    return tokens_of(p, s) ? (cells_of(p, s) + 15u) / 16u : 0u;
}
__device__ __forceinline__ uint64_t share_of(uint64_t total, uint32_t grid) {
    const uint64_t s = (total + grid - 1u) / grid;
    return s > MIN_SHARE ? s : MIN_SHARE;
}

__device__ __forceinline__ void store_out(const AttnParams &p, uint64_t at, float a, float b, float c, float d) {
    if (p.out_dtype == 0) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) = make_float4(a, b, c, d);
    } else if (p.out_dtype == 1) {
        *reinterpret_cast<uint2 *>(static_cast<__half *>(p.out) + at) = make_uint2(brc::pack2<1>(a, b), brc::pack2<1>(c, d));
    } else {
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(p.out) + at) = make_uint2(brc::pack2<2>(a, b), brc::pack2<2>(c, d));
    }
}

// Four values of one output row, gated and stored.  `head_row`: token * n_head + head.
__device__ __forceinline__ void finish_row(const AttnParams &p, uint32_t hd, uint64_t head_row, uint32_t d, float (&v)[4]) {
    if (p.gate) {
        const float *g = p.gate + head_row * p.gate_head_stride + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= 1.f / (1.f + __expf(-g[i]));
    }
    store_out(p, head_row * hd + d, v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ float4 lds128f(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

// One load of q rows in any of the three types: eight consecutive values of head row `r` from column d.
__device__ __forceinline__ void load_q8(const AttnParams &p, uint64_t at, float (&v)[8]) {
    if (p.q_dtype == 0) brc::load8<0>(static_cast<const float *>(p.q) + at, true, v);
    else if (p.q_dtype == 1) brc::load8<1>(static_cast<const __half *>(p.q) + at, true, v);
    else brc::load8<2>(static_cast<const __nv_bfloat16 *>(p.q) + at, true, v);
}

// A share's walk over the units: sequence, unit within it, first page.
struct Cursor {
    uint64_t pos, end;
    uint32_t s, u, pg;
};

struct Segment {
    uint32_t s, u, pg, n, pages;
};

__device__ __forceinline__ bool next_segment(const AttnParams &p, Cursor &c, Segment &g) {
    while (c.pos < c.end) {
        const uint32_t pages = pages_of(p, c.s);
        if (pages == 0 || c.u == p.units_per_seq) {
            ++c.s;
            c.u = c.pg = 0;
            continue;
        }
        const uint64_t left = c.end - c.pos;
        g.s = c.s;
        g.u = c.u;
        g.pg = c.pg;
        g.pages = pages;
        g.n = (uint32_t)(pages - c.pg < left ? pages - c.pg : left);
        c.pos += g.n;
        c.pg = 0;
        ++c.u;
        return true;
    }
    return false;
}

// RT: tiles of eight query rows that a warp carries.  PREC: q and the probabilities as two binary16 parts each.
template <int HD, uint32_t CODE, bool PREC, int RT>
__global__ void __launch_bounds__(THREADS, 1) kv8_attn_kernel(const __grid_constant__ CUtensorMap tm, const AttnParams p) {
    constexpr uint32_t SLABS = HD / 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    const Smem L = smem_layout(HD, p.kvb, p.pass_rows, PREC, p.n_stages);
    const uint32_t base = brc::smem_u32(smem);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t full0 = base + L.bars, empty0 = full0 + MAX_STAGES * 8u;
    uint64_t *chunk_prefix = reinterpret_cast<uint64_t *>(smem + L.sched);   // [257]: pages before each thread's sequences
    Cursor *cursor = reinterpret_cast<Cursor *>(smem + L.sched + 257u * 8u);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- the cut: pages of all sequences, summed by 256 threads over equal runs of sequences
    const uint32_t per_thread = (p.n_seqs + CONSUMERS - 1u) / CONSUMERS;
    if (tid < CONSUMERS) {
        uint64_t sum = 0;
        for (uint32_t i = 0; i < per_thread; ++i) {
            const uint32_t s = tid * per_thread + i;
            if (s >= p.n_seqs) break;
            sum += pages_of(p, s);
            if (blockIdx.x == 0) {
                if (p.seq_lens[s] > p.max_seq_len) { atomicOr(p.status, BRC_DEV_BAD_POS); p.status[1] = p.seq_lens[s]; }
                if (tokens_of(p, s) > p.max_q) { atomicOr(p.status, BRC_DEV_BAD_POS); p.status[1] = tokens_of(p, s); }
            }
        }
        uint64_t run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t up = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= (uint32_t)o) run += up;
        }
        chunk_prefix[tid + 1] = run;   // within the warp, for now
        if (tid == 0) chunk_prefix[0] = 0;
    }
    if (tid == CONSUMERS) {
        const uint32_t users = p.kvb * p.row_groups;
        for (uint32_t i = 0; i < p.n_stages; ++i) {
            brc::mbar_init(full0 + 8u * i, 1u);
            brc::mbar_init(empty0 + 8u * i, users);
        }
        brc::mbar_fence_init();
        brc::tma_prefetch_desc(&tm);
    }
    __syncthreads();
    uint64_t before = 0;
    if (tid < CONSUMERS)
        for (uint32_t w = 0; w < warp; ++w) before += chunk_prefix[w * 32u + 32u];
    __syncthreads();
    if (tid < CONSUMERS) chunk_prefix[tid + 1] += before;
    __syncthreads();
    const uint64_t total = chunk_prefix[CONSUMERS] * p.units_per_seq;
    const uint64_t share = share_of(total, gridDim.x);
    const uint64_t lo = min(total, blockIdx.x * share), hi = min(total, lo + share);
    if (blockIdx.x == 0 && tid < CONSUMERS) {   // for the merging kernel
        uint64_t at = chunk_prefix[tid];
        if (tid == 0) p.prefix[0] = 0;
        for (uint32_t i = 0; i < per_thread; ++i) {
            const uint32_t s = tid * per_thread + i;
            if (s >= p.n_seqs) break;
            at += pages_of(p, s);
            p.prefix[s + 1] = at;
        }
    }
    if (lo >= hi) return;
    if (tid == 0) {
        uint32_t a = 0, b = CONSUMERS;   // last run of sequences that begins at or before lo and holds pages behind it
        while (b - a > 1u) {
            const uint32_t mid = (a + b) >> 1;
            if (chunk_prefix[mid] * p.units_per_seq <= lo) a = mid; else b = mid;
        }
        uint64_t at = chunk_prefix[a] * p.units_per_seq;
        uint32_t s = a * per_thread;
        uint32_t pages;
        while (true) {
            pages = pages_of(p, s);
            if (at + (uint64_t)pages * p.units_per_seq > lo) break;
            at += (uint64_t)pages * p.units_per_seq;
            ++s;
        }
        cursor->pos = lo;
        cursor->end = hi;
        cursor->s = s;
        cursor->u = (uint32_t)((lo - at) / pages);
        cursor->pg = (uint32_t)((lo - at) % pages);
    }
    __syncthreads();
    Cursor cur = *cursor;
    Segment g;

    if (warp == WARPS) {
        // ------------------------------------------------------------------ producer: one page-unit per stage
        const uint64_t policy = brc::l2_policy_evict_first();
        uint32_t stage = 0, parity = 1;   // the first round finds every stage empty
        bool ok = true;
        while (ok && next_segment(p, cur, g)) {
            const uint32_t row = (g.u / p.passes) * p.kvb * 16u;
            const uint32_t *table = p.block_tables + (uint64_t)g.s * p.table_stride + g.pg;
            uint32_t ahead = lane < g.n ? table[lane] : 0u;
            for (uint32_t i0 = 0; ok && i0 < g.n; i0 += 32u) {
                const uint32_t ids = ahead;
                if (i0 + 32u + lane < g.n) ahead = table[i0 + 32u + lane];
                const uint32_t m = min(32u, g.n - i0);
                for (uint32_t i = 0; i < m; ++i) {
                    uint32_t id = __shfl_sync(0xffffffffu, ids, i);
                    if (id >= p.n_pages) id = 0;   // the consumers report it and mask the cells
                    ok = brc::mbar_wait(empty0 + 8u * stage, parity);
                    if (!ok) break;
                    if (lane == 0) {
                        brc::mbar_arrive_expect_tx(full0 + 8u * stage, L.stage_bytes);
#pragma unroll
                        for (uint32_t sl = 0; sl < SLABS; ++sl)
                            brc::tma_load_4d(base + stage * L.stage_bytes + sl * (L.stage_bytes / SLABS), &tm, (int32_t)(sl * 128u), (int32_t)row,
                                             (int32_t)(p.page0 + id), 0, full0 + 8u * stage, policy);
                    }
                    if (++stage == p.n_stages) { stage = 0; parity ^= 1u; }
                }
            }
        }
        if (!ok && lane == 0) { atomicOr(p.status, BRC_DEV_WAIT_LIMIT); p.status[1] = blockIdx.x; }
        return;
    }

    // ---------------------------------------------------------------------- consumers
    const uint32_t t = lane & 3u, gr = lane >> 2;            // thread of a group, group
    const uint32_t hk = warp % p.kvb, rg = warp / p.kvb % p.row_groups;
    const uint32_t lanes = WARPS / (p.kvb * p.row_groups);   // warps that take pages in turn
    const uint32_t pl = warp / (p.kvb * p.row_groups);
    const uint32_t slab_bytes = p.kvb * 2u * 16u * 128u;     // [K|V][head][cell][128]
    float *scratch = reinterpret_cast<float *>(smem + L.scratch);
    float4 *stat = reinterpret_cast<float4 *>(smem + L.stat);
    float *row_fac = reinterpret_cast<float *>(smem + L.row_fac);
    uint32_t *row_vis = reinterpret_cast<uint32_t *>(smem + L.row_vis);
    const uint32_t q_frag = base + L.q + (hk * p.pass_rows + rg * RT * 8u) * HD * 2u + lane * 16u;
    const uint32_t q_frag_lo = base + L.q_lo + (hk * p.pass_rows + rg * RT * 8u) * HD * 2u + lane * 16u;
    const uint64_t code_bytes = (uint64_t)p.n_kv * 16u * HD;
    uint32_t done = 0;   // page-units of the segments before this one
    bool ok = true;

    while (next_segment(p, cur, g)) {
        const uint32_t hg = g.u / p.passes, pass = g.u % p.passes;
        const uint32_t n_q = tokens_of(p, g.s), len = cells_of(p, g.s);
        const uint64_t tok0 = p.cu_q ? p.cu_q[g.s] : (uint64_t)g.s * p.max_q;
        const uint32_t rows = min(n_q, p.max_q) * p.group;   // of a kv head, over all passes

        // q rows of this unit, scaled by a power of two to at most 2^15 in magnitude and laid out as the B fragments of the
        // K product: [8-row tile][pair of 16-column steps][lane][2 x 4 values]; column d belongs to step
        // 8 (d / 128) + 4 (d / 16 % 2) + d / 4 % 4 and thread d / 32 % 4 of its row's group.
        for (uint32_t r0 = warp; r0 < p.kvb * p.pass_rows; r0 += WARPS) {
            const uint32_t h = r0 / p.pass_rows, r = r0 % p.pass_rows, gr_row = pass * p.pass_rows + r;
            const bool live = gr_row < rows;
            const uint32_t tok = gr_row / p.group, head = (hg * p.kvb + h) * p.group + gr_row % p.group;
            const uint32_t d = lane * 8u;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
            if (live && d < HD) load_q8(p, ((tok0 + tok) * p.n_head + head) * HD + d, v);
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
            for (int m = 16; m; m >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
            const int ex = max((int)(__float_as_uint(amax) >> 23) - 127, -100);
            const float up = brc::exp2_int(14 - min(ex, 127));
            if (lane == 0) {
                row_fac[r0] = amax <= 3.402823466e38f ? brc::exp2_int(ex - 14) * p.scale_log2 : __uint_as_float(0x7fffffffu);
                if (h == 0) row_vis[r] = live && len + tok + 1u > n_q ? len + tok + 1u - n_q : 0u;
            }
            if (d < HD) {
                const uint32_t tile = r / 8u, step = 8u * (d / 128u) + 4u * (d / 16u % 2u) + d / 4u % 4u;   // of the first four; the next four are step + 1
                const uint32_t frag_lane = (r % 8u) * 4u + d / 32u % 4u;
                const uint32_t at = (h * p.pass_rows + tile * 8u) * HD * 2u + ((step / 2u) * 32u + frag_lane) * 16u;
                float hi16[8], lo16[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float x = v[i] * up;
                    hi16[i] = __half2float(__float2half_rn(x));
                    lo16[i] = x - hi16[i];
                }
                *reinterpret_cast<uint4 *>(smem + L.q + at) = make_uint4(brc::pack_half2(hi16[0], hi16[1]), brc::pack_half2(hi16[2], hi16[3]),
                                                                         brc::pack_half2(hi16[4], hi16[5]), brc::pack_half2(hi16[6], hi16[7]));
                if (PREC)
                    *reinterpret_cast<uint4 *>(smem + L.q_lo + at) = make_uint4(brc::pack_half2(lo16[0], lo16[1]), brc::pack_half2(lo16[2], lo16[3]),
                                                                                brc::pack_half2(lo16[4], lo16[5]), brc::pack_half2(lo16[6], lo16[7]));
            }
        }
        brc::named_bar_sync(1, CONSUMERS);

        float o[RT][SLABS * 8][4];
        float m_run[RT][2], w_run[RT][2], l_run[RT][2], fac[RT][2];
        uint32_t vis[RT][2];
#pragma unroll
        for (int n = 0; n < RT; ++n) {
#pragma unroll
            for (int j = 0; j < (int)SLABS * 8; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[n][j][i] = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t r = (rg * RT + n) * 8u + 2u * t + i;
                m_run[n][i] = w_run[n][i] = NONE;
                l_run[n][i] = 0.f;
                fac[n][i] = row_fac[hk * p.pass_rows + r];
                vis[n][i] = row_vis[r];
            }
        }

        // scales of this warp's next 32 page-units, one a lane, fetched a batch ahead; a page id out of range shows as a
        // negative scale
        const uint32_t *table = p.block_tables + (uint64_t)g.s * p.table_stride + g.pg;
        const uint32_t first = (pl + lanes - done % lanes) % lanes;
        auto fetch = [&](uint32_t i0, float &ks, float &vs) {
            const uint32_t i = i0 + lanes * lane;
            ks = vs = 1.f;
            if (i < g.n) {
                const uint32_t id = table[i];
                if (id < p.n_pages) {
                    const uint64_t at = id * p.page_bytes + code_bytes + (hg * p.kvb + hk) * 4u;
                    ks = *reinterpret_cast<const float *>(p.k_layer + at);
                    vs = *reinterpret_cast<const float *>(p.v_layer + at);
                } else {
                    ks = -1.f;
                    atomicOr(p.status, BRC_DEV_BAD_PAGE);
                    p.status[1] = id;
                }
            }
        };
        float ks_now, vs_now, ks_next = 1.f, vs_next = 1.f;
        fetch(first, ks_next, vs_next);
        ks_now = ks_next;
        vs_now = vs_next;

        for (uint32_t i = first, k = 0; i < g.n; i += lanes, ++k) {
            if (k % 32u == 0u) {
                ks_now = ks_next;
                vs_now = vs_next;
                fetch(i + lanes * 32u, ks_next, vs_next);
            }
            const float ks = __shfl_sync(0xffffffffu, ks_now, k % 32u), vs = __shfl_sync(0xffffffffu, vs_now, k % 32u);
            const uint32_t unit = done + i, stage = unit % p.n_stages;
            ok = ok && brc::mbar_wait(full0 + 8u * stage, unit / p.n_stages & 1u);
            if (!ok) break;   // the producer gave up or its copy never came: no further wait, the sums stay as they are
            const uint32_t buf = base + stage * L.stage_bytes;
            const uint32_t cell0 = (g.pg + i) * 16u;

            // ---- S^T[16 cells][8 rows] = K q^T, over exact codes
            float s[RT][4];
            {
                float part[RT][2][4];
#pragma unroll
                for (int n = 0; n < RT; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) part[n][0][x] = part[n][1][x] = 0.f;
                const uint32_t k_row = buf + (hk * 16u + gr) * 128u;
#pragma unroll
                for (uint32_t c = 0; c < SLABS * 2u; ++c) {   // 16-byte column groups of this thread
                    const uint32_t col = ((2u * t + (c & 1u)) ^ gr) * 16u;
                    const uint4 a = lds128(k_row + (c >> 1) * slab_bytes + col), b = lds128(k_row + (c >> 1) * slab_bytes + col + 8u * 128u);
                    const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                    for (uint32_t x = 0; x < 4; x += 2) {
                        uint32_t f0[4], f1[4];
                        brc::kv8_decode4<CODE>(wa[x], f0[0], f0[2]);
                        brc::kv8_decode4<CODE>(wb[x], f0[1], f0[3]);
                        brc::kv8_decode4<CODE>(wa[x + 1], f1[0], f1[2]);
                        brc::kv8_decode4<CODE>(wb[x + 1], f1[1], f1[3]);
                        const uint32_t at = (c * 2u + x / 2u) * 512u;
#pragma unroll
                        for (int n = 0; n < RT; ++n) {
                            const uint4 qf = lds128(q_frag + n * 8u * HD * 2u + at);
                            brc::mma_16816(part[n][0], f0, qf.x, qf.y);
                            brc::mma_16816(part[n][1], f1, qf.z, qf.w);
                            if (PREC) {
                                const uint4 ql = lds128(q_frag_lo + n * 8u * HD * 2u + at);
                                brc::mma_16816(part[n][0], f0, ql.x, ql.y);
                                brc::mma_16816(part[n][1], f1, ql.z, ql.w);
                            }
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < RT; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[n][x] = part[n][0][x] + part[n][1][x];
            }

            // ---- softmax over the running maxima; weights to B fragments [cells][rows]
            const bool good = ks > 0.f;
            const float ev = (float)brc::kv8_scale_exponent(vs);
            uint32_t pw[RT][2], pw_lo[RT][2];
#pragma unroll
            for (int n = 0; n < RT; ++n) {
                float f[2], wt[4];
#pragma unroll
                for (int x = 0; x < 2; ++x) {   // the thread's two rows: cells gr and gr + 8
                    const float kf = fac[n][x] * ks;
                    const bool see0 = good && cell0 + gr < vis[n][x], see1 = good && cell0 + gr + 8u < vis[n][x];
                    const float s0 = see0 ? s[n][x] * kf : -INFINITY, s1 = see1 ? s[n][x + 2] * kf : -INFINITY;
                    float top = fmaxf(s0, s1);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float m_new = fmaxf(m_run[n][x], top), w_new = fmaxf(w_run[n][x], top + ev);
                    l_run[n][x] = l_run[n][x] * brc::fast_exp2(m_run[n][x] - m_new) + (brc::fast_exp2(s0 - m_new) + brc::fast_exp2(s1 - m_new));
                    f[x] = brc::fast_exp2(w_run[n][x] - w_new);
                    const float shift = ev - w_new + 15.f;
                    wt[x] = brc::fast_exp2(s0 + shift);
                    wt[x + 2] = brc::fast_exp2(s1 + shift);
                    m_run[n][x] = m_new;
                    w_run[n][x] = w_new;
                }
                if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
                    for (int j = 0; j < (int)SLABS * 8; ++j) {
                        o[n][j][0] *= f[0];
                        o[n][j][1] *= f[1];
                        o[n][j][2] *= f[0];
                        o[n][j][3] *= f[1];
                    }
                }
                const uint32_t a = brc::pack_half2(wt[0], wt[1]), b = brc::pack_half2(wt[2], wt[3]);
                pw[n][0] = brc::movmatrix_trans(a);
                pw[n][1] = brc::movmatrix_trans(b);
                if (PREC) {
                    const float2 ha = __half22float2(*reinterpret_cast<const __half2 *>(&a)), hb = __half22float2(*reinterpret_cast<const __half2 *>(&b));
                    pw_lo[n][0] = brc::movmatrix_trans(brc::pack_half2(wt[0] - ha.x, wt[1] - ha.y));
                    pw_lo[n][1] = brc::movmatrix_trans(brc::pack_half2(wt[2] - hb.x, wt[3] - hb.y));
                }
            }

            // ---- O^T[head_dim][8 rows] += V^T P.  Output row gr of tile j is column 16 gr + j, row gr + 8 column 16 gr + 8 + j.
            const bool tail = cell0 + 16u > len || !good;   // cells nobody sees may hold anything, NaN codes too: 0 x NaN
#pragma unroll
            for (uint32_t sl = 0; sl < SLABS; ++sl) {
                uint32_t w[4][4];
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) {
                    const uint32_t c = 2u * t + (x & 1u) + 8u * (x >> 1);
                    const uint4 v = lds128(buf + sl * slab_bytes + ((p.kvb + hk) * 16u + c) * 128u + ((gr ^ (c & 7u)) * 16u));
                    w[x][0] = v.x;
                    w[x][1] = v.y;
                    w[x][2] = v.z;
                    w[x][3] = v.w;
                    if (tail && (!good || cell0 + c >= len)) w[x][0] = w[x][1] = w[x][2] = w[x][3] = 0u;
                }
#pragma unroll
                for (uint32_t y = 0; y < 2; ++y) {   // columns 4 y .. 4 y + 3 and those + 8
                    uint32_t fa[4][4];               // [column][a0 a1 a2 a3]
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {        // columns + 8 h
#pragma unroll
                        for (uint32_t x = 0; x < 2; ++x) {    // cells 2t, 2t+1, then those + 8
                            const uint32_t u = w[2 * x][y + 2 * h], v = w[2 * x + 1][y + 2 * h];
                            uint32_t e0, e1, e2, e3;
                            brc::kv8_decode4<CODE>(__byte_perm(u, v, 0x5140), e0, e1);
                            brc::kv8_decode4<CODE>(__byte_perm(u, v, 0x7362), e2, e3);
                            fa[0][h + 2 * x] = e0;
                            fa[1][h + 2 * x] = e1;
                            fa[2][h + 2 * x] = e2;
                            fa[3][h + 2 * x] = e3;
                        }
                    }
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
#pragma unroll
                        for (int n = 0; n < RT; ++n) {
                            brc::mma_16816(o[n][sl * 8u + 4u * y + j], fa[j], pw[n][0], pw[n][1]);
                            if (PREC) brc::mma_16816(o[n][sl * 8u + 4u * y + j], fa[j], pw_lo[n][0], pw_lo[n][1]);
                        }
                }
            }
            __syncwarp();
            if (lane == 0) brc::mbar_arrive(empty0 + 8u * stage);
        }
        done += g.n;

        // ---- merge the warps that took this unit's pages in turn; finish it, or leave a partial
#pragma unroll
        for (int n = 0; n < RT; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float l = l_run[n][x];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (gr == 0) stat[warp * 16u + n * 8u + 2u * t + x] = make_float4(m_run[n][x], w_run[n][x], l, 0.f);
            }
        const bool whole = g.n == g.pages;
        const uint64_t slot = 2ull * blockIdx.x + (g.pg == 0 ? 1u : 0u);
#pragma unroll
        for (int n = 0; n < RT; ++n) {
#pragma unroll
            for (uint32_t sl = 0; sl < SLABS; ++sl) {
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t x = 0; x < 2; ++x)
#pragma unroll
                        for (uint32_t y = 0; y < 2; ++y) {
                            const float(*a)[4] = &o[n][sl * 8u + 4u * y];
                            *reinterpret_cast<float4 *>(scratch + (warp * 8u + 2u * t + x) * SCRATCH_ROW + 16u * gr + 8u * h + 4u * y) =
                                make_float4(a[0][2 * h + x], a[1][2 * h + x], a[2][2 * h + x], a[3][2 * h + x]);
                        }
                brc::named_bar_sync(1, CONSUMERS);
                const uint32_t items = p.kvb * p.row_groups * 8u * 32u;
                for (uint32_t it = tid; it < items; it += CONSUMERS) {
                    const uint32_t c4 = it % 32u, row8 = it / 32u % 8u, wg = it / 256u;   // wg = head + kvb * row group
                    const uint32_t r = ((wg / p.kvb) * RT + n) * 8u + row8, h = wg % p.kvb;
                    const uint32_t gr_row = pass * p.pass_rows + r;
                    if (gr_row >= rows) continue;
                    float m = NONE, wm = NONE;
                    for (uint32_t q = 0; q < lanes; ++q) {
                        const float4 st = stat[(wg + q * p.kvb * p.row_groups) * 16u + n * 8u + row8];
                        m = fmaxf(m, st.x);
                        wm = fmaxf(wm, st.y);
                    }
                    float l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
                    for (uint32_t q = 0; q < lanes; ++q) {
                        const uint32_t w = wg + q * p.kvb * p.row_groups;
                        const float4 st = stat[w * 16u + n * 8u + row8];
                        l += st.z * brc::fast_exp2(st.x - m);
                        const float f = brc::fast_exp2(st.y - wm);
                        const float4 x = lds128f(base + L.scratch + ((w * 8u + row8) * SCRATCH_ROW + c4 * 4u) * 4u);
                        v[0] += x.x * f;
                        v[1] += x.y * f;
                        v[2] += x.z * f;
                        v[3] += x.w * f;
                    }
                    const uint32_t d = sl * 128u + c4 * 4u;
                    if (whole) {
                        const float f = l == 0.f ? 0.f : brc::fast_exp2(wm - m - 15.f) / l;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] *= f;
                        const uint32_t tok = gr_row / p.group, head = (hg * p.kvb + h) * p.group + gr_row % p.group;
                        finish_row(p, HD, (tok0 + tok) * p.n_head + head, d, v);
                    } else {
                        const uint64_t at = slot * p.kvb * p.pass_rows + h * p.pass_rows + r;
                        *reinterpret_cast<float4 *>(p.acc + at * HD + d) = make_float4(v[0], v[1], v[2], v[3]);
                        if (d == 0) *reinterpret_cast<float4 *>(p.ml + at * 4u) = make_float4(m, wm, l, 0.f);
                    }
                }
                brc::named_bar_sync(1, CONSUMERS);
            }
        }
    }
    if (!ok && lane == 0) { atomicOr(p.status, BRC_DEV_WAIT_LIMIT); p.status[1] = blockIdx.x; }
}

// One CTA per (unit, query row): the partials that the shares' boundaries left of it, in share order; zeros for a sequence
// without cells.  Units that one share covered are finished already.
template <int HD>
__global__ void __launch_bounds__(256) kv8_merge_kernel(const AttnParams p, uint32_t grid) {
    constexpr uint32_t PER = HD / 32;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float part[8][HD];
    const uint32_t s = blockIdx.x / p.units_per_seq, u = blockIdx.x % p.units_per_seq;
    const uint64_t before = p.prefix[s], pages = p.prefix[s + 1] - before;
    const uint64_t share = share_of(p.prefix[p.n_seqs] * p.units_per_seq, grid);
    const uint64_t begin = before * p.units_per_seq + u * pages;
    const uint64_t c0 = begin / share, c1 = pages ? (begin + pages - 1u) / share : c0;
    if (pages && c0 == c1) return;
    const uint32_t hg = u / p.passes, pass = u % p.passes;
    const uint32_t h = blockIdx.y / p.pass_rows, r = blockIdx.y % p.pass_rows, gr_row = pass * p.pass_rows + r;
    const uint32_t n_q = min(tokens_of(p, s), p.max_q);
    if (gr_row >= n_q * p.group) return;
    const uint64_t tok0 = p.cu_q ? p.cu_q[s] : (uint64_t)s * p.max_q;
    const uint64_t head_row = (tok0 + gr_row / p.group) * p.n_head + (hg * p.kvb + h) * p.group + gr_row % p.group;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t n = pages ? (uint32_t)(c1 - c0 + 1u) : 0u;
    auto at = [&](uint32_t i) { return ((2ull * (c0 + i) + (i == 0 ? 1u : 0u)) * p.kvb + h) * p.pass_rows + r; };

    float m = NONE, wm = NONE, l = 0.f;
    for (uint32_t i = lane; i < n; i += 32u) {
        const float4 st = *reinterpret_cast<const float4 *>(p.ml + at(i) * 4u);
        const float m_new = fmaxf(m, st.x);
        l = l * brc::fast_exp2(m - m_new) + st.z * brc::fast_exp2(st.x - m_new);
        m = m_new;
        wm = fmaxf(wm, st.y);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
        const float m_new = fmaxf(m, m2);
        l = l * brc::fast_exp2(m - m_new) + l2 * brc::fast_exp2(m2 - m_new);
        m = m_new;
        wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
    }
    float v[PER];
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) v[j] = 0.f;
#pragma unroll 4
    for (uint32_t i = warp; i < n; i += 8u) {
        const float f = brc::fast_exp2(p.ml[at(i) * 4u + 1u] - wm);
        const float *a = p.acc + at(i) * HD + lane * 4u;
#pragma unroll
        for (uint32_t j = 0; j < PER; j += 4) {
            const float4 x = *reinterpret_cast<const float4 *>(a + 32u * j);
            v[j] += x.x * f;
            v[j + 1] += x.y * f;
            v[j + 2] += x.z * f;
            v[j + 3] += x.w * f;
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < PER; j += 4) *reinterpret_cast<float4 *>(&part[warp][lane * 4u + 32u * j]) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    __syncthreads();
    const uint32_t d = threadIdx.x * 4u;
    if (d >= HD) return;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t w = 0; w < 8; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += part[w][d + e];
    const float f = l == 0.f ? 0.f : brc::fast_exp2(wm - m - 15.f) / l;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] *= f;
    finish_row(p, HD, head_row, d, x);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
struct Shape {
    uint32_t group, kvb, rt, row_groups, pass_rows, passes, units_per_seq;
    uint64_t prefix_bytes, ml_bytes, acc_bytes;
    uint64_t workspace() const { return prefix_bytes + ml_bytes + acc_bytes; }
};

Shape shape_of(const brc_pool *pool, uint32_t n_seqs, uint32_t n_head, uint32_t max_q) {
    Shape s;
    s.group = n_head / pool->n_kv_head;
    s.kvb = brc_kv8_kvb(pool);
    const uint64_t rows = (uint64_t)s.group * max_q;
    // Eight rows: one tile a warp, half the registers, and the least work on padding; nine to sixteen: two; more: two warps
    // side by side on the same pages, up to PASS_ROWS a pass.
    s.rt = rows <= 8u ? 1u : 2u;
    s.row_groups = rows <= 16u ? 1u : 2u;
    s.pass_rows = std::min(s.rt * s.row_groups * 8u, PASS_ROWS);
    s.passes = (uint32_t)((rows + s.pass_rows - 1u) / s.pass_rows);
    s.units_per_seq = pool->n_kv_head / s.kvb * s.passes;
    const uint64_t slots = 2ull * (uint64_t)pool->sm_count * s.kvb * s.pass_rows;
    s.prefix_bytes = (((uint64_t)n_seqs + 1u) * 8u + 255u) / 256u * 256u;
    s.ml_bytes = slots * 16u;
    s.acc_bytes = slots * pool->head_dim * 4u;
    return s;
}

template <int HD, uint32_t CODE, bool PREC, int RT>
brc_status launch(const brc_pool *pool, AttnParams p, uint32_t grid, uint32_t merge_rows, cudaStream_t st) {
    auto kern = kv8_attn_kernel<HD, CODE, PREC, RT>;
    const uint32_t turns = WARPS / (p.kvb * p.row_groups);
    // Ring depth: what fits, in multiples of the warps that take pages in turn, so that a stage is always consumed by the same
    // warps (a parity wait is only valid for a warp that knows the previous round of the barrier is over).
    const Smem none = smem_layout(HD, p.kvb, p.pass_rows, PREC, 0);
    p.n_stages = std::min((SMEM_LIMIT - none.total) / none.stage_bytes, MAX_STAGES) / turns * turns;
    const uint32_t smem = smem_layout(HD, p.kvb, p.pass_rows, PREC, p.n_stages).total;
    static std::atomic<uint64_t> ready{0};   // devices on which this kernel may use all shared memory
    const uint64_t bit = 1ull << (pool->device & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit) || pool->device > 63) {
        BRC_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_LIMIT));
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    kern<<<grid, THREADS, smem, st>>>(pool->tm_kv8, p);
    BRC_CUDA(cudaGetLastError());
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.n_seqs * p.units_per_seq, merge_rows);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    BRC_CUDA(cudaLaunchKernelEx(&cfg, kv8_merge_kernel<HD>, p, grid));
    return BRC_OK;
}

template <int HD, uint32_t CODE>
brc_status launch_rows(const brc_pool *pool, const AttnParams &p, uint32_t grid, bool prec, uint32_t rt, uint32_t merge_rows, cudaStream_t st) {
    if (prec) return rt == 1 ? launch<HD, CODE, true, 1>(pool, p, grid, merge_rows, st) : launch<HD, CODE, true, 2>(pool, p, grid, merge_rows, st);
    return rt == 1 ? launch<HD, CODE, false, 1>(pool, p, grid, merge_rows, st) : launch<HD, CODE, false, 2>(pool, p, grid, merge_rows, st);
}

bool known_dtype(int32_t d) { return d == BRC_DTYPE_F32 || d == BRC_DTYPE_F16 || d == BRC_DTYPE_BF16; }

}  // namespace

brc_status brc_kv8_workspace(const brc_pool *pool, uint32_t n_seqs, uint32_t n_head, uint32_t max_q, uint64_t *out_bytes) {
    *out_bytes = 0;
    if (n_head == 0 || n_head % pool->n_kv_head != 0)
        return brc_fail(BRC_ERR_INVALID, "8-bit attention: %u query heads do not divide over %u kv heads", n_head, pool->n_kv_head);
    *out_bytes = shape_of(pool, n_seqs, n_head, std::max(max_q, 1u)).workspace();
    return BRC_OK;
}

brc_status brc_kv8_attend(brc_pool *pool, const char *who, const brc_kv8_attn_args &a, void *stream) {
    if (!pool) return brc_fail(BRC_ERR_INVALID, "%s: pool is NULL", who);
    if (pool->device < 0 || !pool->k_base)
        return brc_fail(BRC_ERR_CUDA, "%s: this pool holds bookkeeping only (no device memory); compute calls need a GPU pool", who);
    if (!pool->kv8) return brc_fail(BRC_ERR_UNSUPPORTED, "%s: the pool's pages are not 8-bit (brc_pool_create_kv8)", who);
    if (a.layer >= pool->n_layers) return brc_fail(BRC_ERR_INVALID, "%s: layer %u but the pool has %u", who, a.layer, pool->n_layers);
    if (!known_dtype(a.q_dtype) || !known_dtype(a.out_dtype))
        return brc_fail(BRC_ERR_INVALID, "%s: q_dtype %d / out_dtype %d: f32 (0), f16 (1) or bf16 (2)", who, a.q_dtype, a.out_dtype);
    if (a.n_head == 0 || a.n_head % pool->n_kv_head != 0)
        return brc_fail(BRC_ERR_INVALID, "%s: %u query heads do not divide over %u kv heads", who, a.n_head, pool->n_kv_head);
    const uint64_t capacity = (uint64_t)a.table_stride * pool->page_tokens;
    if (a.max_seq_len > capacity)
        return brc_fail(BRC_ERR_CAPACITY, "%s would read cells up to %u but each block table holds %llu (%u pages of %u cells)", who,
                        a.max_seq_len, (unsigned long long)capacity, a.table_stride, pool->page_tokens);
    if (a.gate && a.gate_head_stride < pool->head_dim)
        return brc_fail(BRC_ERR_INVALID, "%s: gate_head_stride %u < head_dim %u", who, a.gate_head_stride, pool->head_dim);
    if (a.n_seqs == 0 || a.max_q == 0) return BRC_OK;
    if (!a.q || !a.block_tables || !a.seq_lens || !a.out)
        return brc_fail(BRC_ERR_INVALID, "%s: NULL query, block table, length or output pointer", who);
    if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.workspace)) & 15u)
        return brc_fail(BRC_ERR_INVALID, "%s: query, output and workspace pointers must be 16-byte aligned", who);
    const Shape s = shape_of(pool, a.n_seqs, a.n_head, a.max_q);
    if ((uint64_t)a.max_q * s.group >= (1ull << 31) || (uint64_t)a.n_seqs * s.units_per_seq >= (1ull << 31))
        return brc_fail(BRC_ERR_UNSUPPORTED, "%s: %u sequences of %u tokens with %u heads per kv head in one call", who, a.n_seqs, a.max_q, s.group);
    if (!a.workspace || a.workspace_bytes < s.workspace())
        return brc_fail(BRC_ERR_INVALID, "%s: workspace of %llu bytes, %llu needed", who, (unsigned long long)a.workspace_bytes,
                        (unsigned long long)s.workspace());
    brc_device_guard guard(pool->device);
    if (!guard.ok) return brc_fail(BRC_ERR_CUDA, "%s: cannot make device %d current", who, pool->device);
    AttnParams p = {};
    p.q = a.q;
    p.out = a.out;
    p.gate = a.gate;
    p.block_tables = a.block_tables;
    p.seq_lens = a.seq_lens;
    p.cu_q = a.cu_q;
    p.k_layer = pool->k_base + (uint64_t)a.layer * pool->layer_bytes;
    p.v_layer = pool->v_base + (uint64_t)a.layer * pool->v_layer_bytes;
    uint8_t *ws = static_cast<uint8_t *>(a.workspace);
    p.prefix = reinterpret_cast<uint64_t *>(ws);
    p.ml = reinterpret_cast<float *>(ws + s.prefix_bytes);
    p.acc = reinterpret_cast<float *>(ws + s.prefix_bytes + s.ml_bytes);
    p.status = pool->status_dev;
    p.page_bytes = pool->half_page_bytes;
    p.q_dtype = (uint32_t)a.q_dtype;
    p.out_dtype = (uint32_t)a.out_dtype;
    p.gate_head_stride = a.gate_head_stride;
    p.table_stride = a.table_stride;
    p.n_seqs = a.n_seqs;
    p.max_seq_len = a.max_seq_len;
    p.max_q = a.max_q;
    p.n_pages = pool->n_pages;
    p.page0 = a.layer * pool->n_pages;
    p.n_head = a.n_head;
    p.n_kv = pool->n_kv_head;
    p.group = s.group;
    p.kvb = s.kvb;
    p.row_groups = s.row_groups;
    p.pass_rows = s.pass_rows;
    p.passes = s.passes;
    p.units_per_seq = s.units_per_seq;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    const uint64_t most = (uint64_t)a.n_seqs * s.units_per_seq * ((a.max_seq_len + 15ull) / 16u);   // page-units at most
    const uint32_t grid = (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>(pool->sm_count, (most + MIN_SHARE - 1u) / MIN_SHARE));
    const bool prec = a.q_dtype == BRC_DTYPE_F32 || a.out_dtype == BRC_DTYPE_F32;
    const uint32_t merge_rows = s.kvb * s.pass_rows;
    cudaStream_t st = brc_stream(stream);
    brc_stage_begin(pool, BRC_STAGE_ATTN_PARTIAL, st);
    brc_status rc;
    if (pool->head_dim == 256)
        rc = pool->kv8 == brc::KV8_E4M3 ? launch_rows<256, brc::KV8_E4M3>(pool, p, grid, prec, s.rt, merge_rows, st)
                                        : launch_rows<256, brc::KV8_INT8>(pool, p, grid, prec, s.rt, merge_rows, st);
    else
        rc = pool->kv8 == brc::KV8_E4M3 ? launch_rows<128, brc::KV8_E4M3>(pool, p, grid, prec, s.rt, merge_rows, st)
                                        : launch_rows<128, brc::KV8_INT8>(pool, p, grid, prec, s.rt, merge_rows, st);
    brc_stage_end(pool, BRC_STAGE_ATTN_PARTIAL, st);
    return rc;
}

extern "C" {

brc_status brc_kv8_attn_workspace_bytes(const brc_pool *pool, uint32_t n_seqs, uint32_t n_head, uint32_t max_q, uint64_t *out_bytes) {
    if (!pool || !out_bytes) return brc_fail(BRC_ERR_INVALID, "brc_kv8_attn_workspace_bytes: NULL argument");
    if (!pool->kv8) return brc_fail(BRC_ERR_UNSUPPORTED, "brc_kv8_attn_workspace_bytes: the pool's pages are not 8-bit (brc_pool_create_kv8)");
    return brc_kv8_workspace(pool, n_seqs, n_head, max_q, out_bytes);
}

brc_status brc_kv8_attn(brc_pool *pool, uint32_t layer, const void *q_dev, int32_t q_dtype, uint32_t n_head, const float *gate_dev,
                        uint32_t gate_head_stride, const uint32_t *block_tables_dev, uint32_t table_stride,
                        const uint32_t *seq_lens_dev, const uint32_t *cu_q_dev, uint32_t n_seqs, uint32_t max_q, uint32_t max_seq_len,
                        float scale, void *out_dev, int32_t out_dtype, void *workspace_dev, uint64_t workspace_bytes, void *stream) {
    brc_kv8_attn_args a;
    a.layer = layer;
    a.q = q_dev;
    a.q_dtype = q_dtype;
    a.n_head = n_head;
    a.gate = gate_dev;
    a.gate_head_stride = gate_head_stride;
    a.block_tables = block_tables_dev;
    a.table_stride = table_stride;
    a.seq_lens = seq_lens_dev;
    a.cu_q = cu_q_dev;
    a.n_seqs = n_seqs;
    a.max_q = max_q;
    a.max_seq_len = max_seq_len;
    a.scale = scale;
    a.out = out_dev;
    a.out_dtype = out_dtype;
    a.workspace = workspace_dev;
    a.workspace_bytes = workspace_bytes;
    return brc_kv8_attend(pool, "brc_kv8_attn", a, stream);
}

}  // extern "C"
