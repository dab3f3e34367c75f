// Attention over 8-bit pages (value = code * 2^e, one exponent per page, kv head and side; brc_pool_create_kv8), for one
// or several tokens per sequence.
//
//   out[i,h] = sigmoid(gate) * sum_c softmax_c(scale * q.k_c) v_c,   c < len - (T - 1 - i)
//
// What bounds it: one token of 8 heads per kv head does 16 FLOP per cached byte, far under the 260 a B200's tensor cores
// have per byte of HBM, so the cache stream is the floor - if converting it keeps up: 24 bytes per SM and clock have to
// become binary16 operands.  Hence:
//   - the codes go to the tensor cores as the exact binary16 numbers they are (cvt of e4m3 pairs; byte permute and one
//     subtraction for int8), never scaled: K's scale multiplies the finished dot product, V's joins the exponent of
//     the probability, so scales cost one multiply per 16 cells and row instead of one per value;
//   - mma.sync m16n8k16 with the CACHE as the 16-row operand and the query rows as the 8-column one.  tcgen05 would pad 8
//     rows to 64 or 128 and want the converted operand written back to shared memory, twice the bytes the codes
//     themselves cost; the warp-level form takes it from the registers the conversion leaves it in.  Its rate is
//     not the limit: 48 of them per page and head of 256 (16 for the scores, 32 for the weights' two parts) against 350
//     clocks of HBM time; the pipe is busy 21 to 29 % of the time;
//   - fragments are cut so that a thread's sixteen consecutive bytes are one 16-byte shared-memory read: the sum over
//     head_dim may run in any order, so K's columns are dealt out 16 bytes to a thread, and V's columns likewise become
//     the output rows; the 128-byte swizzle of the TMA box keeps every such read free of bank conflicts;
//   - all (sequence, kv-head group, pass) units form one list of page-units cut into equal shares, one persistent CTA per
//     SM; one warp streams the pages with TMA into a ring, eight or twelve consume.  A unit cut by a share boundary leaves partial
//     results in the caller's workspace, and a second kernel, launched with its prologue overlapped (programmatic
//     dependent launch), merges them.  No counters and no flags: nothing survives a call, so calls with workspaces of
//     their own may overlap.
//
// Two reference exponents per row, near the running maxima: m of the scores s (for the sum of probabilities), and M of
// s + e_v, the exponent at which a cell's V codes enter the result, kept as M - m (a difference of two large scores is exact,
// what is added to one is lost).  Weights are 2^(s + e_v - M + 7), below 2^15 even when a
// score lies 2^8 over its reference, so binary16 keeps cells down to 2^-31 of the heaviest one, and a page whose V scale
// dwarfs the others' neither overflows nor silences them.  A weight goes to the tensor cores as two binary16 parts, 22 of its 24 bits,
// whatever the types of q and out: one part's 2^-12 shows in a 16-bit result wherever values cancel.
#include <algorithm>
#include <atomic>

#include "brc_internal.h"
#include "kv8.cuh"

namespace {

constexpr uint32_t PASS_ROWS = 32;       // query rows (tokens x heads of a kv head) that share one stream of the cache
constexpr uint32_t MIN_SHARE = 4;        // page-units a CTA takes at least
constexpr uint32_t SMEM_LIMIT = 232448;  // 227 KiB
constexpr uint32_t MAX_STAGES = 48;
constexpr float HEADROOM = 8.f, WEIGHT_SHIFT = 7.f;   // a weight is at most 2^(WEIGHT_SHIFT + HEADROOM), half of binary16's greatest
constexpr float NONE = -3e38f;           // running maximum before any cell

struct AttnParams {
    const void *q;
    void *out;
    const float *gate;
    const uint32_t *block_tables, *seq_lens, *cu_q;
    const uint8_t *k_layer, *v_layer;
    uint32_t *prefix;        // workspace: cost of the sequences before each
    float *ml;               // [slot][row of a unit][m, M - m, l, -]
    float *acc;              // [slot][row of a unit][head_dim]
    uint32_t *status;
    uint64_t page_bytes;
    uint32_t q_dtype, out_dtype, gate_head_stride;
    uint32_t table_stride, n_seqs, max_seq_len, max_q, n_pages, page0;   // page0: layer * n_pages
    uint32_t total_q;        // rows of q and out behind which cu_q must not lead
    uint32_t n_head, n_kv, group, kvb, row_groups;                        // row_groups: warps that split a pass's rows
    uint32_t pass_rows, head_groups, units_per_seq, n_stages, q_bufs, unit_cost;   // units_per_seq: the longest q's
    float scale_log2;
};

struct Smem {   // byte offsets behind the ring
    uint32_t stage_bytes, q, q_lo, q_bytes, scratch, stat, row_fac, row_vis, bars, sched, total;
};

__host__ __device__ inline Smem smem_layout(uint32_t hd, uint32_t warps, uint32_t kvb, uint32_t pass_rows, bool split_q, uint32_t n_stages,
                                            uint32_t q_bufs) {
    Smem s;
    s.stage_bytes = kvb * 2u * 16u * hd;
    uint32_t at = n_stages * s.stage_bytes;
    s.q = at;
    s.q_bytes = kvb * pass_rows * hd * 2u;
    at += q_bufs * s.q_bytes;
    s.q_lo = at;
    if (split_q) at += q_bufs * s.q_bytes;
    s.scratch = at;                       // [warp][row of a tile][head_dim + one 16-byte group]
    at += warps * 8u * (hd + 4u) * 4u;
    s.stat = at;                          // [warp][row of two tiles][m, M - m, l, -]
    at += warps * 16u * 16u;
    s.row_fac = at;                       // [buffer][head][row]
    at += q_bufs * kvb * pass_rows * 4u;
    s.row_vis = at;                       // [buffer][row]
    at += q_bufs * pass_rows * 4u;
    s.bars = at;                          // full, empty (ring); full, empty (q)
    at += 2u * MAX_STAGES * 8u + 32u;
    s.sched = at;
    at += warps * 4u + 64u;
    s.total = at;
    return s;
}

// T of a sequence (none where its prefix goes backwards), and how many of its tokens the call has rows for.
__device__ __forceinline__ uint32_t tokens_of(const AttnParams &p, uint32_t s) {
    if (!p.cu_q) return p.max_q;
    const uint32_t b = p.cu_q[s], e = p.cu_q[s + 1];
    return e > b ? e - b : 0u;
}
__device__ __forceinline__ uint32_t rows_of(const AttnParams &p, uint32_t s) {
    const uint32_t t = min(tokens_of(p, s), p.max_q);
    return p.cu_q ? min(t, p.total_q - min(p.cu_q[s], p.total_q)) : t;
}
__device__ __forceinline__ uint32_t cells_of(const AttnParams &p, uint32_t s) { return min(p.seq_lens[s], p.max_seq_len); }
__device__ __forceinline__ uint32_t pages_of(const AttnParams &p, uint32_t s) {
    return rows_of(p, s) ? (cells_of(p, s) + 15u) / 16u : 0u;
}
// Passes that a sequence's own rows fill (at least one), and its units: kv-head groups x passes.  MANY: the call's longest sequence fills
// more than one; known at compile time, since the divisions by it would add 0.3 to 1 us in front of the first page of every other call.
template <bool MANY>
__device__ __forceinline__ uint32_t passes_of(const AttnParams &p, uint32_t s) {
    return MANY ? max((rows_of(p, s) * p.group + PASS_ROWS - 1u) / PASS_ROWS, 1u) : 1u;
}
template <bool MANY>
__device__ __forceinline__ uint32_t units_of(const AttnParams &p, uint32_t s) { return p.head_groups * passes_of<MANY>(p, s); }
// What a unit counts for when the work is cut: its pages and, in front of them, what starting and finishing a unit costs.
// (The host refuses a call whose costs could add up to 2^31.)
template <bool MANY>
__device__ __forceinline__ uint32_t cost_of(const AttnParams &p, uint32_t s) {
    const uint32_t pages = pages_of(p, s);
    return pages ? (pages + p.unit_cost) * units_of<MANY>(p, s) : 0u;
}
__device__ __forceinline__ uint32_t share_of(uint32_t total, uint32_t grid) { return max((total + grid - 1u) / grid, MIN_SHARE); }

__device__ __forceinline__ void store_out(const AttnParams &p, uint64_t at, float a, float b, float c, float d) {
    if (p.out_dtype == 0) {
        *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + at) = make_float4(a, b, c, d);
    } else if (p.out_dtype == 1) {
        *reinterpret_cast<uint2 *>(static_cast<__half *>(p.out) + at) = make_uint2(brc::pack2<1>(a, b), brc::pack2<1>(c, d));
    } else {
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(p.out) + at) = make_uint2(brc::pack2<2>(a, b), brc::pack2<2>(c, d));
    }
}

// As in the binary16 decode attention.  (With __expf the result would be off by 2^-18 of itself at -80, and zero below -89.)
__device__ __forceinline__ float sigmoid_f32(float x) {
    if (x >= 0.f) return 1.f / (1.f + expf(-x));
    const float e = expf(x);
    return e / (1.f + e);
}

// Four values of one output row, gated and stored.  `head_row`: token * n_head + head.
__device__ __forceinline__ void finish_row(const AttnParams &p, uint32_t hd, uint64_t head_row, uint32_t d, float (&v)[4]) {
    if (p.gate) {
        const float *g = p.gate + head_row * p.gate_head_stride + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= sigmoid_f32(g[i]);
    }
    store_out(p, head_row * hd + d, v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ uint4 lds128(const uint8_t *smem, uint32_t at) { return *reinterpret_cast<const uint4 *>(smem + at); }

// D(16x8, f32) += A(16x16, f16, row) * B(16x8, f16, col).  Not volatile: the compiler may interleave it with the conversions.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Keeps a rare case a branch: selects in its place would be paid by every page (40 of them at 256 columns).
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// One load of q rows in any of the three types: eight consecutive values of head row `r` from column d.
template <int DT>
__device__ __forceinline__ void load_q8_as(const AttnParams &p, uint64_t at, float (&v)[8]) {
    brc::raw8<DT> r;
    r.load(static_cast<const typename brc::elem<DT>::t *>(p.q) + at, true);
    r.values(v);
}
__device__ __forceinline__ void load_q8(const AttnParams &p, uint64_t at, float (&v)[8]) {
    if (p.q_dtype == 0) load_q8_as<0>(p, at, v);
    else if (p.q_dtype == 1) load_q8_as<1>(p, at, v);
    else load_q8_as<2>(p, at, v);
}

// A share's walk over the units: [lo, hi) on the axis of costs, and where the unit in hand begins on it.
struct Cursor {
    uint32_t at, lo, hi, s, hg, pass;
};

struct Segment {   // pages [pg, pg + n) of one unit: kv-head group hg of sequence s, pass `pass` of its rows
    uint32_t s, hg, pass, pg, n, pages;
};

struct Start {   // of a share: its first segment (n = 0: none) and where to go on
    Cursor cur;
    Segment seg;
};

template <bool MANY>
__device__ __forceinline__ bool next_segment(const AttnParams &p, Cursor &c, Segment &g) {
    while (c.at < c.hi) {
        const uint32_t pages = pages_of(p, c.s);
        if (pages == 0 || c.hg == p.head_groups) {
            ++c.s;
            c.hg = 0;
            continue;
        }
        const uint32_t first = c.at + p.unit_cost;   // page 0's place on the axis
        const uint32_t from = min(c.lo > first ? c.lo - first : 0u, pages), to = min(c.hi > first ? c.hi - first : 0u, pages);
        g.s = c.s;
        g.hg = c.hg;
        g.pass = MANY ? c.pass : 0u;
        g.pages = pages;
        g.pg = from;
        g.n = to > from ? to - from : 0u;
        c.at = first + pages;
        if (!MANY || ++c.pass == passes_of<MANY>(p, g.s)) {
            c.pass = 0;
            ++c.hg;
        }
        if (g.n) return true;   // a share may end inside a unit's cost, in front of its first page
    }
    return false;
}

// q rows of a unit, scaled by a power of two to at most 2^15 in magnitude and laid out as the B fragments of the K product:
// [8-row tile][pair of 16-column steps][lane][2 x 4 values]; column d belongs to step 8 (d / 128) + 4 (d / 16 % 2) +
// d / 4 % 4 and thread d / 32 % 4 of its row's group.  A row takes HD / 8 lanes; warp `w` of `n_w` has every n_w-th set of
// 256 / HD rows, U sets of loads in flight; `meanwhile` runs behind the first loads.
template <int HD, bool SPLIT_Q, int U, class F>
__device__ __forceinline__ void stage_q(const AttnParams &p, const Smem &L, uint8_t *smem, const Segment &g, uint32_t buf, uint32_t w,
                                        uint32_t n_w, uint32_t lane, F &&meanwhile) {
    constexpr uint32_t LANES = HD / 8, SET = 32 / LANES;
    const uint32_t hg = g.hg, pass = g.pass;
    const uint32_t n_q = tokens_of(p, g.s), len = cells_of(p, g.s);
    const uint64_t tok0 = p.cu_q ? p.cu_q[g.s] : (uint64_t)g.s * p.max_q;
    const uint32_t rows = rows_of(p, g.s) * p.group, all = p.kvb * p.pass_rows, d = lane % LANES * 8u;
    float *row_fac = reinterpret_cast<float *>(smem + L.row_fac) + buf * all;
    uint32_t *row_vis = reinterpret_cast<uint32_t *>(smem + L.row_vis) + buf * p.pass_rows;
    for (uint32_t r0 = w * SET + lane / LANES; r0 / SET * SET < all; r0 += n_w * SET * U) {   // (all is a multiple of SET: whole warps)
        float v[U][8];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const uint32_t rr = r0 + k * n_w * SET, h = rr / p.pass_rows, gr_row = pass * p.pass_rows + rr % p.pass_rows;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = 0.f;
            if (rr < all && gr_row < rows)
                load_q8(p, ((tok0 + gr_row / p.group) * p.n_head + (hg * p.kvb + h) * p.group + gr_row % p.group) * HD + d, v[k]);
        }
        if (r0 < n_w * SET) meanwhile();
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const uint32_t rr = r0 + k * n_w * SET;
            if (rr >= all) break;
            const uint32_t h = rr / p.pass_rows, r = rr % p.pass_rows, gr_row = pass * p.pass_rows + r;
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[k][i]));
#pragma unroll
            for (int m = LANES / 2; m; m >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
            const int ex = min(max((int)(__float_as_uint(amax) >> 23) - 127, -100), 127);
            const float up = brc::exp2_int(14 - ex);
            if (d == 0) {
                row_fac[rr] = amax <= 3.402823466e38f ? brc::exp2_int(ex - 14) * p.scale_log2 : __uint_as_float(0x7fffffffu);
                if (h == 0) {   // cells that the row sees; rows of no token: like the last token's
                    const uint32_t tok = gr_row / p.group;
                    row_vis[r] = gr_row >= rows ? len : len + tok + 1u > n_q ? len + tok + 1u - n_q : 0u;
                }
            }
            const uint32_t step = 8u * (d / 128u) + 4u * (d / 16u % 2u) + d / 4u % 4u;   // of the first four values; the next four: step + 1
            const uint32_t at = buf * L.q_bytes + (h * p.pass_rows + r / 8u * 8u) * HD * 2u +
                                ((step / 2u) * 32u + (r % 8u) * 4u + d / 32u % 4u) * 16u;
            uint32_t a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = v[k][2 * i] * up, y = v[k][2 * i + 1] * up;
                a[i] = brc::pack_half2(x, y);
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&a[i]));
                b[i] = brc::pack_half2(x - f.x, y - f.y);
            }
            *reinterpret_cast<uint4 *>(smem + L.q + at) = make_uint4(a[0], a[1], a[2], a[3]);
            if (SPLIT_Q) *reinterpret_cast<uint4 *>(smem + L.q_lo + at) = make_uint4(b[0], b[1], b[2], b[3]);
        }
    }
}

// RT: tiles of eight query rows that a warp carries; RG: warps side by side on a page's rows; KVB: kv heads of a unit; W: consuming
// warps.  SPLIT_Q: q as two binary16 parts (f32; of the 16-bit types one part loses only what lies under 2^-32 of the row's largest).
template <int HD, uint32_t CODE, bool SPLIT_Q, int RT, int RG, int KVB, int W>
__global__ void __launch_bounds__(W * 32 + 128, 1) kv8_attn_kernel(const __grid_constant__ CUtensorMap tm, const AttnParams p) {
    constexpr uint32_t SLABS = HD / 128, CONSUMERS = W * 32, ROW = HD + 4;
    constexpr uint32_t STEP = KVB * RG, LANES = W / STEP, PASS = RG * RT * 8, STAGE = KVB * 2 * 16 * HD, SLAB = STAGE / SLABS;   // LANES: warps that take pages in turn
    constexpr bool MANY = RG == 2;   // more than PASS_ROWS rows take the widest form
    static_assert(W % STEP == 0 && CONSUMERS % (HD / 4) == 0, "");
    extern __shared__ __align__(1024) uint8_t smem[];
    const Smem L = smem_layout(HD, W, KVB, PASS, SPLIT_Q, p.n_stages, p.q_bufs);
    const uint32_t base = brc::smem_u32(smem);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t full0 = base + L.bars, empty0 = full0 + MAX_STAGES * 8u, q_full0 = empty0 + MAX_STAGES * 8u, q_empty0 = q_full0 + 16u;
    uint32_t *warp_cost = reinterpret_cast<uint32_t *>(smem + L.sched);   // [W]: cost of each warp's sequences
    Start *start = reinterpret_cast<Start *>(smem + L.sched + W * 4u);
    if (tid == CONSUMERS) {
        for (uint32_t i = 0; i < p.n_stages; ++i) {
            brc::mbar_init(full0 + 8u * i, 1u);
            brc::mbar_init(empty0 + 8u * i, STEP);       // the warps that read a stage
        }
        for (uint32_t i = 0; i < p.q_bufs; ++i) {
            brc::mbar_init(q_full0 + 8u * i, 3u);                        // helper warps
            brc::mbar_init(q_empty0 + 8u * i, W);
        }
        brc::mbar_fence_init();
        brc::tma_prefetch_desc(&tm);
    }
    // Everything up to here may overlap the end of the kernel in front of this one; what it wrote is read from here on.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    // ---- the cut: costs of all sequences, summed by the consumers over equal runs of sequences
    const uint32_t per_thread = (p.n_seqs + CONSUMERS - 1u) / CONSUMERS;
    uint32_t sum = 0, run = 0;
    if (tid < CONSUMERS) {
        for (uint32_t i = 0; i < per_thread; ++i) {
            const uint32_t s = tid * per_thread + i;
            if (s >= p.n_seqs) break;
            sum += cost_of<MANY>(p, s);
            if (blockIdx.x == 0) {
                if (p.seq_lens[s] > p.max_seq_len) { atomicOr(p.status, BRC_DEV_BAD_POS); p.status[1] = p.seq_lens[s]; }
                if (tokens_of(p, s) > p.max_q) { atomicOr(p.status, BRC_DEV_BAD_POS); p.status[1] = tokens_of(p, s); }
                if (p.cu_q && (p.cu_q[s + 1] > p.total_q || p.cu_q[s + 1] < p.cu_q[s])) { atomicOr(p.status, BRC_DEV_BAD_POS); p.status[1] = p.cu_q[s + 1]; }
            }
        }
        run = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= (uint32_t)o) run += up;
        }
        if (lane == 31u) warp_cost[warp] = run;
    }
    __syncthreads();
    uint32_t before = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < W; ++w) {
        before += w < warp ? warp_cost[w] : 0u;
        total += warp_cost[w];
    }
    const uint32_t share = share_of(total, gridDim.x), lo = min(total, blockIdx.x * share), hi = min(total, lo + share);
    if (tid < CONSUMERS) {
        uint32_t at = before + run - sum;   // cost in front of this thread's sequences
        if (lo < hi && at <= lo && lo < at + sum) {
            uint32_t a = at, c;
            uint32_t s = tid * per_thread;
            while (a + (c = cost_of<MANY>(p, s)) <= lo) {
                a += c;
                ++s;
            }
            c /= units_of<MANY>(p, s);
            const uint32_t u = (lo - a) / c, passes = passes_of<MANY>(p, s), hg = u / passes;
            Cursor first{a + u * c, lo, hi, s, hg, u - hg * passes};
            Segment seg = {};
            seg.n = next_segment<MANY>(p, first, seg) ? seg.n : 0u;
            start->cur = first;
            start->seg = seg;
        }
        if (blockIdx.x == 0) {   // for the merging kernel
            if (tid == 0) p.prefix[0] = 0;
            for (uint32_t i = 0; i < per_thread; ++i) {
                const uint32_t s = tid * per_thread + i;
                if (s >= p.n_seqs) break;
                at += cost_of<MANY>(p, s);
                p.prefix[s + 1] = at;
            }
        }
    }
    if (lo >= hi) return;
    __syncthreads();
    Cursor cur = start->cur;
    Segment g = start->seg;
    bool more = g.n != 0;

    // Registers: launched with 168 / 128 a thread (8 / 12 consuming warps and four more), of which the four others
    // keep 56 and hand the rest to the consumers; the sums stay within what the block was launched with.
    static_assert(W == 8 || W == 12, "");
    if (warp >= W) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        bool ok = true;
        if (warp > W) {
            // -------------------------------------------------------------- helpers: q of every unit but the first
            uint32_t idx = 0;
            for (; more; more = next_segment<MANY>(p, cur, g)) {
                if (idx) {
                    const uint32_t buf = idx % p.q_bufs;
                    if (idx >= p.q_bufs) ok = brc::mbar_wait(q_empty0 + 8u * buf, (idx - p.q_bufs) / p.q_bufs & 1u);
                    if (!ok) break;
                    stage_q<HD, SPLIT_Q, 2>(p, L, smem, g, buf, warp - W - 1u, 3u, lane, [] {});
                    __syncwarp();
                    if (lane == 0) brc::mbar_arrive(q_full0 + 8u * buf);
                }
                ++idx;
            }
        } else {
            // -------------------------------------------------------------- producer: one page-unit per stage, four boxes at a time,
            // a lane each (one lane alone takes 390 clocks for wait, arrival and box; the stream wants a stage of 8 KiB every 345)
            constexpr uint32_t BATCH = 4 / SLABS;   // stages of a round
            const uint64_t policy = brc::l2_policy_evict_first();
            const uint32_t j = lane / SLABS, sl = lane % SLABS;
            uint32_t stage = 0, parity = 1;   // the first round finds every stage empty
            for (; ok && more; more = next_segment<MANY>(p, cur, g)) {
                const uint32_t row0 = g.hg * KVB * 16u;
                const uint32_t *table = p.block_tables + (uint64_t)g.s * p.table_stride + g.pg;
                uint32_t ahead = lane < g.n ? table[lane] : 0u;
                for (uint32_t i0 = 0; ok && i0 < g.n; i0 += 32u) {
                    const uint32_t ids = ahead;
                    if (i0 + 32u + lane < g.n) ahead = table[i0 + 32u + lane];
                    const uint32_t m = min(32u, g.n - i0);
                    for (uint32_t i = 0; ok && i < m; i += BATCH) {
                        uint32_t id = __shfl_sync(0xffffffffu, ids, (i + j) & 31u);
                        if (id >= p.n_pages) id = 0;   // the consumers report it and mask the cells
                        const bool mine = j < BATCH && i + j < m;
                        const bool wrap = stage + j >= p.n_stages;
                        const uint32_t st = wrap ? stage + j - p.n_stages : stage + j;
                        if (mine) {
                            ok = brc::mbar_wait(empty0 + 8u * st, wrap ? parity ^ 1u : parity);
                            if (ok && sl == 0) brc::mbar_arrive_expect_tx(full0 + 8u * st, STAGE);
                        }
                        ok = __all_sync(0xffffffffu, ok);
                        if (mine && ok)
                            brc::tma_load_4d(base + st * STAGE + sl * (SLAB), &tm, (int32_t)(sl * 128u), (int32_t)row0,
                                             (int32_t)(p.page0 + id), 0, full0 + 8u * st, policy);
                        if (ok) stage += min(BATCH, m - i);
                        if (stage >= p.n_stages) { stage -= p.n_stages; parity ^= 1u; }
                    }
                }
            }
            if (!ok)   // a wait ran out: the block may not end while copies into its shared memory are under way
                for (uint32_t i = 0; i < p.n_stages; ++i) brc::mbar_wait(full0 + 8u * i, i < stage ? parity ^ 1u : parity, 1u << 16);
        }
        if (!ok && lane == 0) { atomicOr(p.status, BRC_DEV_WAIT_LIMIT); p.status[1] = blockIdx.x; }
        return;
    }
    if constexpr (W == 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");

    // ---------------------------------------------------------------------- consumers
    const uint32_t t = lane & 3u, gr = lane >> 2;            // thread of a group, group
    const uint32_t hk = warp % KVB, rg = warp / KVB % RG, pl = warp / STEP;
    float *scratch = reinterpret_cast<float *>(smem + L.scratch);
    float4 *stat = reinterpret_cast<float4 *>(smem + L.stat);
    const uint64_t code_bytes = (uint64_t)p.n_kv * 16u * HD;
    // Scales of this warp's next 32 page-units of a segment, one a lane, in two steps so that nobody waits for a page id:
    // ids_of asks for the ids, scales_of some time later for the scales.  An id out of range shows as a negative scale.
    auto ids_of = [&](const Segment &g, uint32_t i0) {
        const uint32_t i = i0 + LANES * lane;
        return i < g.n ? p.block_tables[(uint64_t)g.s * p.table_stride + g.pg + i] : 0u;
    };
    auto scales_of = [&](const Segment &g, uint32_t id, float &ks, float &ev) {
        if (id < p.n_pages) {
            const uint64_t at = id * p.page_bytes + code_bytes + (g.hg * KVB + hk) * 4u;
            ks = *reinterpret_cast<const float *>(p.k_layer + at);
            ev = (float)brc::kv8_scale_exponent(*reinterpret_cast<const float *>(p.v_layer + at));
        } else {
            ks = -1.f;
            ev = 0.f;
            atomicOr(p.status, BRC_DEV_BAD_PAGE);
            p.status[1] = id;
        }
    };
    uint32_t stage = pl, parity = 0;   // of this warp's next page-unit
    uint32_t done = 0, idx = 0;   // page-units and units of the segments before this one
    bool ok = true;

    Segment g_next;
    uint32_t ids = more ? ids_of(g, pl) : 0u;
    while (more) {
        const uint32_t hg = g.hg, pass = g.pass;
        const uint32_t n_q = tokens_of(p, g.s), len = cells_of(p, g.s);
        const uint64_t tok0 = p.cu_q ? p.cu_q[g.s] : (uint64_t)g.s * p.max_q;
        const uint32_t rows = rows_of(p, g.s) * p.group;                 // of a kv head, over all passes
        const uint32_t vis_min = len + 1u > n_q ? len + 1u - n_q : 0u;   // cells that every row sees
        const uint32_t buf_q = idx % p.q_bufs;
        float ks_now = 1.f, ev_now = 0.f, ks_next = 1.f, ev_next = 0.f;
        if (idx == 0) {   // the first unit's q: nobody has anything else to do yet
            // (scales asked for with the q rows: behind the first pages' boxes they would come 3 us later)
            bool asked = false;
            stage_q<HD, SPLIT_Q, RT == 1 ? 2 : 4>(p, L, smem, g, 0, warp, W, lane, [&] { scales_of(g, ids, ks_next, ev_next); asked = true; });
            if (!asked) scales_of(g, ids, ks_next, ev_next);
            brc::named_bar_sync(1, CONSUMERS);
        } else {
            scales_of(g, ids, ks_next, ev_next);
            ok = ok && brc::mbar_wait(q_full0 + 8u * buf_q, (idx - 1u) / p.q_bufs & 1u);
        }
        const float *row_fac = reinterpret_cast<const float *>(smem + L.row_fac) + (buf_q * KVB + hk) * PASS;
        const uint32_t *row_vis = reinterpret_cast<const uint32_t *>(smem + L.row_vis) + buf_q * PASS;
        const uint32_t q_at = buf_q * L.q_bytes + (hk * PASS + rg * RT * 8u) * HD * 2u + lane * 16u;
        const uint32_t q_frag = L.q + q_at, q_frag_lo = L.q_lo + q_at;

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
                fac[n][i] = row_fac[r];
                vis[n][i] = row_vis[r];
            }
        }

        for (uint32_t i = (pl + LANES - done % LANES) % LANES, k = 0; i < g.n; i += LANES, ++k) {
            if (k % 32u == 0u) {
                ks_now = ks_next;
                ev_now = ev_next;
                ids = ids_of(g, i + LANES * 32u);
            } else if (k % 32u == 16u) {
                scales_of(g, ids, ks_next, ev_next);
            }
            const float ks = __shfl_sync(0xffffffffu, ks_now, k % 32u), ev = __shfl_sync(0xffffffffu, ev_now, k % 32u);
            ok = ok && brc::mbar_wait(full0 + 8u * stage, parity);
            if (!ok) break;   // the producer gave up or its copy never came: no further wait, the sums stay as they are
            const uint32_t buf = stage * STAGE;
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
                    const uint4 a = lds128(smem, k_row + (c >> 1) * SLAB + col), b = lds128(smem, k_row + (c >> 1) * SLAB + col + 8u * 128u);
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
                            const uint4 qf = lds128(smem, q_frag + n * 8u * HD * 2u + at);
                            mma(part[n][0], f0, qf.x, qf.y);
                            mma(part[n][1], f1, qf.z, qf.w);
                            if (SPLIT_Q) {
                                const uint4 ql = lds128(smem, q_frag_lo + n * 8u * HD * 2u + at);
                                mma(part[n][0], f0, ql.x, ql.y);
                                mma(part[n][1], f1, ql.z, ql.w);
                            }
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < RT; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[n][x] = part[n][0][x] + part[n][1][x];
            }

            // ---- softmax against the rows' reference exponents; weights to B fragments [cells][rows].  The references
            // move only when a score passes one by more than 2^HEADROOM, so an ordinary page needs no maximum across the warp.
            // The weights' reference is kept relative to the scores' one, and scores enter as differences from that: small
            // numbers beside a large score would be lost.  (The fused difference sees the unrounded score; where its rounding alone passes
            // the reference by 2^HEADROOM, beyond 2^27, the branch takes the rounded one.)
            const bool good = ks > 0.f;
            const bool edge = cell0 + 16u > vis_min || !good;
            uint32_t pw[RT][2], pw_lo[RT][2];
#pragma unroll
            for (int n = 0; n < RT; ++n) {
                float df[4], wt[4];   // scores less their reference, weights
                bool over = false;
#pragma unroll
                for (int x = 0; x < 2; ++x) {   // the thread's two rows: cells gr and gr + 8
                    const float kf = fac[n][x] * ks;
                    df[x] = fmaf(s[n][x], kf, -m_run[n][x]);
                    df[x + 2] = fmaf(s[n][x + 2], kf, -m_run[n][x]);
                    if (edge) {
                        keep_branch();
                        if (!good || cell0 + gr >= vis[n][x]) df[x] = -INFINITY;
                        if (!good || cell0 + gr + 8u >= vis[n][x]) df[x + 2] = -INFINITY;
                    }
                    over |= fmaxf(df[x], df[x + 2]) > fminf(0.f, w_run[n][x] - ev) + HEADROOM;
                }
                if (__any_sync(0xffffffffu, over)) {
                    float f[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float kf = fac[n][x] * ks;
                        const float s0 = df[x] == -INFINITY ? df[x] : s[n][x] * kf, s1 = df[x + 2] == -INFINITY ? df[x + 2] : s[n][x + 2] * kf;
                        float top = fmaxf(s0, s1);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const float m_new = fmaxf(m_run[n][x], top), by = m_run[n][x] - m_new;
                        const float w_old = w_run[n][x] + by, w_new = fmaxf(w_old, top - m_new + ev);
                        l_run[n][x] *= brc::fast_exp2(by);
                        f[x] = brc::fast_exp2(w_old - w_new);
                        m_run[n][x] = m_new;
                        w_run[n][x] = w_new;
                        df[x] = s0 - m_new;
                        df[x + 2] = s1 - m_new;
                    }
#pragma unroll
                    for (int j = 0; j < (int)SLABS * 8; ++j) {
                        o[n][j][0] *= f[0];
                        o[n][j][1] *= f[1];
                        o[n][j][2] *= f[0];
                        o[n][j][3] *= f[1];
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float shift = ev - w_run[n][x] + WEIGHT_SHIFT;
                    l_run[n][x] += brc::fast_exp2(df[x]) + brc::fast_exp2(df[x + 2]);
                    wt[x] = brc::fast_exp2(df[x] + shift);
                    wt[x + 2] = brc::fast_exp2(df[x + 2] + shift);
                }
                const uint32_t a = brc::pack_half2(wt[0], wt[1]), b = brc::pack_half2(wt[2], wt[3]);
                pw[n][0] = brc::movmatrix_trans(a);
                pw[n][1] = brc::movmatrix_trans(b);
                const float2 ha = __half22float2(*reinterpret_cast<const __half2 *>(&a)), hb = __half22float2(*reinterpret_cast<const __half2 *>(&b));
                pw_lo[n][0] = brc::movmatrix_trans(brc::pack_half2(wt[0] - ha.x, wt[1] - ha.y));
                pw_lo[n][1] = brc::movmatrix_trans(brc::pack_half2(wt[2] - hb.x, wt[3] - hb.y));
            }

            // ---- O^T[head_dim][8 rows] += V^T P.  Output row gr of tile j is column 16 gr + j, row gr + 8 column 16 gr + 8 + j.
            const bool tail = cell0 + 16u > len || !good;   // cells nobody sees may hold anything, NaN codes too: 0 x NaN
#pragma unroll
            for (uint32_t sl = 0; sl < SLABS; ++sl) {
                uint32_t w[4][4];
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) {
                    const uint32_t c = 2u * t + (x & 1u) + 8u * (x >> 1);
                    const uint4 v = lds128(smem, buf + sl * SLAB + ((KVB + hk) * 16u + c) * 128u + ((gr ^ (c & 7u)) * 16u));
                    w[x][0] = v.x;
                    w[x][1] = v.y;
                    w[x][2] = v.z;
                    w[x][3] = v.w;
                }
                if (tail) {
                    keep_branch();
#pragma unroll
                    for (uint32_t x = 0; x < 4; ++x)
                        if (!good || cell0 + 2u * t + (x & 1u) + 8u * (x >> 1) >= len) w[x][0] = w[x][1] = w[x][2] = w[x][3] = 0u;
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
                            mma(o[n][sl * 8u + 4u * y + j], fa[j], pw[n][0], pw[n][1]);
                            mma(o[n][sl * 8u + 4u * y + j], fa[j], pw_lo[n][0], pw_lo[n][1]);
                        }
                }
            }
            __syncwarp();
            if (lane == 0) brc::mbar_arrive(empty0 + 8u * stage);
            stage += LANES;
            if (stage >= p.n_stages) { stage -= p.n_stages; parity ^= 1u; }   // (n_stages is a multiple of LANES)
        }
        done += g.n;
        __syncwarp();
        if (lane == 0) brc::mbar_arrive(q_empty0 + 8u * buf_q);
        ++idx;

        // ---- merge the warps that took this unit's pages in turn: they agree on the rows' references, bring their sums to them and
        // add up; then the row is finished, or a partial left
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
        const uint64_t slot = (2ull * blockIdx.x + (g.pg == 0 ? 1u : 0u)) * (KVB * PASS);
        more = next_segment<MANY>(p, cur, g_next);
        if (more) ids = ids_of(g_next, (pl + LANES - done % LANES) % LANES);   // on their way while this unit is merged
        brc::named_bar_sync(1, CONSUMERS);
#pragma unroll
        for (int n = 0; n < RT; ++n) {
            float f[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float4 *st = stat + (warp % STEP) * 16u + n * 8u + 2u * t + x;
                float m = NONE, wm = NONE, l = 0.f;
#pragma unroll
                for (uint32_t q = 0; q < LANES; ++q) {
                    m = fmaxf(m, st[q * STEP * 16u].x);
                }
#pragma unroll
                for (uint32_t q = 0; q < LANES; ++q) {
                    const float by = st[q * STEP * 16u].x - m;
                    wm = fmaxf(wm, st[q * STEP * 16u].y + by);
                    l += st[q * STEP * 16u].z * brc::fast_exp2(by);
                }
                f[x] = brc::fast_exp2(w_run[n][x] + (m_run[n][x] - m) - wm);
                if (whole) f[x] *= l == 0.f ? 0.f : brc::fast_exp2(wm - WEIGHT_SHIFT) / l;
                else if (pl == 0 && gr == 0)
                    *reinterpret_cast<float4 *>(p.ml + (slot + hk * PASS + (rg * RT + n) * 8u + 2u * t + x) * 4u) = make_float4(m, wm, l, 0.f);
            }
#pragma unroll
            for (uint32_t sl = 0; sl < SLABS; ++sl)
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t y = 0; y < 2; ++y)
#pragma unroll
                        for (uint32_t x = 0; x < 2; ++x) {
                            const float(*a)[4] = &o[n][sl * 8u + 4u * y];
                            *reinterpret_cast<float4 *>(scratch + (warp * 8u + 2u * t + x) * ROW + 128u * sl + 16u * gr + 8u * h + 4u * y) =
                                make_float4(a[0][2 * h + x] * f[x], a[1][2 * h + x] * f[x], a[2][2 * h + x] * f[x], a[3][2 * h + x] * f[x]);
                        }
            brc::named_bar_sync(1, CONSUMERS);
            constexpr uint32_t C4 = HD / 4, ITEMS = STEP * 8 * C4, IT = (ITEMS + CONSUMERS - 1) / CONSUMERS;   // groups of four values
            const uint32_t d = tid % C4 * 4u;   // CONSUMERS is a multiple of C4
            float4 v[IT];
#pragma unroll
            for (uint32_t k = 0; k < IT; ++k) {
                const uint32_t row = (tid + k * CONSUMERS) / C4;   // row of a tile + 8 * (head + kvb * row group)
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (ITEMS % CONSUMERS != 0 && row >= STEP * 8u) continue;
#pragma unroll
                for (uint32_t q = 0; q < LANES; ++q) {
                    const float4 x = *reinterpret_cast<const float4 *>(scratch + (row + q * STEP * 8u) * ROW + d);
                    v[k].x += x.x;
                    v[k].y += x.y;
                    v[k].z += x.z;
                    v[k].w += x.w;
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < IT; ++k) {
                const uint32_t row = (tid + k * CONSUMERS) / C4, wg = row / 8u, r = ((wg / KVB) * RT + n) * 8u + row % 8u, h = wg % KVB;
                const uint32_t gr_row = pass * PASS + r;
                if ((ITEMS % CONSUMERS != 0 && row >= STEP * 8u) || gr_row >= rows) continue;
                if (whole) {
                    const uint32_t tok = gr_row / p.group, head = (hg * KVB + h) * p.group + (gr_row - tok * p.group);
                    float y[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
                    finish_row(p, HD, (tok0 + tok) * p.n_head + head, d, y);
                } else {
                    *reinterpret_cast<float4 *>(p.acc + (slot + h * PASS + r) * HD + d) = v[k];
                }
            }
            brc::named_bar_sync(1, CONSUMERS);
        }
        g = g_next;
    }
    if (!ok && lane == 0) { atomicOr(p.status, BRC_DEV_WAIT_LIMIT); p.status[1] = blockIdx.x; }
}

// A load under a predicate, for rows of many partials: left to the compiler they become branches, and each load waits for the one in
// front of it (the merge of 131 072 cells: 8.6 us, 6.8 so; the few partials of a batch's rows are better off with the branch: a
// call of 33.0 us, 33.7 so).
__device__ __forceinline__ void load_if(bool live, const float *at, float4 &v) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t@p ld.global.v4.f32 {%0,%1,%2,%3}, [%5];\n\t}"
                 : "+f"(v.x), "+f"(v.y), "+f"(v.z), "+f"(v.w) : "r"((uint32_t)live), "l"(at) : "memory");
}

// The partials that the shares' boundaries left of each (unit, query row), merged in share order; zeros for a sequence without
// cells.  Units that one share covered are finished already.  W warps per row, ROWS rows per CTA, B partials of a warp
// in flight (their sums and exponents together: one round trip).
template <int HD, int W, int ROWS, int B, bool MANY>
__global__ void __launch_bounds__(W * ROWS * 32) kv8_merge_kernel(const AttnParams p, uint32_t grid) {
    constexpr uint32_t PER = HD / 32;
    __shared__ float part[W == 1 ? 1 : W][HD];
    __shared__ float4 warp_stat[W];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t s = blockIdx.x / p.units_per_seq, u = blockIdx.x % p.units_per_seq;
    const uint32_t before = p.prefix[s], all = p.prefix[s + 1] - before;
    const uint32_t units = units_of<MANY>(p, s);
    if (u >= units) return;   // the longest sequence's passes, not this one's
    const uint32_t share = share_of(p.prefix[p.n_seqs], grid), unit = all / units;
    const uint32_t begin = before + u * unit + p.unit_cost;   // page 0
    const uint32_t c0 = begin / share, c1 = all ? (begin + unit - p.unit_cost - 1u) / share : c0;
    if (all && c0 == c1) return;
    const uint32_t warp = W == 1 ? 0u : threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t passes = passes_of<MANY>(p, s), hg = u / passes, pass = u % passes, row = blockIdx.y * ROWS + (W == 1 ? threadIdx.x >> 5 : 0u);
    const uint32_t h = row / p.pass_rows, r = row % p.pass_rows, gr_row = pass * p.pass_rows + r;
    if (row >= p.kvb * p.pass_rows || gr_row >= rows_of(p, s) * p.group) return;   // whole warps; W > 1: the whole CTA
    const uint32_t n = all ? c1 - c0 + 1u : 0u;

    float m = NONE, wm = NONE, l = 0.f, v[PER];
#pragma unroll
    for (uint32_t j = 0; j < PER; ++j) v[j] = 0.f;
    for (uint32_t i0 = warp; i0 < n; i0 += B * W) {
        float4 st[B], x[B][PER / 4];
#pragma unroll
        for (uint32_t q = 0; q < B; ++q) {
            const uint32_t i = i0 + W * q;
            const uint64_t a = (uint64_t)((2u * (c0 + i) + (i == 0 ? 1u : 0u)) * p.kvb + h) * p.pass_rows + r;
            st[q] = make_float4(NONE, NONE, 0.f, 0.f);
#pragma unroll
            for (uint32_t j = 0; j < PER / 4; ++j) x[q][j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (W > 1) {
                load_if(i < n, p.ml + a * 4u, st[q]);
#pragma unroll
                for (uint32_t j = 0; j < PER / 4; ++j) load_if(i < n, p.acc + a * HD + lane * 4u + 128u * j, x[q][j]);
            } else if (i < n) {
                st[q] = *reinterpret_cast<const float4 *>(p.ml + a * 4u);
#pragma unroll
                for (uint32_t j = 0; j < PER / 4; ++j) x[q][j] = *reinterpret_cast<const float4 *>(p.acc + a * HD + lane * 4u + 128u * j);
            }
        }
        float m_new = m;
#pragma unroll
        for (uint32_t q = 0; q < B; ++q) m_new = fmaxf(m_new, st[q].x);
        const float w_old = wm + (m - m_new);   // relative to the new maximum, as w_new
        float w_new = w_old;
#pragma unroll
        for (uint32_t q = 0; q < B; ++q) w_new = fmaxf(w_new, st[q].y + (st[q].x - m_new));
        const float f = brc::fast_exp2(w_old - w_new);
        l *= brc::fast_exp2(m - m_new);
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) v[j] *= f;
#pragma unroll
        for (uint32_t q = 0; q < B; ++q) {
            const float g = brc::fast_exp2(st[q].y + (st[q].x - m_new) - w_new);
            l += st[q].z * brc::fast_exp2(st[q].x - m_new);
#pragma unroll
            for (uint32_t j = 0; j < PER / 4; ++j) {
                v[4 * j] += x[q][j].x * g;
                v[4 * j + 1] += x[q][j].y * g;
                v[4 * j + 2] += x[q][j].z * g;
                v[4 * j + 3] += x[q][j].w * g;
            }
        }
        m = m_new;
        wm = w_new;
    }
    const uint64_t tok0 = p.cu_q ? p.cu_q[s] : (uint64_t)s * p.max_q;
    const uint64_t head_row = (tok0 + gr_row / p.group) * p.n_head + (hg * p.kvb + h) * p.group + gr_row % p.group;
    if constexpr (W == 1) {
        const float f = l == 0.f ? 0.f : brc::fast_exp2(wm - WEIGHT_SHIFT) / l;
#pragma unroll
        for (uint32_t j = 0; j < PER; j += 4) {
            float x[4] = {v[j] * f, v[j + 1] * f, v[j + 2] * f, v[j + 3] * f};
            finish_row(p, HD, head_row, lane * 4u + 32u * j, x);
        }
    } else {
#pragma unroll
        for (uint32_t j = 0; j < PER; j += 4) *reinterpret_cast<float4 *>(&part[warp][lane * 4u + 32u * j]) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
        if (lane == 0) warp_stat[warp] = make_float4(m, wm, l, 0.f);
        __syncthreads();
        const uint32_t d = threadIdx.x * 4u;
        if (d >= HD) return;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        m = wm = NONE;
        l = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) m = fmaxf(m, warp_stat[w].x);
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) wm = fmaxf(wm, warp_stat[w].y + (warp_stat[w].x - m));
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            const float4 st = warp_stat[w];
            const float g = brc::fast_exp2(st.y + (st.x - m) - wm);
            l += st.z * brc::fast_exp2(st.x - m);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += part[w][d + e] * g;
        }
        const float f = l == 0.f ? 0.f : brc::fast_exp2(wm - WEIGHT_SHIFT) / l;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] *= f;
        finish_row(p, HD, head_row, d, x);
    }
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
    s.prefix_bytes = (((uint64_t)n_seqs + 1u) * 4u + 255u) / 256u * 256u;
    s.ml_bytes = slots * 16u;
    s.acc_bytes = slots * pool->head_dim * 4u;
    return s;
}

template <int HD, uint32_t CODE, bool SPLIT_Q, int RT, int RG, int KVB, int W>
brc_status launch(const brc_pool *pool, AttnParams p, uint32_t grid, uint32_t merge_rows, cudaStream_t st) {
    auto kern = kv8_attn_kernel<HD, CODE, SPLIT_Q, RT, RG, KVB, W>;
    const uint32_t turns = W / (KVB * RG);
    // Ring depth: what fits, in multiples of the warps that take pages in turn, so that a stage is always consumed by the same
    // warps (a parity wait is only valid for a warp that knows the previous round of the barrier is over).
    auto depth = [&](uint32_t q_bufs) {
        uint32_t n = MAX_STAGES / turns * turns;
        while (n > turns && smem_layout(HD, W, p.kvb, p.pass_rows, SPLIT_Q, n, q_bufs).total > SMEM_LIMIT) n -= turns;
        return n;
    };
    p.q_bufs = depth(2) == depth(1) ? 2u : 1u;   // the next unit's q is staged ahead where that costs no ring stage
    p.n_stages = depth(p.q_bufs);
    const uint32_t smem = smem_layout(HD, W, p.kvb, p.pass_rows, SPLIT_Q, p.n_stages, p.q_bufs).total;
    if (smem > SMEM_LIMIT) return brc_fail(BRC_ERR_UNSUPPORTED, "8-bit attention: %u bytes of shared memory", smem);
    static std::atomic<uint64_t> ready{0};   // devices on which this kernel may use all shared memory
    const uint64_t bit = 1ull << (pool->device & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit) || pool->device > 63) {
        BRC_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_LIMIT));
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    // Both kernels are launched so that they may come up while the one in front of them runs out (they wait for its end before they
    // read anything).
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(W * 32 + 128);
    cfg.dynamicSmemBytes = smem;
    BRC_CUDA(cudaLaunchKernelEx(&cfg, kern, pool->tm_kv8, p));
    cfg.dynamicSmemBytes = 0;
    if ((uint64_t)p.n_seqs * p.units_per_seq * 8u <= grid) {
        // Few units have many partials each (one long sequence: one from every SM): 16 warps a row fetch eighty at a time.  Whole call (us)
        // with 16 warps a row and with one, 16 heads over 2 of 256 (a unit a sequence): 1 of 131 072 cells 32.9, 58.0; 8 of 4000-9000
        // 21.0, 24.4; 12 25.7, 26.2; 18 33.3, 32.7; 32 of 512-8192 38.2, 33.6.  8 kv heads of 128 (four units): 4 sequences 20.7, 20.7; 24 77.9, 52.5.
        cfg.gridDim = dim3(p.n_seqs * p.units_per_seq, merge_rows);
        cfg.blockDim = dim3(512);
        BRC_CUDA(cudaLaunchKernelEx(&cfg, kv8_merge_kernel<HD, 16, 1, 5, RG == 2>, p, grid));
    } else {   // many units have a few: a warp a row
        cfg.gridDim = dim3(p.n_seqs * p.units_per_seq, (merge_rows + 7u) / 8u);
        cfg.blockDim = dim3(256);
        BRC_CUDA(cudaLaunchKernelEx(&cfg, kv8_merge_kernel<HD, 1, 8, 6, RG == 2>, p, grid));
    }
    return BRC_OK;
}

template <int HD, uint32_t CODE, bool SPLIT_Q, int KVB>
brc_status launch_rows(const brc_pool *pool, const AttnParams &p, uint32_t grid, uint32_t rt, uint32_t merge_rows, cudaStream_t st) {
    // Warps: what the registers of the sums allow and the ring bears (a stage for each warp that takes pages in turn, twice
    // over).  Measured (us) at 8 and 12 warps of head_dim 128: 32 sequences of 512-8192 cells, 8 kv heads 55.6, 50.4; drafts of 24
    // sequences 53.4, 52.5; eight tokens each 87.3, 81.8; 7 heads over 7 58.6, 60.1.
    constexpr int W = HD == 128 ? 12 : 8;
    if (rt == 1) return launch<HD, CODE, SPLIT_Q, 1, 1, KVB, W>(pool, p, grid, merge_rows, st);
    return p.row_groups == 1 ? launch<HD, CODE, SPLIT_Q, 2, 1, KVB, W>(pool, p, grid, merge_rows, st) : launch<HD, CODE, SPLIT_Q, 2, 2, KVB, W>(pool, p, grid, merge_rows, st);
}

template <int HD, uint32_t CODE>
brc_status launch_kind(const brc_pool *pool, const AttnParams &p, uint32_t grid, bool split_q, uint32_t rt, uint32_t merge_rows, cudaStream_t st) {
    if (p.kvb == 2) return split_q ? launch_rows<HD, CODE, true, 2>(pool, p, grid, rt, merge_rows, st) : launch_rows<HD, CODE, false, 2>(pool, p, grid, rt, merge_rows, st);
    return split_q ? launch_rows<HD, CODE, true, 1>(pool, p, grid, rt, merge_rows, st) : launch_rows<HD, CODE, false, 1>(pool, p, grid, rt, merge_rows, st);
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
    if (a.n_seqs == 0 || a.max_q == 0 || a.total_q == 0) return BRC_OK;
    if (!a.q || !a.block_tables || !a.seq_lens || !a.out)
        return brc_fail(BRC_ERR_INVALID, "%s: NULL query, block table, length or output pointer", who);
    if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.workspace)) & 15u)
        return brc_fail(BRC_ERR_INVALID, "%s: query, output and workspace pointers must be 16-byte aligned", who);
    const Shape s = shape_of(pool, a.n_seqs, a.n_head, a.max_q);
    if ((uint64_t)a.max_q * s.group >= (1ull << 31) || (uint64_t)(pool->n_kv_head / s.kvb) * s.passes >= (1ull << 31) || (uint64_t)a.n_seqs * s.units_per_seq >= (1ull << 31))
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
    p.prefix = reinterpret_cast<uint32_t *>(ws);
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
    p.total_q = a.total_q;
    p.n_pages = pool->n_pages;
    p.page0 = a.layer * pool->n_pages;
    p.n_head = a.n_head;
    p.n_kv = pool->n_kv_head;
    p.group = s.group;
    p.kvb = s.kvb;
    p.row_groups = s.row_groups;
    p.pass_rows = s.pass_rows;
    p.head_groups = pool->n_kv_head / s.kvb;
    p.units_per_seq = s.units_per_seq;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    // Starting and finishing a unit takes a CTA about as long as streaming 128 KiB for each of the unit's heads, half as much again where
    // two row tiles of 256 columns are merged.  Measured (us) at 64, 96, 128, 192, 256 KiB a head, sequences of 512-8192 cells, one row tile: 32 of
    // 16 heads over 2 of 256 33.8, 33.1, 33.0, 33.4, 33.6; 32 heads over 8 of 128 50.6, 50.5, 50.5, 52.6, 54.3; 7 over 7 of 128 58.8, 59.2, 60.3, 63.1, 64.2.
    // Two tiles of 128: drafts of 24 53.8, 51.6, 52.5, 55.1, 58.3.  Two tiles of 256: 16 heads over 2, two tokens 48.6, 47.2, 45.6, 43.3, 42.4, four
    // 78.3, 75.8, 72.7, 68.8, 70.8; 8 over 1, four tokens 48.5, 47.4, 45.6, 43.5, 42.0.
    const uint32_t unit_kib = 128u * s.kvb * (s.rt == 2u && pool->head_dim == 256 ? 3u : 2u) / 2u;
    p.unit_cost = std::max(1u, unit_kib * 1024u / (s.kvb * 2u * 16u * pool->head_dim));
    const uint64_t most = (uint64_t)a.n_seqs * s.units_per_seq * ((a.max_seq_len + 15ull) / 16u + p.unit_cost);   // cost at most
    if (most >= (1ull << 31))
        return brc_fail(BRC_ERR_UNSUPPORTED, "%s: %u sequences of up to %u cells in %u passes each are too much for one call", who, a.n_seqs, a.max_seq_len,
                        s.units_per_seq);
    const uint32_t grid = (uint32_t)std::max<uint64_t>(1u, std::min<uint64_t>(pool->sm_count, (most + MIN_SHARE - 1u) / MIN_SHARE));
    const bool split_q = a.q_dtype == BRC_DTYPE_F32;
    const uint32_t merge_rows = s.kvb * s.pass_rows;
    cudaStream_t st = brc_stream(stream);
    brc_stage_begin(pool, BRC_STAGE_ATTN_PARTIAL, st);
    brc_status rc;
    if (pool->head_dim == 256)
        rc = pool->kv8 == brc::KV8_E4M3 ? launch_kind<256, brc::KV8_E4M3>(pool, p, grid, split_q, s.rt, merge_rows, st)
                                        : launch_kind<256, brc::KV8_INT8>(pool, p, grid, split_q, s.rt, merge_rows, st);
    else
        rc = pool->kv8 == brc::KV8_E4M3 ? launch_kind<128, brc::KV8_E4M3>(pool, p, grid, split_q, s.rt, merge_rows, st)
                                        : launch_kind<128, brc::KV8_INT8>(pool, p, grid, split_q, s.rt, merge_rows, st);
    brc_stage_end(pool, BRC_STAGE_ATTN_PARTIAL, st);
    return rc;
}

extern "C" {

brc_status brc_kv8_attn_workspace_bytes(const brc_pool *pool, uint32_t n_seqs, uint32_t n_head, uint32_t max_q, uint64_t *out_bytes) {
    if (!pool || !out_bytes) return brc_fail(BRC_ERR_INVALID, "brc_kv8_attn_workspace_bytes: NULL argument");
    if (!pool->kv8) return brc_fail(BRC_ERR_UNSUPPORTED, "brc_kv8_attn_workspace_bytes: the pool's pages are not 8-bit (brc_pool_create_kv8)");
    return brc_kv8_workspace(pool, n_seqs, n_head, max_q, out_bytes);
}

brc_status brc_kv8_attn(brc_pool *pool, uint32_t layer, const void *q_dev, int32_t q_dtype, uint32_t n_head,
                        const float *gate_dev, uint32_t gate_head_stride, const uint32_t *block_tables_dev, uint32_t table_stride,
                        const uint32_t *seq_lens_dev, const uint32_t *cu_q_dev, uint32_t n_seqs, uint32_t max_q, uint32_t max_seq_len,
                        float scale, void *out_dev, int32_t out_dtype, void *workspace_dev, uint64_t workspace_bytes, void *stream) {
    brc_kv8_attn_args a = {layer,    q_dev,    q_dtype, n_head,      gate_dev, gate_head_stride, block_tables_dev, table_stride,  seq_lens_dev,
                           cu_q_dev, UINT32_MAX, n_seqs, max_seq_len, max_q,    scale,            out_dev,          out_dtype,     workspace_dev,
                           workspace_bytes};
    return brc_kv8_attend(pool, "brc_kv8_attn", a, stream);
}

brc_status brc_kv8_attn_ragged(brc_pool *pool, uint32_t layer, const void *q_dev, int32_t q_dtype, uint32_t total_q, uint32_t n_head,
                               const float *gate_dev, uint32_t gate_head_stride, const uint32_t *block_tables_dev,
                               uint32_t table_stride, const uint32_t *seq_lens_dev, const uint32_t *cu_q_dev, uint32_t n_seqs,
                               uint32_t max_q, uint32_t max_seq_len, float scale, void *out_dev, int32_t out_dtype, void *workspace_dev,
                               uint64_t workspace_bytes, void *stream) {
    if (!cu_q_dev) return brc_fail(BRC_ERR_INVALID, "brc_kv8_attn_ragged: NULL prefix of the sequences' rows");
    brc_kv8_attn_args a = {layer,    q_dev,   q_dtype, n_head,      gate_dev, gate_head_stride, block_tables_dev, table_stride,  seq_lens_dev,
                           cu_q_dev, total_q, n_seqs,  max_seq_len, max_q,    scale,            out_dev,          out_dtype,     workspace_dev,
                           workspace_bytes};
    return brc_kv8_attend(pool, "brc_kv8_attn_ragged", a, stream);
}

}  // extern "C"
