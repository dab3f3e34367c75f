// The 8-bit cache as it is written and read back (value = code * 2^e, one exponent per page, kv head and side).
//
// brc_kv8_append: one CTA per (page touched, side, group of kv heads).  The page is the unit because the scale is:
// its 128 threads hold a head's new rows in registers (16 x head_dim values, eight consecutive ones at a time), take
// their largest magnitude, and with it the exponent; a page that already holds cells of this sequence keeps the
// larger of its own and the needed exponent, and only when it grows are the kept codes read and rounded again.  K may
// be rotated on the way, so that neither the rotated rows nor a second launch go through memory; the cos / sin pairs of
// the page's positions are computed once for all heads of the CTA.  While a head is encoded the next one's rows are on
// their way.  Bound: HBM for chunks (source rows once, one byte per value written), the launch for a decode step.
//
// brc_kv8_read: the inverse, one CTA per (page, side); HBM.
#include <algorithm>

#include "brc_internal.h"
#include "kv8.cuh"

namespace {

using brc::page_tile;

struct PagesParams {
    uint8_t *k_layer, *v_layer;
    const uint32_t *block_tables, *pos0, *cu_tokens;
    const void *k_src, *v_src;          // append
    void *k_out, *v_out;                // read
    uint32_t k_stride, v_stride;        // elements from one token's source row to the next (16 rows of them fit 32 bits)
    const uint64_t *turns;              // append: rotate K (NULL: as it comes)
    uint32_t *status;
    uint64_t page_bytes;
    uint32_t table_stride, n_seqs, tokens_per_seq, total_tokens, max_pos_end, n_pages, n_kv_head, heads_per_cta;
    uint32_t n_rot, interleaved;
    double factor;
    bool k_vec, v_vec;
};

__device__ void report(uint32_t *status, uint32_t bit, uint32_t value) {
    atomicOr(status, bit);
    status[1] = value;
}

// The CTA's tile; false for an idle slot.  A cut-off position is reported once, by the CTA `first`.
__device__ __forceinline__ bool tile_of(const PagesParams &p, bool first, page_tile &t) {
    uint32_t cut;
    const bool live = brc::find_tile(blockIdx.x, p.cu_tokens, p.tokens_per_seq, p.total_tokens, p.n_seqs, p.pos0, p.max_pos_end, t, &cut);
    if (cut != UINT32_MAX && first && threadIdx.x == 0) report(p.status, BRC_DEV_BAD_POS, cut);
    return live;
}

// The eight values from column d of one new K row, rotated.  `row`: the row in memory, for pairs that no shuffle reaches.
template <int DT, int HD>
__device__ __forceinline__ void rotate8(const PagesParams &p, const typename brc::elem<DT>::t *row, const float2 *cs, uint32_t d, bool live,
                                        const brc::raw8<DT> &raw, float (&v)[8]) {
    const uint32_t half = p.n_rot / 2u;
    if (p.interleaved) {
#pragma unroll
        for (uint32_t j = 0; j < 8; j += 2)
            if (d + j < p.n_rot) {
                const float2 a = cs[(d + j) / 2u];
                const float x = v[j], y = v[j + 1];
                v[j] = x * a.x - y * a.y;
                v[j + 1] = x * a.y + y * a.x;
            }
    } else if (half % 8u == 0u) {   // a chunk lies in one half, its partners are the chunk half / 8 lanes away
        const bool second = d >= half;
        const uint32_t lane = threadIdx.x & 31u, from = d >= p.n_rot ? lane : second ? lane - half / 8u : lane + half / 8u;
        brc::raw8<DT> other;   // of the first half: negated, (x c - y s); of the second: (y c + x s)
        const uint32_t sign = second ? 0u : DT == 0 ? 0x80000000u : 0x80008000u;
#pragma unroll
        for (int j = 0; j < brc::raw8<DT>::WORDS; ++j) other.w[j] = __shfl_sync(0xffffffffu, raw.w[j], from) ^ sign;
        if (d < p.n_rot) {
            float o[8];
            other.values(o);
            const float4 *a4 = reinterpret_cast<const float4 *>(cs + (second ? d - half : d));   // 16-byte aligned: d and half are multiples of 8
#pragma unroll
            for (uint32_t j = 0; j < 8; j += 2) {
                const float4 a = a4[j / 2u];
                v[j] = v[j] * a.x + o[j] * a.y;
                v[j + 1] = v[j + 1] * a.z + o[j + 1] * a.w;
            }
        }
    } else if (live) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t e = d + j;
            if (e >= p.n_rot) break;
            const bool second = e >= half;
            const float2 a = cs[second ? e - half : e];
            const float o = brc::to_f32(row[second ? e - half : e + half]);
            v[j] = second ? o * a.y + v[j] * a.x : v[j] * a.x - o * a.y;
        }
    }
}

// CTAs an SM that the compiler has to leave registers for: more of them hide the loads and barriers of one another until the
// registers spill.  16 000 tokens, measured (us) with one CTA fewer, as chosen, with one more.  8 heads of 128, rotated: bf16 (8) 35.3, 34.0, 34.0,
// f32 (6) 44.3, 40.1, 40.7; as they come (9): bf16 25.2, 25.0, 26.0, f32 31.4, 31.4, 32.3.  2 heads of 256, rotated: f16 (5) 24.5, 22.6, 23.5,
// f32 (4) 31.5, 28.3, 33.5; as they come: f16 (6) 15.3, 14.2, 14.9, f32 (4) 18.8, 18.8, 18.6.
constexpr int append_ctas(int dt, int hd, bool rope) { return hd == 128 ? (rope ? (dt == 0 ? 6 : 8) : 9) : dt == 0 ? 4 : rope ? 5 : 6; }

template <uint32_t CODE, int DT, int HD, bool ROPE>
__global__ void __launch_bounds__(128, append_ctas(DT, HD, ROPE)) kv8_append_kernel(const PagesParams p) {
    constexpr uint32_t CHUNKS = HD / 8, ROWS = 128 / CHUNKS, STEPS = 16 / ROWS;   // 8-value chunks of a row; rows at once; rounds
    using T = typename brc::elem<DT>::t;
    extern __shared__ __align__(16) float2 cos_sin[];   // [16 cells][n_rot / 2] (ROPE, K only)
    __shared__ uint32_t warp_max[2][4];
    const bool is_v = blockIdx.y & 1u;
    const uint32_t h0 = (blockIdx.y >> 1) * p.heads_per_cta, h1 = min(h0 + p.heads_per_cta, p.n_kv_head);
    const uint32_t tid = threadIdx.x, chunk = tid % CHUNKS, row0 = tid / CHUNKS, d = chunk * 8u;
    page_tile t;
    if (!tile_of(p, blockIdx.y == 0, t)) return;
    const uint32_t stride = is_v ? p.v_stride : p.k_stride;
    const T *src = static_cast<const T *>(is_v ? p.v_src : p.k_src) + (uint64_t)t.token0 * stride;
    const bool vec = is_v ? p.v_vec : p.k_vec;
    const bool rotate = ROPE && !is_v;
    brc::raw8<DT> next[STEPS];
    auto load = [&](uint32_t h) {
#pragma unroll
        for (uint32_t i = 0; i < STEPS; ++i) {
            const uint32_t r = row0 + i * ROWS;   // the r-th new row of the page
            if (r < t.count) next[i].load(src + (r * stride + h * HD + d), vec);
            else next[i].zero();
        }
    };
    load(h0);   // the rows do not wait for the page's id
    const uint32_t page = p.block_tables[(uint64_t)t.seq * p.table_stride + t.cell0 / 16u];
    if (page >= p.n_pages) {
        if (blockIdx.y == 0 && tid == 0) report(p.status, BRC_DEV_BAD_PAGE, page);
        return;
    }
    uint8_t *base = (is_v ? p.v_layer : p.k_layer) + (uint64_t)page * p.page_bytes;
    float *scales = reinterpret_cast<float *>(base + (uint64_t)p.n_kv_head * 16u * HD);
    const uint32_t half = p.n_rot / 2u;
    if (rotate)
        for (uint32_t i = tid; i < t.count * half; i += 128u)
            cos_sin[i] = brc::rope_cos_sin(t.cell0 + t.first + i / half, p.turns[i % half], p.factor);
    __syncthreads();
    for (uint32_t h = h0; h < h1; ++h) {
        brc::raw8<DT> raw[STEPS];
        float v[STEPS][8];   // rotated K alone; else the raw words are unpacked where they are encoded
        uint32_t top = 0u;
#pragma unroll
        for (uint32_t i = 0; i < STEPS; ++i) raw[i] = next[i];
        if (h + 1u < h1) load(h + 1u);
        if (rotate) {
#pragma unroll
            for (uint32_t i = 0; i < STEPS; ++i) {
                const uint32_t r = row0 + i * ROWS;
                raw[i].values(v[i]);
                rotate8<DT, HD>(p, src + (r * stride + h * HD), cos_sin + (r < t.count ? r : 0u) * half, d, r < t.count, raw[i], v[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) top = brc::max_magnitude(top, v[i][j]);
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < STEPS; ++i) raw[i].top(top);
            top = brc::raw8<DT>::top_f32(top);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if ((tid & 31u) == 0u) warp_max[h & 1u][tid >> 5] = top;
        const float old_scale = t.first ? scales[h] : 0.f;   // read by every thread in front of the barrier, written behind it
        __syncthreads();                                     // two buffers: the next head's maxima cannot overtake this head's reads
        top = max(max(warp_max[h & 1u][0], warp_max[h & 1u][1]), max(warp_max[h & 1u][2], warp_max[h & 1u][3]));
        const bool bad = top >= 0x7f800000u;   // an infinity or NaN among them: the largest finite magnitude, once more and apart
        if (bad) {
            top = 0u;
#pragma unroll
            for (uint32_t i = 0; i < STEPS; ++i) {
                if (!rotate) raw[i].values(v[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t a = __float_as_uint(v[i][j]) & 0x7fffffffu;
                    if (a < 0x7f800000u) top = max(top, a);
                }
            }
            top = __reduce_max_sync(0xffffffffu, top);
            __syncthreads();
            if ((tid & 31u) == 0u) warp_max[h & 1u][tid >> 5] = top;
            __syncthreads();
            top = max(max(warp_max[h & 1u][0], warp_max[h & 1u][1]), max(warp_max[h & 1u][2], warp_max[h & 1u][3]));
            if (tid == 0) report(p.status, BRC_DEV_BAD_VALUE, t.token0);
        }
        int e = brc::kv8_exponent<CODE>(__uint_as_float(top));
        uint8_t *codes = base + (uint64_t)h * 16u * HD;
        if (t.first) {
            const int e_old = brc::kv8_scale_exponent(old_scale);
            if (e > e_old) {   // the kept cells move to the larger scale
                const int by = e_old - e;
                const float f = by < -126 ? 0.f : brc::exp2_int(by);
#pragma unroll
                for (uint32_t i = 0; i < STEPS; ++i) {
                    const uint32_t c = row0 + i * ROWS;
                    if (c >= t.first) continue;
                    uint2 *at = reinterpret_cast<uint2 *>(codes + c * HD + d);
                    const uint2 w = *at;
                    float a[4], b[4];
                    brc::kv8_decode4_f32<CODE>(w.x, a);
                    brc::kv8_decode4_f32<CODE>(w.y, b);
                    *at = make_uint2(brc::kv8_encode4<CODE>(a[0] * f, a[1] * f, a[2] * f, a[3] * f),
                                     brc::kv8_encode4<CODE>(b[0] * f, b[1] * f, b[2] * f, b[3] * f));
                }
            }
            e = max(e, e_old);
        }
        const float inv = brc::exp2_int(-e);
        const bool plain = !bad && __uint_as_float(top) * inv <= (CODE == brc::KV8_E4M3 ? 448.f : 127.f);   // (the exponent's upper clamp may leave some to saturate)
#pragma unroll
        for (uint32_t i = 0; i < STEPS; ++i) {
            const uint32_t r = row0 + i * ROWS;
            if (r >= t.count) continue;
            if (!rotate) raw[i].values(v[i]);
            uint2 w;
            if (plain)
                w = make_uint2(brc::kv8_encode4_finite<CODE>(v[i][0], v[i][1], v[i][2], v[i][3], inv),
                               brc::kv8_encode4_finite<CODE>(v[i][4], v[i][5], v[i][6], v[i][7], inv));
            else
                w = make_uint2(brc::kv8_encode4<CODE>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv),
                               brc::kv8_encode4<CODE>(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv));
            *reinterpret_cast<uint2 *>(codes + (t.first + r) * HD + d) = w;
        }
        if (tid == 0) scales[h] = brc::exp2_int(e);
    }
}

template <uint32_t CODE, int DT, int HD>
__global__ void __launch_bounds__(256) kv8_read_kernel(const PagesParams p) {
    constexpr uint32_t N = DT == 0 ? 4 : 8, CHUNKS = HD / N, U = 4;   // a chunk: sixteen bytes of output; U of them in flight a thread
    using T = typename brc::elem<DT>::t;
    const bool is_v = blockIdx.y & 1u;
    page_tile t;
    if (!tile_of(p, blockIdx.y == 0, t)) return;
    const uint32_t page = p.block_tables[(uint64_t)t.seq * p.table_stride + t.cell0 / 16u];
    if (page >= p.n_pages) {
        if (blockIdx.y == 0 && threadIdx.x == 0) report(p.status, BRC_DEV_BAD_PAGE, page);
        return;
    }
    const uint8_t *base = (is_v ? p.v_layer : p.k_layer) + (uint64_t)page * p.page_bytes;
    const float *scales = reinterpret_cast<const float *>(base + (uint64_t)p.n_kv_head * 16u * HD);
    const uint32_t per_row = p.n_kv_head * CHUNKS, dr = 256u / per_row, dc = 256u % per_row;
    T *out = static_cast<T *>(is_v ? p.v_out : p.k_out) + (uint64_t)t.token0 * per_row * N;
    uint32_t r = threadIdx.x / per_row, c = threadIdx.x % per_row;
    while (r < t.count) {
        uint32_t w[U][N / 4];
        float s[U];
        uint32_t at[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            at[u] = UINT32_MAX;
            if (r < t.count) {
                const uint32_t h = c / CHUNKS;
                at[u] = r * per_row + c;
                const uint8_t *from = base + (h * 16u + t.first + r) * HD + (c % CHUNKS) * N;
                if constexpr (N == 8) {
                    const uint2 x = __ldcs(reinterpret_cast<const uint2 *>(from));
                    w[u][0] = x.x;
                    w[u][1] = x.y;
                } else {
                    w[u][0] = __ldcs(reinterpret_cast<const uint32_t *>(from));
                }
                s[u] = __ldg(scales + h);
            }
            r += dr;
            c += dc;
            if (c >= per_row) { c -= per_row; ++r; }
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            if (at[u] == UINT32_MAX) break;
            float v[N];
#pragma unroll
            for (uint32_t x = 0; x < N / 4; ++x) {
                float a[4];
                brc::kv8_decode4_f32<CODE>(w[u][x], a);
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y) v[4 * x + y] = a[y] * s[u];
            }
            T *to = out + (uint64_t)at[u] * N;
            if constexpr (N == 8)
                *reinterpret_cast<uint4 *>(to) = make_uint4(brc::pack2<DT>(v[0], v[1]), brc::pack2<DT>(v[2], v[3]), brc::pack2<DT>(v[4], v[5]), brc::pack2<DT>(v[6], v[7]));
            else *reinterpret_cast<float4 *>(to) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

template <uint32_t CODE, int DT>
cudaError_t launch_append(const PagesParams &p, uint32_t hd, dim3 grid, cudaStream_t st) {
    const uint32_t smem = p.turns ? 16u * (p.n_rot / 2u) * (uint32_t)sizeof(float2) : 0u;
    if (hd == 256) {
        if (p.turns) kv8_append_kernel<CODE, DT, 256, true><<<grid, 128, smem, st>>>(p);
        else kv8_append_kernel<CODE, DT, 256, false><<<grid, 128, 0, st>>>(p);
    } else {
        if (p.turns) kv8_append_kernel<CODE, DT, 128, true><<<grid, 128, smem, st>>>(p);
        else kv8_append_kernel<CODE, DT, 128, false><<<grid, 128, 0, st>>>(p);
    }
    return cudaGetLastError();
}

template <uint32_t CODE, int DT>
cudaError_t launch_read(const PagesParams &p, uint32_t hd, dim3 grid, cudaStream_t st) {
    if (hd == 256) kv8_read_kernel<CODE, DT, 256><<<grid, 256, 0, st>>>(p);
    else kv8_read_kernel<CODE, DT, 128><<<grid, 256, 0, st>>>(p);
    return cudaGetLastError();
}

#define BRC_KV8_DISPATCH(fn, pool, dtype, ...)                                                                              \
    ((pool)->kv8 == brc::KV8_E4M3                                                                                            \
         ? ((dtype) == BRC_DTYPE_F32 ? fn<brc::KV8_E4M3, 0>(__VA_ARGS__)                                                    \
                                     : (dtype) == BRC_DTYPE_F16 ? fn<brc::KV8_E4M3, 1>(__VA_ARGS__) : fn<brc::KV8_E4M3, 2>(__VA_ARGS__)) \
         : ((dtype) == BRC_DTYPE_F32 ? fn<brc::KV8_INT8, 0>(__VA_ARGS__)                                                    \
                                     : (dtype) == BRC_DTYPE_F16 ? fn<brc::KV8_INT8, 1>(__VA_ARGS__) : fn<brc::KV8_INT8, 2>(__VA_ARGS__)))

// What append and read check alike.  *go = false: nothing to do.
brc_status validate(const brc_pool *pool, const char *who, const char *verb, uint32_t layer, const void *tables, uint32_t table_stride,
                    const void *pos0, uint32_t n_seqs, uint32_t tokens_per_seq, const void *cu, uint32_t total, uint32_t max_pos_end,
                    const void *k, const void *v, int32_t dtype, bool *go) {
    *go = false;
    if (!pool) return brc_fail(BRC_ERR_INVALID, "%s: pool is NULL", who);
    if (pool->device < 0 || !pool->k_base)
        return brc_fail(BRC_ERR_CUDA, "%s: this pool holds bookkeeping only (no device memory); compute calls need a GPU pool", who);
    if (!pool->kv8) return brc_fail(BRC_ERR_UNSUPPORTED, "%s: the pool's pages are not 8-bit (brc_pool_create_kv8)", who);
    if (layer >= pool->n_layers) return brc_fail(BRC_ERR_INVALID, "%s: layer %u but the pool has %u", who, layer, pool->n_layers);
    if (dtype != BRC_DTYPE_F32 && dtype != BRC_DTYPE_F16 && dtype != BRC_DTYPE_BF16)
        return brc_fail(BRC_ERR_INVALID, "%s: dtype %d is none of f32 (0), f16 (1), bf16 (2)", who, dtype);
    if (!cu && (uint64_t)n_seqs * tokens_per_seq != total)
        return brc_fail(BRC_ERR_INVALID, "%s: %u sequences x %u tokens != total_tokens %u", who, n_seqs, tokens_per_seq, total);
    const uint64_t capacity = (uint64_t)table_stride * pool->page_tokens;
    if (max_pos_end > capacity)
        return brc_fail(BRC_ERR_CAPACITY, "%s would %s cells up to %u but each block table holds %llu (%u pages of %u cells)", who, verb,
                        max_pos_end, (unsigned long long)capacity, table_stride, pool->page_tokens);
    if (total == 0 || n_seqs == 0) return BRC_OK;
    if (!tables || !pos0 || !k || !v) return brc_fail(BRC_ERR_INVALID, "%s: NULL block table, position, K or V pointer", who);
    if (brc::tile_slots(total, n_seqs) >= (1ull << 31))
        return brc_fail(BRC_ERR_UNSUPPORTED, "%s: %u tokens of %u sequences in one call", who, total, n_seqs);
    *go = true;
    return BRC_OK;
}

}  // namespace

extern "C" {

brc_status brc_kv8_append(brc_pool *pool, uint32_t layer, const uint32_t *block_tables_dev, uint32_t table_stride,
                          const uint32_t *pos0_dev, uint32_t n_seqs, uint32_t tokens_per_seq, const uint32_t *cu_tokens_dev,
                          uint32_t total_tokens, uint32_t max_pos_end, const void *k_src_dev, uint64_t k_token_stride,
                          const void *v_src_dev, uint64_t v_token_stride, int32_t src_dtype, const uint64_t *rope_turns_dev,
                          uint32_t n_rot, int32_t rope_layout, double rope_factor, void *stream) {
    const char *who = "brc_kv8_append";
    bool go;
    if (brc_status rc = validate(pool, who, "write", layer, block_tables_dev, table_stride, pos0_dev, n_seqs, tokens_per_seq,
                                 cu_tokens_dev, total_tokens, max_pos_end, k_src_dev, v_src_dev, src_dtype, &go))
        return rc;
    const uint32_t row = pool->n_kv_head * pool->head_dim, size = src_dtype == BRC_DTYPE_F32 ? 4u : 2u;
    if (k_token_stride == 0) k_token_stride = row;
    if (v_token_stride == 0) v_token_stride = row;
    if (k_token_stride < row || v_token_stride < row)
        return brc_fail(BRC_ERR_INVALID, "%s: token strides %llu / %llu but a token has %u values", who, (unsigned long long)k_token_stride,
                        (unsigned long long)v_token_stride, row);
    if (k_token_stride >= (1ull << 27) || v_token_stride >= (1ull << 27))
        return brc_fail(BRC_ERR_UNSUPPORTED, "%s: token strides %llu / %llu (below 2^27)", who, (unsigned long long)k_token_stride, (unsigned long long)v_token_stride);
    if (rope_turns_dev) {
        if (n_rot == 0 || n_rot % 2u || n_rot > pool->head_dim)
            return brc_fail(BRC_ERR_INVALID, "%s: n_rot %u (even, 2 .. head_dim %u)", who, n_rot, pool->head_dim);
        if (rope_layout != BRC_ROPE_HALF && rope_layout != BRC_ROPE_INTERLEAVED)
            return brc_fail(BRC_ERR_INVALID, "%s: rope_layout %d is neither half (0) nor interleaved (1)", who, rope_layout);
    }
    if (!go) return BRC_OK;
    if ((reinterpret_cast<uintptr_t>(k_src_dev) | reinterpret_cast<uintptr_t>(v_src_dev)) & (size - 1u))
        return brc_fail(BRC_ERR_INVALID, "%s: source pointers must be multiples of the element size", who);
    brc_device_guard guard(pool->device);
    if (!guard.ok) return brc_fail(BRC_ERR_CUDA, "%s: cannot make device %d current", who, pool->device);
    PagesParams p = {};
    p.k_layer = pool->k_base + (uint64_t)layer * pool->layer_bytes;
    p.v_layer = pool->v_base + (uint64_t)layer * pool->v_layer_bytes;
    p.block_tables = block_tables_dev;
    p.pos0 = pos0_dev;
    p.cu_tokens = cu_tokens_dev;
    p.k_src = k_src_dev;
    p.v_src = v_src_dev;
    p.k_stride = (uint32_t)k_token_stride;
    p.v_stride = (uint32_t)v_token_stride;
    p.turns = rope_turns_dev;
    p.status = pool->status_dev;
    p.page_bytes = pool->half_page_bytes;
    p.table_stride = table_stride;
    p.n_seqs = n_seqs;
    p.tokens_per_seq = tokens_per_seq;
    p.total_tokens = total_tokens;
    p.max_pos_end = max_pos_end;
    p.n_pages = pool->n_pages;
    p.n_kv_head = pool->n_kv_head;
    p.n_rot = n_rot;
    p.interleaved = rope_layout == BRC_ROPE_INTERLEAVED;
    p.factor = rope_factor;
    p.k_vec = ((reinterpret_cast<uintptr_t>(k_src_dev) | (k_token_stride * size)) & 15u) == 0;
    p.v_vec = ((reinterpret_cast<uintptr_t>(v_src_dev) | (v_token_stride * size)) & 15u) == 0;
    const uint64_t tiles = brc::tile_slots(total_tokens, n_seqs);
    // Heads a CTA: as many as leave an SM five CTAs with work (the search, the positions' cos and sin and the start are then paid
    // once for several heads, and the next head's rows travel while one is encoded).  Pages that the call touches are counted from below; of
    // the slots, a decode step leaves every other one idle.  One, two, four, eight heads a CTA, one token each in 8 heads of 128, bf16,
    // rotated: 32 sequences 4.2, 5.0, 6.6, 9.8 us (one taken); 64: 6.2, 5.2, 6.9, 10.1 (two); 144: 10.1, 8.0, 8.1, 10.5 (four); 512: 27.8, 19.6,
    // 15.9, 15.8 (eight); one sequence of 5000 tokens 16.7, 12.9, 11.9, 13.0 (four); 64 of 100 25.8, 19.3, 17.4, 17.4 (eight).
    // Two heads of 256, where a CTA takes one up to 185 pages: 144 sequences 5.7 and 6.2 rotated, 4.3 and 3.7 not.
    const uint64_t pages = std::max<uint64_t>(total_tokens / 16u, std::min(n_seqs, total_tokens)), want = 5ull * pool->sm_count;
    const uint32_t most = (uint32_t)std::min<uint64_t>((2u * pages * pool->n_kv_head + want - 1u) / want, pool->n_kv_head);
    const uint32_t groups = (pool->n_kv_head + most - 1u) / most;
    p.heads_per_cta = (pool->n_kv_head + groups - 1u) / groups;
    const dim3 grid((uint32_t)tiles, 2u * groups);
    brc_stage_begin(pool, BRC_STAGE_KV_APPEND, brc_stream(stream));
    const cudaError_t e = BRC_KV8_DISPATCH(launch_append, pool, src_dtype, p, pool->head_dim, grid, brc_stream(stream));
    brc_stage_end(pool, BRC_STAGE_KV_APPEND, brc_stream(stream));
    BRC_CUDA(e);
    return BRC_OK;
}

brc_status brc_kv8_read(brc_pool *pool, uint32_t layer, const uint32_t *block_tables_dev, uint32_t table_stride,
                        const uint32_t *pos0_dev, uint32_t n_seqs, uint32_t tokens_per_seq, const uint32_t *cu_tokens_dev,
                        uint32_t total_tokens, uint32_t max_pos_end, void *k_out_dev, void *v_out_dev, int32_t out_dtype, void *stream) {
    const char *who = "brc_kv8_read";
    bool go;
    if (brc_status rc = validate(pool, who, "read", layer, block_tables_dev, table_stride, pos0_dev, n_seqs, tokens_per_seq,
                                 cu_tokens_dev, total_tokens, max_pos_end, k_out_dev, v_out_dev, out_dtype, &go))
        return rc;
    if (!go) return BRC_OK;
    if ((reinterpret_cast<uintptr_t>(k_out_dev) | reinterpret_cast<uintptr_t>(v_out_dev)) & 15u)
        return brc_fail(BRC_ERR_INVALID, "%s: output pointers must be 16-byte aligned", who);
    brc_device_guard guard(pool->device);
    if (!guard.ok) return brc_fail(BRC_ERR_CUDA, "%s: cannot make device %d current", who, pool->device);
    PagesParams p = {};
    p.k_layer = pool->k_base + (uint64_t)layer * pool->layer_bytes;
    p.v_layer = pool->v_base + (uint64_t)layer * pool->v_layer_bytes;
    p.block_tables = block_tables_dev;
    p.pos0 = pos0_dev;
    p.cu_tokens = cu_tokens_dev;
    p.k_out = k_out_dev;
    p.v_out = v_out_dev;
    p.status = pool->status_dev;
    p.page_bytes = pool->half_page_bytes;
    p.table_stride = table_stride;
    p.n_seqs = n_seqs;
    p.tokens_per_seq = tokens_per_seq;
    p.total_tokens = total_tokens;
    p.max_pos_end = max_pos_end;
    p.n_pages = pool->n_pages;
    p.n_kv_head = pool->n_kv_head;
    const dim3 grid((uint32_t)brc::tile_slots(total_tokens, n_seqs), 2u);
    brc_stage_begin(pool, BRC_STAGE_PAGE_GATHER, brc_stream(stream));
    const cudaError_t e = BRC_KV8_DISPATCH(launch_read, pool, out_dtype, p, pool->head_dim, grid, brc_stream(stream));
    brc_stage_end(pool, BRC_STAGE_PAGE_GATHER, brc_stream(stream));
    BRC_CUDA(e);
    return BRC_OK;
}

}  // extern "C"
