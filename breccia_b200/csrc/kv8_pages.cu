// The 8-bit cache as it is written and read back (value = code * 2^e, one exponent per page, kv head and side).
//
// brc_kv8_append: one CTA per (page touched, side, group of kv heads).  The page is the unit because the scale is:
// its 128 threads hold the page's new rows in registers (16 x head_dim values, eight consecutive ones at a time), take
// their largest magnitude, and with it the exponent; a page that already holds cells of this sequence keeps the
// larger of its own and the needed exponent, and only when it grows are the kept codes read and rounded again.  K may
// be rotated on the way, so that neither the rotated rows nor a second launch go through memory.
// Bound: HBM for chunks (source rows once, one byte per value written), the launch for a decode step.
//
// brc_kv8_read: the inverse, one CTA per (page, side); HBM.
#include "brc_internal.h"
#include "kv8.cuh"

namespace {

using brc::page_tile;

struct PagesParams {
    uint8_t *k_layer, *v_layer;
    const uint32_t *block_tables, *pos0, *cu_tokens;
    const void *k_src, *v_src;          // append
    void *k_out, *v_out;                // read
    uint64_t k_stride, v_stride;        // elements from one token's source row to the next
    const uint64_t *turns;              // append: rotate K (NULL: as it comes)
    uint32_t *status;
    uint64_t page_bytes;
    uint32_t table_stride, n_seqs, tokens_per_seq, total_tokens, max_pos_end, n_pages, n_kv_head, heads_per_cta;
    uint32_t n_rot, interleaved;
    float factor;
    bool k_vec, v_vec;
};

__device__ void report(uint32_t *status, uint32_t bit, uint32_t value) {
    atomicOr(status, bit);
    status[1] = value;
}

// The tile and its page; false for an idle slot or a refused page (reported once, by the CTA `first`).
__device__ __forceinline__ bool tile_page(const PagesParams &p, bool first, page_tile &t, uint32_t &page) {
    uint32_t cut;
    const bool live = brc::find_tile(blockIdx.x, p.cu_tokens, p.tokens_per_seq, p.total_tokens, p.n_seqs, p.pos0, p.max_pos_end, t, &cut);
    if (cut != UINT32_MAX && first && threadIdx.x == 0) report(p.status, BRC_DEV_BAD_POS, cut);
    if (!live) return false;
    page = p.block_tables[(uint64_t)t.seq * p.table_stride + t.cell0 / 16u];
    if (page < p.n_pages) return true;
    if (first && threadIdx.x == 0) report(p.status, BRC_DEV_BAD_PAGE, page);
    return false;
}

template <uint32_t CODE, int DT, int HD, bool ROPE>
__global__ void __launch_bounds__(128) kv8_append_kernel(const PagesParams p) {
    constexpr uint32_t CHUNKS = HD / 8, ROWS = 128 / CHUNKS, STEPS = 16 / ROWS;   // 8-value chunks of a row; rows at once; rounds
    using T = typename brc::elem<DT>::t;
    extern __shared__ float2 cos_sin[];   // [16 cells][n_rot / 2] (ROPE, K only)
    __shared__ float warp_max[2][4];
    __shared__ int bad_any;
    const bool is_v = blockIdx.y & 1u;
    const uint32_t h0 = (blockIdx.y >> 1) * p.heads_per_cta;
    const uint32_t tid = threadIdx.x, chunk = tid % CHUNKS, row0 = tid / CHUNKS, d = chunk * 8u;
    page_tile t;
    uint32_t page;
    if (!tile_page(p, blockIdx.y == 0, t, page)) return;
    const T *src = static_cast<const T *>(is_v ? p.v_src : p.k_src);
    const uint64_t stride = is_v ? p.v_stride : p.k_stride;
    const bool vec = is_v ? p.v_vec : p.k_vec;
    uint8_t *base = (is_v ? p.v_layer : p.k_layer) + (uint64_t)page * p.page_bytes;
    float *scales = reinterpret_cast<float *>(base + (uint64_t)p.n_kv_head * 16u * HD);
    const bool rotate = ROPE && !is_v;
    const uint32_t half = p.n_rot / 2u;
    if (tid == 0) bad_any = 0;
    if (rotate)
        for (uint32_t i = tid; i < t.count * half; i += 128u)
            cos_sin[i] = brc::rope_cos_sin(t.cell0 + t.first + i / half, p.turns[i % half], p.factor);
    __syncthreads();
    bool bad = false;
    for (uint32_t h = h0; h < min(h0 + p.heads_per_cta, p.n_kv_head); ++h) {
        float v[STEPS][8];
        float amax = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < STEPS; ++i) {
            const uint32_t r = row0 + i * ROWS;   // the r-th new row of the page
            if (r >= t.count) continue;
            const T *row = src + (uint64_t)(t.token0 + r) * stride + (uint64_t)h * HD;
            brc::load8<DT>(row + d, vec, v[i]);
            if (rotate && d < p.n_rot) {
                const float2 *cs = cos_sin + r * half;
                if (p.interleaved) {
#pragma unroll
                    for (uint32_t j = 0; j < 8; j += 2)
                        if (d + j < p.n_rot) {
                            const float2 a = cs[(d + j) / 2u];
                            const float x = v[i][j], y = v[i][j + 1];
                            v[i][j] = x * a.x - y * a.y;
                            v[i][j + 1] = x * a.y + y * a.x;
                        }
                } else if (vec && half % 8u == 0u) {
                    const bool second = d >= half;   // a chunk lies in one half: its partners are a chunk too
                    float o[8];
                    brc::load8<DT>(row + (second ? d - half : d + half), true, o);
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const float2 a = cs[second ? d + j - half : d + j];
                        v[i][j] = second ? o[j] * a.y + v[i][j] * a.x : v[i][j] * a.x - o[j] * a.y;
                    }
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const uint32_t e = d + j;
                        if (e >= p.n_rot) break;
                        const bool second = e >= half;
                        const float2 a = cs[second ? e - half : e];
                        const float o = brc::to_f32(row[second ? e - half : e + half]);
                        v[i][j] = second ? o * a.y + v[i][j] * a.x : v[i][j] * a.x - o * a.y;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float a = fabsf(v[i][j]);
                const bool finite = a <= 3.402823466e38f;   // infinities saturate and NaN becomes 0: neither sets the scale
                bad |= !finite;
                amax = fmaxf(amax, finite ? a : 0.f);
            }
        }
#pragma unroll
        for (int m = 16; m; m >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, m));
        if ((tid & 31u) == 0u) warp_max[h & 1u][tid >> 5] = amax;
        const float old_scale = scales[h];   // read by every thread before the barrier, written behind it
        __syncthreads();                     // two buffers: the next head's maxima cannot overtake this head's reads
        amax = fmaxf(fmaxf(warp_max[h & 1u][0], warp_max[h & 1u][1]), fmaxf(warp_max[h & 1u][2], warp_max[h & 1u][3]));
        int e = brc::kv8_exponent<CODE>(amax);
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
#pragma unroll
        for (uint32_t i = 0; i < STEPS; ++i) {
            const uint32_t r = row0 + i * ROWS;
            if (r >= t.count) continue;
            *reinterpret_cast<uint2 *>(codes + (t.first + r) * HD + d) =
                make_uint2(brc::kv8_encode4<CODE>(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv),
                           brc::kv8_encode4<CODE>(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv));
        }
        if (tid == 0) scales[h] = brc::exp2_int(e);
    }
    if (bad) bad_any = 1;
    __syncthreads();
    if (tid == 0 && bad_any) report(p.status, BRC_DEV_BAD_VALUE, t.token0);
}

template <uint32_t CODE, int DT, int HD>
__global__ void __launch_bounds__(256) kv8_read_kernel(const PagesParams p) {
    constexpr uint32_t CHUNKS = HD / 8;
    using T = typename brc::elem<DT>::t;
    const bool is_v = blockIdx.y & 1u;
    page_tile t;
    uint32_t page;
    if (!tile_page(p, blockIdx.y == 0, t, page)) return;
    const uint8_t *base = (is_v ? p.v_layer : p.k_layer) + (uint64_t)page * p.page_bytes;
    const float *scales = reinterpret_cast<const float *>(base + (uint64_t)p.n_kv_head * 16u * HD);
    const uint64_t row = (uint64_t)p.n_kv_head * HD;
    T *out = static_cast<T *>(is_v ? p.v_out : p.k_out) + t.token0 * row;
    const uint32_t per_row = p.n_kv_head * CHUNKS, n = t.count * per_row;
    constexpr uint32_t U = 4;
    for (uint32_t i0 = threadIdx.x; i0 < n; i0 += 256u * U) {   // U loads in flight a thread
        uint2 w[U];
        float s[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t i = i0 + 256u * u;
            if (i < n) {
                const uint32_t r = i / per_row, c = i % per_row, h = c / CHUNKS;
                w[u] = *reinterpret_cast<const uint2 *>(base + ((uint64_t)h * 16u + t.first + r) * HD + (c % CHUNKS) * 8u);
                s[u] = scales[h];
            }
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t i = i0 + 256u * u;
            if (i >= n) break;
            float a[4], b[4];
            brc::kv8_decode4_f32<CODE>(w[u].x, a);
            brc::kv8_decode4_f32<CODE>(w[u].y, b);
            const float v[8] = {a[0] * s[u], a[1] * s[u], a[2] * s[u], a[3] * s[u], b[0] * s[u], b[1] * s[u], b[2] * s[u], b[3] * s[u]};
            brc::store8<DT>(out + (uint64_t)(i / per_row) * row + (i % per_row) * 8u, true, v);
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
                          uint32_t n_rot, int32_t rope_layout, float rope_factor, void *stream) {
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
    p.k_stride = k_token_stride;
    p.v_stride = v_token_stride;
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
    p.heads_per_cta = 1;
    const dim3 grid((uint32_t)tiles, 2u * ((pool->n_kv_head + p.heads_per_cta - 1u) / p.heads_per_cta));
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
