// Rotary positions of query and key rows: pairs in the half layout (j, j + n_rot / 2) or interleaved (2j, 2j + 1), the
// first n_rot values of a head (the others pass through), frequencies scaled for long contexts or not.
//
//   (x, y) -> factor * (x cos a - y sin a, x sin a + y cos a),   a = 2 pi * position * turns_j
//
// The angle is an integer product (kv8.cuh, rope_cos_sin): exact to position * 2^-65 turns at every position, without a
// table (one of cos and sin for 10^6 positions of 128 pairs would be 1 GB).  A CTA computes the cos / sin pairs of its
// tokens once, in shared memory, for all their heads, of q and k alike; then every thread moves 16-byte chunks, both
// halves of a pair by the same thread, so a call may work in place.  Bound: HBM (each value read and written once);
// the launch for a decode step.
#include <algorithm>
#include <cmath>

#include "brc_internal.h"
#include "kv8.cuh"

namespace {

struct RopeSide {
    const void *in;
    void *out;
    uint64_t in_stride, out_stride;   // elements from token to token
    uint32_t heads, vec;              // vec: rows may be moved in 16-byte pieces
};

struct RopeParams {
    RopeSide side[2];
    const uint32_t *positions;
    const uint64_t *turns;
    uint32_t n_tokens, tokens_per_cta, head_dim, n_rot, interleaved;
    float factor;
};

// Pairs [j, j + 8) of a head in the half layout, or values [d, d + 8) otherwise, eight at a time.
template <int DT>
__device__ __forceinline__ void rotate_side(const RopeParams &p, const RopeSide &s, const float2 *cos_sin, uint32_t tok0, uint32_t n_tok) {
    using T = typename brc::elem<DT>::t;
    const T *in = static_cast<const T *>(s.in);
    T *out = static_cast<T *>(s.out);
    const uint32_t half = p.n_rot / 2u, hd = p.head_dim;
    const bool in_place = s.in == s.out && s.in_stride == s.out_stride;
    if (s.vec) {
        // items of a head: half layout: half / 8 chunk pairs then the untouched chunks; interleaved: all chunks
        const uint32_t rot_items = p.interleaved ? p.n_rot / 8u : half / 8u;
        const uint32_t items = rot_items + (in_place ? 0u : (hd - p.n_rot) / 8u);
        const uint32_t per_tok = s.heads * items, n = n_tok * per_tok;
        for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
            const uint32_t tk = i / per_tok, r = i % per_tok, h = r / items, c = r % items;
            const T *x = in + (uint64_t)(tok0 + tk) * s.in_stride + (uint64_t)h * hd;
            T *y = out + (uint64_t)(tok0 + tk) * s.out_stride + (uint64_t)h * hd;
            const float2 *cs = cos_sin + tk * half;
            float a[8];
            if (c >= rot_items) {
                const uint32_t d = p.n_rot + (c - rot_items) * 8u;
                brc::load8<DT>(x + d, true, a);
                brc::store8<DT>(y + d, true, a);
            } else if (p.interleaved) {
                const uint32_t d = c * 8u;
                brc::load8<DT>(x + d, true, a);
                float o[8];
#pragma unroll
                for (uint32_t j = 0; j < 8; j += 2) {
                    const float2 w = cs[(d + j) / 2u];
                    o[j] = a[j] * w.x - a[j + 1] * w.y;
                    o[j + 1] = a[j] * w.y + a[j + 1] * w.x;
                }
                brc::store8<DT>(y + d, true, o);
            } else {
                const uint32_t d = c * 8u;
                float b[8], o[8], q[8];
                brc::load8<DT>(x + d, true, a);
                brc::load8<DT>(x + d + half, true, b);
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    const float2 w = cs[d + j];
                    o[j] = a[j] * w.x - b[j] * w.y;
                    q[j] = a[j] * w.y + b[j] * w.x;
                }
                brc::store8<DT>(y + d, true, o);
                brc::store8<DT>(y + d + half, true, q);
            }
        }
        return;
    }
    const uint32_t items = half + (in_place ? 0u : hd - p.n_rot);   // pairs, then single untouched values
    const uint32_t per_tok = s.heads * items;
    const uint64_t n = (uint64_t)n_tok * per_tok;
    for (uint64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint32_t tk = (uint32_t)(i / per_tok), r = (uint32_t)(i % per_tok), h = r / items, c = r % items;
        const T *x = in + (uint64_t)(tok0 + tk) * s.in_stride + (uint64_t)h * hd;
        T *y = out + (uint64_t)(tok0 + tk) * s.out_stride + (uint64_t)h * hd;
        if (c >= half) {
            const uint32_t d = p.n_rot + (c - half);
            y[d] = x[d];
            continue;
        }
        const uint32_t d0 = p.interleaved ? 2u * c : c, d1 = p.interleaved ? 2u * c + 1u : c + half;
        const float a = brc::to_f32(x[d0]), b = brc::to_f32(x[d1]);
        const float2 w = cos_sin[tk * half + c];
        y[d0] = brc::from_f32<DT>(a * w.x - b * w.y);
        y[d1] = brc::from_f32<DT>(a * w.y + b * w.x);
    }
}

// blockIdx.y = 0: q, 1: k (its own CTAs, so that a decode step's few tokens spread)
template <int DT>
__global__ void __launch_bounds__(256) rope_kernel(const RopeParams p) {
    extern __shared__ float2 cos_sin[];
    const uint32_t tok0 = blockIdx.x * p.tokens_per_cta;
    const uint32_t n_tok = min(p.tokens_per_cta, p.n_tokens - tok0), half = p.n_rot / 2u;
    for (uint32_t i = threadIdx.x; i < n_tok * half; i += blockDim.x)
        cos_sin[i] = brc::rope_cos_sin(p.positions[tok0 + i / half], p.turns[i % half], p.factor);
    __syncthreads();
    for (uint32_t s = 0; s < 2; ++s)
        if (p.side[s].in) rotate_side<DT>(p, p.side[s], cos_sin, tok0, n_tok);
}

}  // namespace

extern "C" {

brc_status brc_rope_freqs(const brc_rope_params *a, uint64_t *out_turns, float *out_factor) {
    const char *who = "brc_rope_freqs";
    if (!a || !out_turns || !out_factor) return brc_fail(BRC_ERR_INVALID, "%s: NULL argument", who);
    if (a->n_rot == 0 || a->n_rot % 2u || a->n_rot > 256u)
        return brc_fail(BRC_ERR_INVALID, "%s: n_rot %u (even, 2 .. 256)", who, a->n_rot);
    if (!(a->theta >= 1.0) || !std::isfinite(a->theta)) return brc_fail(BRC_ERR_INVALID, "%s: theta %g (>= 1)", who, a->theta);
    if (a->scaling < BRC_ROPE_NONE || a->scaling > BRC_ROPE_BANDS) return brc_fail(BRC_ERR_INVALID, "%s: scaling %d", who, a->scaling);
    if (a->scaling != BRC_ROPE_NONE && (!(a->factor >= 1.0) || !std::isfinite(a->factor)))
        return brc_fail(BRC_ERR_INVALID, "%s: scaling factor %g (>= 1)", who, a->factor);
    const bool by_band = a->scaling == BRC_ROPE_YARN || a->scaling == BRC_ROPE_BANDS;
    if (by_band && (a->orig_ctx == 0 || !(a->turns_low > 0.0) || !(a->turns_high > a->turns_low) || !std::isfinite(a->turns_high)))
        return brc_fail(BRC_ERR_INVALID, "%s: original context %u, band of %g .. %g turns (0 < low < high)", who, a->orig_ctx, a->turns_low,
                        a->turns_high);
    if (a->scaling == BRC_ROPE_YARN && !(a->theta > 1.0)) return brc_fail(BRC_ERR_INVALID, "%s: yarn needs theta > 1", who);
    if (!(a->mscale >= 0.0) || !std::isfinite(a->mscale)) return brc_fail(BRC_ERR_INVALID, "%s: mscale %g (0: the scaling's own)", who, a->mscale);
    const long double two_pi = 6.283185307179586476925286766559L, n = a->n_rot;
    long double theta = a->theta;
    if (a->scaling == BRC_ROPE_NTK && a->n_rot > 2u) theta *= powl(a->factor, n / (n - 2.0L));
    long double lo = 0.0L, hi = 1.0L;   // yarn: pairs below lo keep their frequency, above hi take it / factor
    if (a->scaling == BRC_ROPE_YARN) {
        auto at = [&](double turns) { return n * logl(a->orig_ctx / (turns * two_pi)) / (2.0L * logl(theta)); };
        lo = fmaxl(floorl(at(a->turns_high)), 0.0L);
        hi = fminl(ceill(at(a->turns_low)), n - 1.0L);
    }
    for (uint32_t j = 0; j < a->n_rot / 2u; ++j) {
        long double f = powl(theta, -2.0L * j / n);
        if (a->scaling == BRC_ROPE_LINEAR) {
            f /= a->factor;
        } else if (a->scaling == BRC_ROPE_YARN) {
            const long double ramp = fminl(fmaxl((j - lo) / fmaxl(hi - lo, 0.001L), 0.0L), 1.0L);
            f = f / a->factor * ramp + f * (1.0L - ramp);
        } else if (a->scaling == BRC_ROPE_BANDS) {
            const long double turns = a->orig_ctx * f / two_pi;   // turns over the original context
            const long double keep = fminl(fmaxl((turns - a->turns_low) / (a->turns_high - a->turns_low), 0.0L), 1.0L);
            f = f / a->factor * (1.0L - keep) + f * keep;
        }
        out_turns[j] = (uint64_t)(f / two_pi * 0x1p64L + 0.5L);   // f <= 1: below 0.16 turns
    }
    *out_factor = a->mscale > 0.0 ? (float)a->mscale : a->scaling == BRC_ROPE_YARN ? (float)(0.1 * std::log(a->factor) + 1.0) : 1.f;
    return BRC_OK;
}

brc_status brc_rope_apply(int32_t device, const void *q_dev, void *q_out_dev, uint32_t n_head, uint64_t q_token_stride,
                          uint64_t q_out_token_stride, const void *k_dev, void *k_out_dev, uint32_t n_kv_head, uint64_t k_token_stride,
                          uint64_t k_out_token_stride, uint32_t head_dim, int32_t dtype, const uint32_t *positions_dev,
                          uint32_t n_tokens, const uint64_t *turns_dev, uint32_t n_rot, int32_t layout, float factor, void *stream) {
    const char *who = "brc_rope_apply";
    if (dtype != BRC_DTYPE_F32 && dtype != BRC_DTYPE_F16 && dtype != BRC_DTYPE_BF16)
        return brc_fail(BRC_ERR_INVALID, "%s: dtype %d is none of f32 (0), f16 (1), bf16 (2)", who, dtype);
    if (layout != BRC_ROPE_HALF && layout != BRC_ROPE_INTERLEAVED)
        return brc_fail(BRC_ERR_INVALID, "%s: layout %d is neither half (0) nor interleaved (1)", who, layout);
    if (head_dim == 0 || head_dim > 1024u) return brc_fail(BRC_ERR_UNSUPPORTED, "%s: head_dim %u (1 .. 1024)", who, head_dim);
    if (n_rot == 0 || n_rot % 2u || n_rot > head_dim || n_rot > 256u)
        return brc_fail(BRC_ERR_INVALID, "%s: n_rot %u (even, 2 .. min(256, head_dim %u))", who, n_rot, head_dim);
    if (n_tokens && !q_dev && !k_dev) return brc_fail(BRC_ERR_INVALID, "%s: neither q nor k", who);
    const uint32_t size = dtype == BRC_DTYPE_F32 ? 4u : 2u;
    RopeParams p = {};
    const void *in[2] = {q_dev, k_dev};
    void *out[2] = {q_out_dev, k_out_dev};
    const uint32_t heads[2] = {n_head, n_kv_head};
    const uint64_t is[2] = {q_token_stride, k_token_stride}, os[2] = {q_out_token_stride, k_out_token_stride};
    uint32_t total_heads = 0;
    for (int s = 0; s < 2; ++s) {
        if (!in[s]) continue;
        const uint64_t row = (uint64_t)heads[s] * head_dim;
        if (!out[s] || heads[s] == 0) return brc_fail(BRC_ERR_INVALID, "%s: %s with %u heads and output %p", who, s ? "k" : "q", heads[s], out[s]);
        if (heads[s] > 65535u) return brc_fail(BRC_ERR_UNSUPPORTED, "%s: %u heads", who, heads[s]);
        RopeSide &r = p.side[s];
        r.in = in[s];
        r.out = out[s];
        r.heads = heads[s];
        r.in_stride = is[s] ? is[s] : row;
        r.out_stride = os[s] ? os[s] : row;
        if (r.in_stride < row || r.out_stride < row)
            return brc_fail(BRC_ERR_INVALID, "%s: token strides %llu / %llu but a token has %llu values", who, (unsigned long long)r.in_stride,
                            (unsigned long long)r.out_stride, (unsigned long long)row);
        const uintptr_t at = reinterpret_cast<uintptr_t>(in[s]) | reinterpret_cast<uintptr_t>(out[s]);
        if (at & (size - 1u)) return brc_fail(BRC_ERR_INVALID, "%s: pointers must be multiples of the element size", who);
        // in place means the same rows; rows that overlap in any other way would be read after they were written
        if (n_tokens) {
            const uint64_t a0 = reinterpret_cast<uintptr_t>(in[s]), a1 = a0 + ((n_tokens - 1) * r.in_stride + row) * size;
            const uint64_t b0 = reinterpret_cast<uintptr_t>(out[s]), b1 = b0 + ((n_tokens - 1) * r.out_stride + row) * size;
            if (a0 < b1 && b0 < a1 && !(a0 == b0 && r.in_stride == r.out_stride))
                return brc_fail(BRC_ERR_INVALID, "%s: %s and its output overlap without being the same rows", who, s ? "k" : "q");
        }
        // 16-byte pieces: aligned rows, and pairs whose chunks of eight do not straddle the rotated part's edges
        r.vec = ((at | (r.in_stride * size) | (r.out_stride * size)) & 15u) == 0 && head_dim % 8u == 0 && n_rot % 8u == 0 &&
                (layout == BRC_ROPE_INTERLEAVED || (n_rot / 2u) % 8u == 0);
        total_heads += heads[s];
    }
    if (n_tokens == 0) return BRC_OK;
    if (!positions_dev || !turns_dev) return brc_fail(BRC_ERR_INVALID, "%s: NULL position or frequency pointer", who);
    brc_device_guard guard(device);
    if (!guard.ok) return brc_fail(BRC_ERR_CUDA, "%s: cannot make device %d current", who, device);
    p.positions = positions_dev;
    p.turns = turns_dev;
    p.n_tokens = n_tokens;
    p.head_dim = head_dim;
    p.n_rot = n_rot;
    p.interleaved = layout == BRC_ROPE_INTERLEAVED;
    p.factor = factor;
    // Tokens per CTA: about 32 KiB of rows (a few hundred chunks a thread's loop can overlap), fewer while that leaves
    // SMs without a CTA, never more cos / sin pairs than 32 KiB of shared memory.
    const uint32_t bytes = total_heads * head_dim * size;
    p.tokens_per_cta = std::min(std::max(1u, 32768u / bytes), std::max(1u, 8192u / n_rot));
    p.tokens_per_cta = std::min(p.tokens_per_cta, std::max(1u, n_tokens / 296u));
    const uint32_t smem = p.tokens_per_cta * (n_rot / 2u) * (uint32_t)sizeof(float2);
    const uint32_t grid = (n_tokens + p.tokens_per_cta - 1u) / p.tokens_per_cta;
    cudaStream_t st = brc_stream(stream);
    if (dtype == BRC_DTYPE_F32) rope_kernel<0><<<grid, 256, smem, st>>>(p);
    else if (dtype == BRC_DTYPE_F16) rope_kernel<1><<<grid, 256, smem, st>>>(p);
    else rope_kernel<2><<<grid, 256, smem, st>>>(p);
    BRC_CUDA(cudaGetLastError());
    return BRC_OK;
}

}  // extern "C"
