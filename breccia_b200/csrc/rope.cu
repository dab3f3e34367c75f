// Rotary positions of query and key rows: pairs in the half layout (j, j + n_rot / 2) or interleaved (2j, 2j + 1), the
// first n_rot values of a head (the others pass through), frequencies scaled for long contexts or not.
//
//   (x, y) -> factor * (x cos a - y sin a, x sin a + y cos a),   a = 2 pi * position * turns_j
//
// The angle is an integer product (kv8.cuh, rope_cos_sin): exact to position * 2^-65 turns at every position, without a
// table (one of cos and sin for 10^6 positions of 128 pairs would be 1 GB).  A warp takes a token: it computes the
// cos / sin pairs of its position once, keeps those of its lanes' columns in registers, and goes over the token's
// heads, of q and k alike, sixteen bytes a lane, the next rows on their way while one is turned.  A row is read whole
// before it is written, so a call may work in place.  A pair's other half comes by shuffle where it lies whole chunks
// away, else through shared memory.  Bound: HBM (each value read and written once); the launch for a decode step.
#include <algorithm>
#include <cmath>

#include "brc_internal.h"
#include "kv8.cuh"

namespace {

struct RopeSide {
    const void *in;
    void *out;
    uint64_t in_stride, out_stride;   // elements from token to token
    uint32_t heads;
};

struct RopeParams {
    RopeSide side[2];
    const uint32_t *positions;
    const uint64_t *turns;
    uint32_t n_tokens, tokens_per_cta, splits, head_dim, n_rot, interleaved, is_signed;
    double factor;
    __device__ __forceinline__ uint64_t position(uint32_t tok) const {
        const uint32_t x = positions[tok];
        return is_signed ? (uint64_t)(int64_t)(int32_t)x : x;
    }
};

// Sixteen bytes of a row in f32.
template <int DT>
struct Chunk {
    static constexpr int N = DT == 0 ? 4 : 8;
    uint4 w;
    __device__ __forceinline__ void values(float (&v)[N]) const {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == 0) {
                v[i] = __uint_as_float(u[i]);
            } else if constexpr (DT == 1) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(u[i] << 16);
                v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            }
        }
    }
    __device__ __forceinline__ void pack(const float (&v)[N]) {
        if constexpr (DT == 0) w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        else w = make_uint4(brc::pack2<DT>(v[0], v[1]), brc::pack2<DT>(v[2], v[3]), brc::pack2<DT>(v[4], v[5]), brc::pack2<DT>(v[6], v[7]));
    }
};

enum Pairing { INTERLEAVED, HALF_CHUNKS, HALF_ANY };   // HALF_CHUNKS: n_rot / 2 is whole chunks

constexpr uint32_t ROPE_WARPS = 8, ROPE_MAX_PAIRS = 128, ROPE_STAGE = 256 + 8;   // staged values of a warp: 256, one word of shift every 32

// Rows of HD values whose addresses are multiples of 16 bytes.  `splits` warps share a token's rows.  64 bytes a lane are turned
// while the next 64 travel, three CTAs an SM: 16384 tokens of 40 x 128 bf16 in 54.9 us interleaved (6.1 TB/s), 56.2 half;
// with 32 bytes a lane 58.0 and 59.7, with 16 and no look-ahead 58.3 and 74.9.
template <int DT, int HD, int PAIR>
__global__ void __launch_bounds__(ROPE_WARPS * 32, 3) rope_kernel(const RopeParams p) {
    using T = typename brc::elem<DT>::t;
    constexpr uint32_t N = Chunk<DT>::N, CHUNKS = HD / N, LPR = CHUNKS < 32 ? CHUNKS : 32, CPL = CHUNKS / LPR, RPW = 32 / LPR;   // lanes of a row, chunks of a lane, rows of a warp
    __shared__ float2 pairs_all[ROPE_WARPS][ROPE_MAX_PAIRS];
    __shared__ float stage_all[PAIR == HALF_ANY ? ROPE_WARPS : 1][PAIR == HALF_ANY ? ROPE_STAGE : 1];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, half = p.n_rot / 2u;
    const uint32_t job = blockIdx.x * ROPE_WARPS + warp, tok = job / p.splits, split = job % p.splits;
    if (tok >= p.n_tokens) return;
    float2 *pairs = pairs_all[warp];
    float *stage = stage_all[PAIR == HALF_ANY ? warp : 0];
    const uint32_t heads_q = p.side[0].in ? p.side[0].heads : 0u, heads = heads_q + (p.side[1].in ? p.side[1].heads : 0u);
    const uint32_t sub = lane / LPR, col = lane % LPR * N;
    // this token's rows of each side (the side's fields picked by value: an indexed parameter would go through local memory)
    const T *q_in = static_cast<const T *>(p.side[0].in) + (uint64_t)tok * p.side[0].in_stride;
    const T *k_in = static_cast<const T *>(p.side[1].in) + (uint64_t)tok * p.side[1].in_stride;
    T *q_out = static_cast<T *>(p.side[0].out) + (uint64_t)tok * p.side[0].out_stride, *k_out = static_cast<T *>(p.side[1].out) + (uint64_t)tok * p.side[1].out_stride;
    uint32_t r = split * RPW + sub;
    const uint32_t step = p.splits * RPW;
    constexpr uint32_t F = 4 / CPL;   // rows of a lane in flight
    Chunk<DT> next[F][CPL];
    auto load = [&](uint32_t r) {
#pragma unroll
        for (uint32_t f = 0; f < F; ++f) {
            const uint32_t rr = r + f * step;
            if (rr >= heads) break;
            const T *x = (rr < heads_q ? q_in + rr * HD : k_in + (rr - heads_q) * HD) + col;
#pragma unroll
            for (uint32_t k = 0; k < CPL; ++k) next[f][k].w = *reinterpret_cast<const uint4 *>(x + k * LPR * N);
        }
    };
    load(r);
    const uint64_t pos = p.position(tok);
    for (uint32_t j = lane; j < half; j += 32u) pairs[j] = brc::rope_cos_sin(pos, p.turns[j], p.factor);
    __syncwarp();
    // cos and sin of the lane's columns (INTERLEAVED: of its pairs); the sine with the sign that a column's partner enters with
    constexpr uint32_t CS = PAIR == INTERLEAVED ? N / 2 : N;
    float c[CPL][CS], s[CPL][CS];
#pragma unroll
    for (uint32_t k = 0; k < CPL; ++k)
#pragma unroll
        for (uint32_t j = 0; j < CS; ++j) {
            const uint32_t e = PAIR == INTERLEAVED ? (col + k * LPR * N) / 2u + j : col + k * LPR * N + j;
            const bool in = e < (PAIR == INTERLEAVED ? half : p.n_rot);
            const float2 w = pairs[!in ? 0u : PAIR == INTERLEAVED || e < half ? e : e - half];
            c[k][j] = w.x;
            s[k][j] = PAIR != INTERLEAVED && e < half ? -w.y : w.y;
        }
    for (uint32_t r0 = split * RPW; r0 < heads; r0 += F * step, r += F * step) {   // whole warps
        Chunk<DT> rows[F][CPL];
#pragma unroll
        for (uint32_t f = 0; f < F; ++f)
#pragma unroll
            for (uint32_t k = 0; k < CPL; ++k) rows[f][k] = next[f][k];
        if (r0 + F * step < heads) load(r + F * step);
#pragma unroll
        for (uint32_t f = 0; f < F; ++f) {
            if (r0 + f * step >= heads) break;
            const uint32_t rr = r + f * step;
            const bool live = rr < heads;   // the lane's row exists
            Chunk<DT>(&now)[CPL] = rows[f];
            float v[CPL][N], o[CPL][N];
#pragma unroll
            for (uint32_t k = 0; k < CPL; ++k) now[k].values(v[k]);
            if constexpr (PAIR == HALF_CHUNKS) {
#pragma unroll
                for (uint32_t k = 0; k < CPL; ++k) {
                    const uint32_t d = col + k * LPR * N;
                    const uint32_t q = d >= p.n_rot ? d / N : (d < half ? d + half : d - half) / N;   // the partner's chunk
                    Chunk<DT> other;
                    uint32_t u[4];
                    const uint32_t from = sub * LPR + q % LPR;
#pragma unroll
                    for (uint32_t x = 0; x < 4; ++x) {
                        u[x] = 0u;
#pragma unroll
                        for (uint32_t kk = 0; kk < CPL; ++kk) {
                            const uint32_t w = __shfl_sync(0xffffffffu, x == 0 ? now[kk].w.x : x == 1 ? now[kk].w.y : x == 2 ? now[kk].w.z : now[kk].w.w, from);
                            if (q / LPR == kk) u[x] = w;
                        }
                    }
                    other.w = make_uint4(u[0], u[1], u[2], u[3]);
                    other.values(o[k]);
                }
            } else if constexpr (PAIR == HALF_ANY) {
                __syncwarp();
#pragma unroll
                for (uint32_t k = 0; k < CPL; ++k)
#pragma unroll
                    for (uint32_t j = 0; j < N; ++j) {
                        const uint32_t i = sub * HD + col + k * LPR * N + j;
                        stage[i + i / 32u] = v[k][j];
                    }
                __syncwarp();
#pragma unroll
                for (uint32_t k = 0; k < CPL; ++k)
#pragma unroll
                    for (uint32_t j = 0; j < N; ++j) {
                        const uint32_t d = col + k * LPR * N + j, i = sub * HD + (d >= p.n_rot ? d : d < half ? d + half : d - half);
                        o[k][j] = stage[i + i / 32u];
                    }
            }
#pragma unroll
            for (uint32_t k = 0; k < CPL; ++k) {
                float y[N];
#pragma unroll
                for (uint32_t j = 0; j < N; ++j) {
                    const uint32_t d = col + k * LPR * N + j;
                    if constexpr (PAIR == INTERLEAVED) {
                        const float x = v[k][j], z = v[k][j ^ 1u], t = j & 1u ? x * c[k][j / 2] + z * s[k][j / 2] : x * c[k][j / 2] - z * s[k][j / 2];
                        y[j] = d < p.n_rot ? t : x;
                    } else {
                        const float t = v[k][j] * c[k][j] + o[k][j] * s[k][j];
                        y[j] = d < p.n_rot ? t : v[k][j];
                    }
                }
                now[k].pack(y);
                if (live) *reinterpret_cast<uint4 *>((rr < heads_q ? q_out + rr * HD : k_out + (rr - heads_q) * HD) + col + k * LPR * N) = now[k].w;
            }
        }
    }
}

// Any head size, any alignment: a pair, or an untouched value, a thread.  Bound by its two-byte accesses and the divisions that
// find an item's head and pair: 16384 tokens of 40 heads in bf16 take 131 us with heads of 96 (floor 39), 114 with heads of 80 (32), 172 with heads
// of 128 whose rows are not 16-byte aligned (52); 18 heads of 192 in f32 168 us (70).
template <int DT>
__global__ void __launch_bounds__(256) rope_any_kernel(const RopeParams p) {
    using T = typename brc::elem<DT>::t;
    extern __shared__ float2 cos_sin[];
    const uint32_t tok0 = blockIdx.x * p.tokens_per_cta;
    const uint32_t n_tok = min(p.tokens_per_cta, p.n_tokens - tok0), half = p.n_rot / 2u, hd = p.head_dim;
    for (uint32_t i = threadIdx.x; i < n_tok * half; i += blockDim.x)
        cos_sin[i] = brc::rope_cos_sin(p.position(tok0 + i / half), p.turns[i % half], p.factor);
    __syncthreads();
    const uint32_t items = half + (hd - p.n_rot);   // pairs, then single untouched values
    for (uint32_t side = 0; side < 2; ++side) {
        const RopeSide &s = p.side[side];
        if (!s.in) continue;
        const uint32_t per_tok = s.heads * items;
        const uint64_t n = (uint64_t)n_tok * per_tok;
        for (uint64_t i = threadIdx.x; i < n; i += blockDim.x) {
            const uint32_t tk = (uint32_t)(i / per_tok), r = (uint32_t)(i % per_tok), h = r / items, c = r % items;
            const T *x = static_cast<const T *>(s.in) + (uint64_t)(tok0 + tk) * s.in_stride + (uint64_t)h * hd;
            T *y = static_cast<T *>(s.out) + (uint64_t)(tok0 + tk) * s.out_stride + (uint64_t)h * hd;
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
}

template <int DT, int HD>
void launch_rows(const RopeParams &p, uint32_t grid, cudaStream_t st) {
    if (p.interleaved) rope_kernel<DT, HD, INTERLEAVED><<<grid, ROPE_WARPS * 32, 0, st>>>(p);
    else if (p.n_rot / 2u % Chunk<DT>::N == 0) rope_kernel<DT, HD, HALF_CHUNKS><<<grid, ROPE_WARPS * 32, 0, st>>>(p);
    else rope_kernel<DT, HD, HALF_ANY><<<grid, ROPE_WARPS * 32, 0, st>>>(p);
}

template <int DT>
void launch(RopeParams &p, bool rows, uint32_t total_heads, int sm_count, cudaStream_t st) {
    if (rows) {
        // A warp a token; its rows over several warps while that leaves SMs short of them.
        const uint32_t rpw = std::max(1u, 32u * Chunk<DT>::N / p.head_dim), most = (total_heads + rpw - 1u) / rpw;
        const uint64_t want = 16ull * sm_count;
        p.splits = (uint32_t)std::min<uint64_t>(most, std::max<uint64_t>(1u, want / p.n_tokens));
        const uint64_t jobs = (uint64_t)p.n_tokens * p.splits;
        const uint32_t grid = (uint32_t)((jobs + ROPE_WARPS - 1u) / ROPE_WARPS);
        if (p.head_dim == 64) launch_rows<DT, 64>(p, grid, st);
        else if (p.head_dim == 128) launch_rows<DT, 128>(p, grid, st);
        else launch_rows<DT, 256>(p, grid, st);
        return;
    }
    // Tokens per CTA: about 32 KiB of rows, fewer while that leaves SMs without a CTA, never more cos / sin pairs than 32 KiB.
    const uint32_t bytes = total_heads * p.head_dim * brc::elem<DT>::size;
    p.tokens_per_cta = std::min(std::max(1u, 32768u / bytes), std::max(1u, 8192u / p.n_rot));
    p.tokens_per_cta = std::min(p.tokens_per_cta, std::max(1u, p.n_tokens / 296u));
    const uint32_t smem = p.tokens_per_cta * (p.n_rot / 2u) * (uint32_t)sizeof(float2);
    const uint32_t grid = (uint32_t)(((uint64_t)p.n_tokens + p.tokens_per_cta - 1u) / p.tokens_per_cta);
    rope_any_kernel<DT><<<grid, 256, smem, st>>>(p);
}

struct Rows {   // n of them: `bytes` each, from `at`, `stride` bytes apart
    uint64_t at, stride, bytes;
};

// No byte of a's rows is one of b's: other ranges, or other columns of rows that are wider than both.
bool apart(const Rows &a, const Rows &b, uint32_t n) {
    if (a.at + (n - 1u) * a.stride + a.bytes <= b.at || b.at + (n - 1u) * b.stride + b.bytes <= a.at) return true;
    if (n == 1u || a.stride != b.stride) return false;
    const uint64_t s = a.stride, d = b.at >= a.at ? (b.at - a.at) % s : (s - (a.at - b.at) % s) % s;
    return d >= a.bytes && d + b.bytes <= s;
}

}  // namespace

extern "C" {

brc_status brc_rope_freqs(const brc_rope_params *a, uint64_t *out_turns, double *out_factor) {
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
    *out_factor = a->mscale > 0.0 ? a->mscale : a->scaling == BRC_ROPE_YARN ? 0.1 * std::log(a->factor) + 1.0 : 1.0;
    return BRC_OK;
}

brc_status brc_rope_apply(int32_t device, const void *q_dev, void *q_out_dev, uint32_t n_head, uint64_t q_token_stride,
                          uint64_t q_out_token_stride, const void *k_dev, void *k_out_dev, uint32_t n_kv_head, uint64_t k_token_stride,
                          uint64_t k_out_token_stride, uint32_t head_dim, int32_t dtype, const uint32_t *positions_dev,
                          uint32_t n_tokens, const uint64_t *turns_dev, uint32_t n_rot, int32_t layout, double factor, void *stream) {
    const char *who = "brc_rope_apply";
    if (dtype != BRC_DTYPE_F32 && dtype != BRC_DTYPE_F16 && dtype != BRC_DTYPE_BF16)
        return brc_fail(BRC_ERR_INVALID, "%s: dtype %d is none of f32 (0), f16 (1), bf16 (2)", who, dtype);
    const bool is_signed = layout & BRC_ROPE_SIGNED;
    layout &= ~BRC_ROPE_SIGNED;
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
    bool rows = head_dim == 64 || head_dim == 128 || head_dim == 256;   // the kernel of whole rows: these sizes, 16-byte aligned
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
        rows = rows && ((at | (r.in_stride * size) | (r.out_stride * size)) & 15u) == 0;
        total_heads += heads[s];
    }
    if (n_tokens == 0) return BRC_OK;
    // in place means the same rows; rows that overlap in any other way would be read after they were written
    for (int s = 0; s < 2; ++s) {
        const RopeSide &r = p.side[s], &other = p.side[1 - s];
        if (!r.in) continue;
        const Rows x{reinterpret_cast<uintptr_t>(r.in), r.in_stride * size, (uint64_t)r.heads * head_dim * size};
        const Rows y{reinterpret_cast<uintptr_t>(r.out), r.out_stride * size, x.bytes};
        if (!(x.at == y.at && (x.stride == y.stride || n_tokens == 1)) && !apart(x, y, n_tokens))
            return brc_fail(BRC_ERR_INVALID, "%s: %s and its output overlap without being the same rows", who, s ? "k" : "q");
        if (!other.in) continue;
        const Rows u{reinterpret_cast<uintptr_t>(other.in), other.in_stride * size, (uint64_t)other.heads * head_dim * size};
        const Rows w{reinterpret_cast<uintptr_t>(other.out), other.out_stride * size, u.bytes};
        if (!apart(y, u, n_tokens) || !apart(y, w, n_tokens))
            return brc_fail(BRC_ERR_INVALID, "%s: the output of %s overlaps the rows of %s", who, s ? "k" : "q", s ? "q" : "k");
    }
    if (!positions_dev || !turns_dev) return brc_fail(BRC_ERR_INVALID, "%s: NULL position or frequency pointer", who);
    brc_device_guard guard(device);
    if (!guard.ok) return brc_fail(BRC_ERR_CUDA, "%s: cannot make device %d current", who, device);
    p.positions = positions_dev;
    p.turns = turns_dev;
    p.n_tokens = n_tokens;
    p.head_dim = head_dim;
    p.n_rot = n_rot;
    p.interleaved = layout == BRC_ROPE_INTERLEAVED;
    p.is_signed = is_signed;
    p.factor = factor;
    int sm_count = 0;
    BRC_CUDA(cudaDeviceGetAttribute(&sm_count, cudaDevAttrMultiProcessorCount, device));
    cudaStream_t st = brc_stream(stream);
    if (dtype == BRC_DTYPE_F32) launch<0>(p, rows, total_heads, sm_count, st);
    else if (dtype == BRC_DTYPE_F16) launch<1>(p, rows, total_heads, sm_count, st);
    else launch<2>(p, rows, total_heads, sm_count, st);
    BRC_CUDA(cudaGetLastError());
    return BRC_OK;
}

}  // extern "C"
