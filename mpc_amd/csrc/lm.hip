// Language-model operators on secret shares: lookup in a shared table and its gradient, the global norm of shared
// tensors and clipping, log probabilities of opened logits and their gradient (include/mpcx.h, "language models on
// shares").  Share arithmetic is exact mod 2^64, so sums may be taken in any order.
#include "mpcx_internal.h"
#include "prg_map.h"

namespace {

template <class F> __global__ __launch_bounds__(256) void lm_ew_kernel(u64 n, F f) {
    for (u64 i = (u64)blockIdx.x * 256 + threadIdx.x; i < n; i += (u64)gridDim.x * 256) f(i);
}
template <class F> int lm_ew(mpcx_ctx *ctx, u64 n, F f) {
    if (n == 0) return 0;
    u64 blocks = ceil_div(n, 256);
    if (blocks > MPCX_MAX_GRID) blocks = MPCX_MAX_GRID;
    hipLaunchKernelGGL(lm_ew_kernel<F>, dim3((u32)blocks), dim3(256), 0, ctx->stream, n, f);
    MPCX_LAUNCH_CHECK();
    return 0;
}

// a product of sizes that stays below 2^60 words (every byte count then fits 64 bits)
bool lm_fits(u64 a, u64 b) { return a == 0 || b <= (1ull << 60) / a; }

__device__ inline void lm_atomic_add(u64 *p, u64 v) { atomicAdd((unsigned long long *)p, (unsigned long long)v); }

// two neighbouring words by one 16-byte access; share arrays are 8-byte aligned only, which the hardware takes
typedef u64 u64x2 __attribute__((ext_vector_type(2)));
typedef u64x2 u64x2u __attribute__((aligned(8)));
__device__ inline u64x2 ld2(const u64 *p) { return *(const u64x2u *)p; }
__device__ inline void st2(u64 *p, u64x2 v) { *(u64x2u *)p = v; }

// ---- lookup.  A row is copied by 2^lg lanes (8 .. 256) of a workgroup, 16 bytes of each share per lane and step; the
// four steps of a lane are all requested before the first is used.
constexpr u32 EMB_STEPS = 4;
template <bool TWO>
__global__ __launch_bounds__(256) void embed_kernel(const u64 *__restrict__ T0, const u64 *__restrict__ T1, u64 vocab, u64 dim,
                                                    const i64 *__restrict__ ids, u64 n, u64 scale, int shift,
                                                    u64 *__restrict__ E0, u64 *__restrict__ E1, u32 lg) {
    const u32 lane = threadIdx.x & ((1u << lg) - 1), rows = 256u >> lg;
    const u64 col0 = 2 * (((u64)blockIdx.y * EMB_STEPS << lg) + lane);
    for (u64 t = (u64)blockIdx.x * rows + (threadIdx.x >> lg); t < n; t += (u64)gridDim.x * rows) {
        const u64 v = (u64)ids[t];
        const bool ok = v < vocab;
        const u64 *r0 = T0 + v * dim, *r1 = TWO ? T1 + v * dim : nullptr;
        u64x2 a[EMB_STEPS] = {}, b[EMB_STEPS] = {};
#pragma unroll
        for (u32 u = 0; u < EMB_STEPS; u++) {
            const u64 c = col0 + ((u64)(2 * u) << lg);
            if (!ok || c >= dim) continue;
            if (c + 1 < dim) {
                a[u] = ld2(r0 + c);
                if (TWO) b[u] = ld2(r1 + c);
            } else {
                a[u].x = r0[c];
                if (TWO) b[u].x = r1[c];
            }
        }
#pragma unroll
        for (u32 u = 0; u < EMB_STEPS; u++) {
            const u64 c = col0 + ((u64)(2 * u) << lg);
            if (c >= dim) continue;
            u64x2 x, y;
            if (TWO) {
                x = a[u] * scale, y = b[u] * scale;
            } else {
                x.x = (u64)((i64)(a[u].x * scale) >> shift), x.y = (u64)((i64)(a[u].y * scale) >> shift);
            }
            if (c + 1 < dim) {
                st2(E0 + t * dim + c, x);
                if (TWO) st2(E1 + t * dim + c, y);
            } else {
                E0[t * dim + c] = x.x;
                if (TWO) E1[t * dim + c] = y.x;
            }
        }
    }
}
inline u32 lanes_log2(u64 dim) { // lanes for a row: enough for its 16-byte pieces, 8 .. 256
    u32 lg = 3;
    while (lg < 8 && (2ull << lg) < dim) lg++;
    return lg;
}

// ---- many tensors in one launch.  The tensors of a call are cut into tiles; up to LM_TENSORS descriptors travel in the
// kernel's own arguments, so nothing is copied to the device and a captured call keeps its descriptors.  A workgroup
// finds the tensor of a tile by one comparison per lane and a population count.
constexpr u32 LM_TENSORS = 96;    // descriptors of 40 bytes: the arguments stay below 4 KiB
constexpr u64 LM_TILE = 4096;     // words
// From this many words on party 1's segment of a tensor is one launch that consumes the stream's words where they are
// regenerated (24 bytes of traffic a word); shorter tensors share a launch that reads the words back (40 bytes).
constexpr u64 CLIP_FUSED_WORDS = 1 << 18;
constexpr u32 LM_GRID = 2048;     // eight workgroups of four waves on each of 256 CUs
struct TensorRef {
    const u64 *x0, *x1;
    u64 n, out, tile0; // words, first word in the call's output, first tile
};
struct TensorTable {
    TensorRef t[LM_TENSORS];
    u32 count;
    u64 tiles;
};
__device__ inline u32 tensor_of(const TensorTable &tab, u64 tile) {
    const u32 lane = threadIdx.x & 63;
    const bool a = lane < tab.count && tab.t[lane].tile0 <= tile;
    const bool b = lane + 64 < tab.count && tab.t[lane + 64 < LM_TENSORS ? lane + 64 : 0].tile0 <= tile;
    const u32 k = (u32)(__popcll(__ballot(a)) + __popcll(__ballot(b))) - 1;
    return __builtin_amdgcn_readfirstlane(k);
}

// sum of x0 (x0 + 2 x1) over the tiles of a workgroup -> part[workgroup]
__global__ __launch_bounds__(256) void sqnorm_kernel(TensorTable tab, u64 *__restrict__ part) {
    __shared__ u64 ws[4];
    const u32 tid = threadIdx.x;
    u64 s = 0;
    for (u64 tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x) {
        const u32 k = tensor_of(tab, tile);
        const u64 at = (tile - tab.t[k].tile0) * LM_TILE, n = tab.t[k].n - at;
        const u64 *x0 = tab.t[k].x0 + at, *x1 = tab.t[k].x1 + at;
        if (n >= LM_TILE) {
#pragma unroll
            for (u32 u = 0; u < LM_TILE / 512; u++) {
                const u64x2 a = ld2(x0 + 512 * u + 2 * tid), b = ld2(x1 + 512 * u + 2 * tid);
                const u64x2 q = a * (a + 2 * b);
                s += q.x + q.y;
            }
        } else {
            for (u64 i = tid; i < n; i += 256) s += x0[i] * (x0[i] + 2 * x1[i]);
        }
    }
    for (u32 d = 32; d; d >>= 1) s += __shfl_xor((unsigned long long)s, d);
    if ((tid & 63) == 0) ws[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) part[blockIdx.x] = ws[0] + ws[1] + ws[2] + ws[3];
}
// z = the sum of the partial sums + A[tA] - B[tB] (one word of each of two generator streams)
__global__ __launch_bounds__(256) void sqnorm_join_kernel(const u64 *__restrict__ part, u64 parts, const PrgCk *__restrict__ ckA,
                                                          const PrgCk *__restrict__ ckB, u64 tA, u64 tB, u64 *__restrict__ z) {
    __shared__ u64 ws[4];
    const u32 tid = threadIdx.x;
    u64 s = 0;
    for (u64 i = tid; i < parts; i += 256) s += part[i];
    if (tid == 0 || tid == 64) {
        PrgCursor g;
        g.open(tid ? ckB : ckA, tid ? tB : tA, true);
        const u64 w = g.next();
        s += tid ? 0 - w : w;
    }
    for (u32 d = 32; d; d >>= 1) s += __shfl_xor((unsigned long long)s, d);
    if ((tid & 63) == 0) ws[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) *z = ws[0] + ws[1] + ws[2] + ws[3];
}

// f to the nearest word, ties to even; beyond the range its ends, 0 for what is no number
__device__ inline i64 nearest_word(float f) {
    const float r = rintf(f);
    if (r >= 9223372036854775808.0f) return INT64_MAX;
    if (r <= -9223372036854775808.0f) return INT64_MIN;
    return r == r ? (i64)r : 0;
}

// the largest c in [0, 2^f] with c^2 S <= R^2
__device__ inline u64 clip_factor(u64 S, u64 R, int f) {
    const u64 one = 1ull << f;
    if (S == 0) return one;
    const double est = (double)R / sqrt((double)S);
    u64 c = est >= (double)one ? one : (u64)est;
    typedef unsigned __int128 u128;
    const u128 R2 = (u128)R * R;
    while (c > 0 && (u128)(c * c) * S > R2) c--;
    while (c < one && (u128)((c + 1) * (c + 1)) * S <= R2) c++;
    return c;
}

struct ClipArgs {
    const u64 *za, *zb, *zc; // the shares of the squared norm
    u64 R;
    int number;
    __device__ u64 factor() const { return clip_factor(*za + *zb + *zc, R, number); }
};
// SUM = false: y = (c x0) >> number (party 0; every workgroup forms the factor, which saves a launch); SUM = true: y =
// ((c (x0 + x1)) >> number) - y, where y holds the words of the stream (party 1; the factor has been written)
template <bool SUM>
__global__ __launch_bounds__(256) void clip_kernel(TensorTable tab, ClipArgs A, i64 *__restrict__ coef, u64 *__restrict__ Y) {
    const u32 tid = threadIdx.x;
    const u64 c = SUM ? (u64)*coef : A.factor();
    if (!SUM && blockIdx.x == 0 && tid == 0) *coef = (i64)c;
    const int sh = A.number;
    for (u64 tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x) {
        const u32 k = tensor_of(tab, tile);
        const u64 at = (tile - tab.t[k].tile0) * LM_TILE, n = tab.t[k].n - at;
        const u64 *x0 = tab.t[k].x0 + at, *x1 = SUM ? tab.t[k].x1 + at : nullptr;
        u64 *y = Y + tab.t[k].out + at;
        if (n >= LM_TILE) {
#pragma unroll
            for (u32 u = 0; u < LM_TILE / 512; u++) {
                const u32 i = 512 * u + 2 * tid;
                u64x2 a = ld2(x0 + i);
                if (SUM) a += ld2(x1 + i);
                a *= c;
                u64x2 r = {(u64)((i64)a.x >> sh), (u64)((i64)a.y >> sh)};
                if (SUM) r -= ld2(y + i);
                st2(y + i, r);
            }
        } else {
            for (u64 i = tid; i < n; i += 256) {
                const u64 r = (u64)((i64)((SUM ? x0[i] + x1[i] : x0[i]) * c) >> sh);
                y[i] = SUM ? r - y[i] : r;
            }
        }
    }
}
__global__ void clip_factor_kernel(ClipArgs A, i64 *coef) { *coef = (i64)A.factor(); }

struct LogitIn {
    const u64 *a, *b, *c;
    __device__ i64 at(u64 i) const {
        u64 x = a[i];
        if (b) x += b[i];
        if (c) x += c[i];
        return (i64)x;
    }
};

__global__ __launch_bounds__(256) void logprobs_kernel(LogitIn in, u64 vocab, float unit, const i64 *__restrict__ ids,
                                                       u64 per_row, u32 top, float *__restrict__ logp,
                                                       float *__restrict__ entropy, i64 *__restrict__ top_ids,
                                                       float *__restrict__ top_logp, i64 *__restrict__ row_max,
                                                       float *__restrict__ log_sum) {
    __shared__ i64 sv[256];
    __shared__ u64 si[256];
    __shared__ float ss[256], st[256];
    const u32 tid = threadIdx.x;
    const u64 row = blockIdx.x, base = row * vocab;
    // the best (value, index) below (pv, pi) in the order value descending, index ascending
    auto best_below = [&](bool first, i64 pv, u64 pi) {
        i64 bv = INT64_MIN;
        u64 bi = ~0ull;
        for (u64 j = tid; j < vocab; j += 256) {
            const i64 x = in.at(base + j);
            if (!first && !(x < pv || (x == pv && j > pi))) continue;
            if (bi == ~0ull || x > bv) bv = x, bi = j;
        }
        __syncthreads();
        sv[tid] = bv, si[tid] = bi;
        __syncthreads();
        for (u32 s = 128; s; s >>= 1) {
            if (tid < s) {
                const i64 ov = sv[tid + s];
                const u64 oi = si[tid + s];
                if (oi != ~0ull && (si[tid] == ~0ull || ov > sv[tid] || (ov == sv[tid] && oi < si[tid]))) sv[tid] = ov, si[tid] = oi;
            }
            __syncthreads();
        }
    };
    best_below(true, 0, 0);
    const i64 m = sv[0];
    float S = 0, T = 0;
    for (u64 j = tid; j < vocab; j += 256) {
        const float d = (float)((u64)m - (u64)in.at(base + j)) * unit, e = expf(-d);
        S += e, T += d * e;
    }
    ss[tid] = S, st[tid] = T;
    __syncthreads();
    for (u32 s = 128; s; s >>= 1) {
        if (tid < s) ss[tid] += ss[tid + s], st[tid] += st[tid + s];
        __syncthreads();
    }
    const float ls = logf(ss[0]);
    if (tid == 0) {
        if (entropy) entropy[row] = ls + st[0] / ss[0];
        if (row_max) row_max[row] = m;
        if (log_sum) log_sum[row] = ls;
    }
    for (u64 t = tid; t < per_row; t += 256) {
        const i64 id = ids[row * per_row + t];
        const bool in_range = id >= 0 && (u64)id < vocab;
        logp[row * per_row + t] = in_range ? -((float)((u64)m - (u64)in.at(base + (u64)id)) * unit + ls) : 0.0f;
    }
    i64 pv = 0;
    u64 pi = 0;
    for (u32 k = 0; k < top; k++) {
        best_below(k == 0, pv, pi);
        pv = sv[0], pi = si[0];
        if (tid == 0) {
            top_ids[row * top + k] = (i64)pi;
            top_logp[row * top + k] = -((float)((u64)m - (u64)pv) * unit + ls);
        }
    }
}

__global__ __launch_bounds__(256) void logprobs_grad_kernel(LogitIn in, u64 vocab, float unit, const i64 *__restrict__ ids,
                                                            u64 per_row, const float *__restrict__ d_logp,
                                                            const float *__restrict__ d_entropy,
                                                            const i64 *__restrict__ row_max, const float *__restrict__ log_sum,
                                                            const float *__restrict__ entropy, float *__restrict__ grad,
                                                            i64 *__restrict__ grad_words, float words) {
    const u64 row = blockIdx.x, base = row * vocab;
    const i64 m = row_max[row];
    const float ls = log_sum[row];
    const float h = d_entropy ? d_entropy[row] : 0.0f, H = d_entropy ? entropy[row] : 0.0f;
    float w = 0;
    for (u64 t = 0; t < per_row; t++) {
        const i64 id = ids[row * per_row + t];
        if (id >= 0 && (u64)id < vocab) w += d_logp[row * per_row + t];
    }
    for (u64 j = threadIdx.x; j < vocab; j += 256) {
        const float lp = -((float)((u64)m - (u64)in.at(base + j)) * unit + ls);
        const float p = expf(lp);
        float g = 0;
        for (u64 t = 0; t < per_row; t++)
            if (ids[row * per_row + t] == (i64)j) g += d_logp[row * per_row + t];
        g -= p * w;
        if (d_entropy) g -= h * p * (lp + H);
        if (grad) grad[base + j] = g;
        if (grad_words) grad_words[base + j] = nearest_word(g * words);
    }
}

} // namespace

extern "C" {

int mpcx_ring_embed(mpcx_ctx *ctx, const int64_t *T0, const int64_t *T1, uint64_t vocab, uint64_t dim, const int64_t *ids,
                    uint64_t n, int64_t scale, int shift, int64_t *E0, int64_t *E1) {
    MPCX_REQUIRE(lm_fits(vocab, dim) && lm_fits(n, dim), "mpcx_ring_embed: sizes too large");
    MPCX_REQUIRE(shift >= 0 && shift < 64, "mpcx_ring_embed: shift %d out of range", shift);
    MPCX_REQUIRE((T1 == nullptr) == (E1 == nullptr), "mpcx_ring_embed: the second share needs a table and an output");
    MPCX_REQUIRE(!(shift && (T1 || E1)), "mpcx_ring_embed: replicated shares are not truncated locally (shift must be 0)");
    if (n == 0 || dim == 0) return 0;
    MPCX_REQUIRE(ids && E0 && (T0 || vocab == 0), "mpcx_ring_embed: NULL pointer");
    MPCX_REQUIRE(ctx, "mpcx_ring_embed: the context is NULL");
    const u32 lg = lanes_log2(dim);
    const u64 slices = ceil_div(dim, 2 * EMB_STEPS << lg);
    MPCX_REQUIRE(slices < 65536, "mpcx_ring_embed: rows of %llu words", (unsigned long long)dim);
    u64 blocks = ceil_div(n, 256u >> lg);
    if (blocks > MPCX_MAX_GRID) blocks = MPCX_MAX_GRID;
    const dim3 grid((u32)blocks, (u32)slices), block(256);
    if (T1)
        hipLaunchKernelGGL(embed_kernel<true>, grid, block, 0, ctx->stream, (const u64 *)T0, (const u64 *)T1, vocab, dim, ids, n,
                           (u64)scale, shift, (u64 *)E0, (u64 *)E1, lg);
    else
        hipLaunchKernelGGL(embed_kernel<false>, grid, block, 0, ctx->stream, (const u64 *)T0, (const u64 *)nullptr, vocab, dim, ids,
                           n, (u64)scale, shift, (u64 *)E0, (u64 *)nullptr, lg);
    MPCX_LAUNCH_CHECK();
    return 0;
}

uint64_t mpcx_ring_embed_grad_scratch(uint64_t n, uint64_t vocab, uint64_t dim) { return 2 * 8 * vocab * dim + 8; }
int mpcx_ring_embed_grad(mpcx_ctx *ctx, const int64_t *G0, const int64_t *G1, const int64_t *ids, uint64_t n, uint64_t vocab,
                         uint64_t dim, int64_t scale, int shift, int accumulate, void *scratch, int64_t *dT0, int64_t *dT1) {
    MPCX_REQUIRE(lm_fits(vocab, dim) && lm_fits(n, dim), "mpcx_ring_embed_grad: sizes too large");
    MPCX_REQUIRE(vocab < (1ull << 31) && n < (1ull << 31), "mpcx_ring_embed_grad: sizes too large");
    MPCX_REQUIRE(shift >= 0 && shift < 64, "mpcx_ring_embed_grad: shift %d out of range", shift);
    MPCX_REQUIRE((G1 == nullptr) == (dT1 == nullptr) || n == 0, "mpcx_ring_embed_grad: the second share needs a gradient and an output");
    MPCX_REQUIRE(!(shift && (G1 || dT1)), "mpcx_ring_embed_grad: replicated shares are not truncated locally (shift must be 0)");
    if (vocab == 0 || dim == 0) return 0;
    MPCX_REQUIRE(dT0 && scratch && (n == 0 || (ids && G0)), "mpcx_ring_embed_grad: NULL pointer");
    MPCX_REQUIRE(ctx, "mpcx_ring_embed_grad: the context is NULL");
    u64 *s0 = (u64 *)scratch, *s1 = s0 + vocab * dim;
    MPCX_TRY(lm_ew(ctx, vocab * dim, [=] __device__(u64 i) { s0[i] = 0, s1[i] = 0; }));
    MPCX_TRY(lm_ew(ctx, n * dim, [=] __device__(u64 i) {
        const u64 t = i / dim, j = i % dim, v = (u64)ids[t];
        if (v >= vocab) return;
        lm_atomic_add(s0 + v * dim + j, (u64)G0[i]);
        if (G1) lm_atomic_add(s1 + v * dim + j, (u64)G1[i]);
    }));
    return lm_ew(ctx, vocab * dim, [=] __device__(u64 i) {
        dT0[i] = (i64)((accumulate ? (u64)dT0[i] : 0) + (u64)((i64)(s0[i] * (u64)scale) >> shift));
        if (dT1) dT1[i] = (i64)((accumulate ? (u64)dT1[i] : 0) + s1[i] * (u64)scale);
    });
}

// the next tensors of a call, from tensor `i` on, as one launch's table; advances i and out
static TensorTable tensor_table(const int64_t *const *X0, const int64_t *const *X1, const uint64_t *lens, u64 count, u64 limit,
                                u64 &i, u64 &out) {
    TensorTable tab;
    tab.count = 0, tab.tiles = 0;
    for (; i < count && tab.count < LM_TENSORS && lens[i] < limit; i++) {
        if (lens[i] == 0) continue;
        tab.t[tab.count++] = TensorRef{X0 ? (const u64 *)X0[i] : nullptr, X1 ? (const u64 *)X1[i] : nullptr, lens[i], out, tab.tiles};
        tab.tiles += ceil_div(lens[i], LM_TILE);
        out += lens[i];
    }
    return tab;
}
static u32 tensor_grid(const TensorTable &tab) { return (u32)(tab.tiles < LM_GRID ? tab.tiles : LM_GRID); }

uint64_t mpcx_aby3_sqnorm_scratch(uint64_t count) { return (ceil_div(count, LM_TENSORS) * LM_GRID + 1) * 8; }
int mpcx_aby3_sqnorm_local(mpcx_ctx *ctx, const int64_t *const *X0, const int64_t *const *X1, const uint64_t *lens,
                           uint64_t count, uint64_t seed_next, uint64_t pop_next, uint64_t seed_prev, uint64_t pop_prev,
                           void *scratch, int64_t *z0) {
    MPCX_REQUIRE(z0 && scratch && (count == 0 || (X0 && X1 && lens)), "mpcx_aby3_sqnorm_local: NULL pointer");
    for (u64 i = 0; i < count; i++) {
        MPCX_REQUIRE(lens[i] < (1ull << 56), "mpcx_aby3_sqnorm_local: tensor %llu is too long", (unsigned long long)i);
        MPCX_REQUIRE(lens[i] == 0 || (X0[i] && X1[i]), "mpcx_aby3_sqnorm_local: tensor %llu: NULL pointer", (unsigned long long)i);
    }
    MPCX_REQUIRE(ctx, "mpcx_aby3_sqnorm_local: the context is NULL");
    const PrgCk *ckA, *ckB;
    const u64 tA = PRG_POP_T0 + pop_next, tB = PRG_POP_T0 + pop_prev;
    MPCX_TRY(mpcx_prg_table(ctx, seed_next, 0, tA + 1, &ckA));
    MPCX_TRY(mpcx_prg_table(ctx, seed_prev, 0, tB + 1, &ckB));
    u64 *part = (u64 *)scratch, parts = 0, out = 0;
    for (u64 i = 0; i < count;) {
        const TensorTable tab = tensor_table(X0, X1, lens, count, ~0ull, i, out);
        if (tab.count == 0) continue;
        const u32 grid = tensor_grid(tab);
        hipLaunchKernelGGL(sqnorm_kernel, dim3(grid), dim3(256), 0, ctx->stream, tab, part + parts);
        MPCX_LAUNCH_CHECK();
        parts += grid;
    }
    hipLaunchKernelGGL(sqnorm_join_kernel, dim3(1), dim3(256), 0, ctx->stream, part, parts, ckA, ckB, tA, tB, (u64 *)z0);
    MPCX_LAUNCH_CHECK();
    return 0;
}

int mpcx_aby3_clip_local(mpcx_ctx *ctx, int party, const int64_t *const *X0, const int64_t *const *X1, const uint64_t *lens,
                         uint64_t count, const int64_t *z_prev, const int64_t *z0, const int64_t *z1, uint64_t max_norm,
                         int number, uint64_t seed12, uint64_t pop12, int64_t *Y0, int64_t *coef) {
    MPCX_REQUIRE(party >= 0 && party <= 2, "mpcx_aby3_clip_local: party %d", party);
    MPCX_REQUIRE(number >= 0 && number <= 31, "mpcx_aby3_clip_local: %d fractional bits", number);
    MPCX_REQUIRE(max_norm < (1ull << (62 - number)), "mpcx_aby3_clip_local: max_norm does not fit %d fractional bits", number);
    MPCX_REQUIRE(z_prev && z0 && z1 && coef && (count == 0 || lens), "mpcx_aby3_clip_local: NULL pointer");
    const u64 R = max_norm << number;
    u64 at = 0;
    for (u64 i = 0; i < count; i++) {
        MPCX_REQUIRE(lens[i] < (1ull << 56) && at + lens[i] < (1ull << 57), "mpcx_aby3_clip_local: tensor %llu is too long", (unsigned long long)i);
        MPCX_REQUIRE(lens[i] == 0 || (Y0 && (party == 2 || (X0 && X0[i])) && (party != 1 || (X1 && X1[i]))),
                     "mpcx_aby3_clip_local: tensor %llu: NULL pointer", (unsigned long long)i);
        at += lens[i];
    }
    MPCX_REQUIRE(ctx, "mpcx_aby3_clip_local: the context is NULL");
    const ClipArgs A{(const u64 *)z_prev, (const u64 *)z0, (const u64 *)z1, R, number};
    if (party || at == 0) {
        hipLaunchKernelGGL(clip_factor_kernel, dim3(1), dim3(1), 0, ctx->stream, A, coef);
        MPCX_LAUNCH_CHECK();
    }
    u64 *Y = (u64 *)Y0;
    if (party == 2) return at ? prg_fill_words(ctx, seed12, 0, PRG_POP_T0 + pop12, at, 1, Y0, nullptr) : 0;
    u64 out = 0;
    for (u64 i = 0; i < count;) {
        if (party == 1 && lens[i] >= CLIP_FUSED_WORDS) {
            const u64 *x0 = (const u64 *)X0[i], *x1 = (const u64 *)X1[i];
            u64 *y = Y + out;
            MPCX_TRY(prg_map1(ctx, seed12, PRG_POP_T0 + pop12 + out, lens[i], [=] __device__(u64 j, u64 w) {
                y[j] = (u64)((i64)((x0[j] + x1[j]) * (u64)*coef) >> number) - w;
            }));
            out += lens[i++];
            continue;
        }
        const u64 first = out;
        const TensorTable tab = tensor_table(X0, party == 1 ? X1 : nullptr, lens, count, party == 1 ? CLIP_FUSED_WORDS : ~0ull, i, out);
        if (tab.count == 0) continue;
        if (party == 1) {
            MPCX_TRY(prg_fill_words(ctx, seed12, 0, PRG_POP_T0 + pop12 + first, out - first, 1, (i64 *)Y + first, nullptr));
            hipLaunchKernelGGL(clip_kernel<true>, dim3(tensor_grid(tab)), dim3(256), 0, ctx->stream, tab, A, coef, Y);
        } else {
            hipLaunchKernelGGL(clip_kernel<false>, dim3(tensor_grid(tab)), dim3(256), 0, ctx->stream, tab, A, coef, Y);
        }
        MPCX_LAUNCH_CHECK();
    }
    return 0;
}

uint64_t mpcx_reveal_logprobs_scratch(uint64_t rows, uint64_t vocab, uint64_t top) { return 8; }
int mpcx_reveal_logprobs(mpcx_ctx *ctx, const int64_t *a, const int64_t *b, const int64_t *c, uint64_t rows, uint64_t vocab,
                         int frac, const int64_t *ids, uint64_t per_row, uint64_t top, void *scratch, float *logp,
                         float *entropy, int64_t *top_ids, float *top_logp, int64_t *row_max, float *log_sum) {
    MPCX_REQUIRE(vocab >= 1 && vocab < (1ull << 31), "mpcx_reveal_logprobs: vocabulary of %llu", (unsigned long long)vocab);
    MPCX_REQUIRE(rows < (1ull << 31) && lm_fits(rows, per_row), "mpcx_reveal_logprobs: sizes too large");
    MPCX_REQUIRE(frac >= 0 && frac <= 62, "mpcx_reveal_logprobs: %d fractional bits", frac);
    MPCX_REQUIRE(top <= 32 && top <= vocab, "mpcx_reveal_logprobs: %llu alternatives", (unsigned long long)top);
    MPCX_REQUIRE(b || !c, "mpcx_reveal_logprobs: the third share without the second");
    if (rows == 0) return 0;
    MPCX_REQUIRE(a && scratch && (per_row == 0 || (ids && logp)) && (top == 0 || (top_ids && top_logp)),
                 "mpcx_reveal_logprobs: NULL pointer");
    MPCX_REQUIRE(ctx, "mpcx_reveal_logprobs: the context is NULL");
    const LogitIn in{(const u64 *)a, (const u64 *)b, (const u64 *)c};
    hipLaunchKernelGGL(logprobs_kernel, dim3((u32)rows), dim3(256), 0, ctx->stream, in, vocab, ldexpf(1.0f, -frac), ids,
                       per_row, (u32)top, logp, entropy, top_ids, top_logp, row_max, log_sum);
    MPCX_LAUNCH_CHECK();
    return 0;
}

int mpcx_reveal_logprobs_grad(mpcx_ctx *ctx, const int64_t *a, const int64_t *b, const int64_t *c, uint64_t rows,
                              uint64_t vocab, int frac, const int64_t *ids, uint64_t per_row, const float *d_logp,
                              const float *d_entropy, const int64_t *row_max, const float *log_sum, const float *entropy,
                              float *grad, int64_t *grad_words, int grad_frac) {
    MPCX_REQUIRE(vocab >= 1 && vocab < (1ull << 31), "mpcx_reveal_logprobs_grad: vocabulary of %llu", (unsigned long long)vocab);
    MPCX_REQUIRE(rows < (1ull << 31) && lm_fits(rows, per_row), "mpcx_reveal_logprobs_grad: sizes too large");
    MPCX_REQUIRE(frac >= 0 && frac <= 62, "mpcx_reveal_logprobs_grad: %d fractional bits", frac);
    MPCX_REQUIRE(!grad_words || (grad_frac >= 0 && grad_frac <= 62), "mpcx_reveal_logprobs_grad: %d fractional bits", grad_frac);
    MPCX_REQUIRE(b || !c, "mpcx_reveal_logprobs_grad: the third share without the second");
    if (rows == 0) return 0;
    MPCX_REQUIRE(a && row_max && log_sum && (grad || grad_words) && (per_row == 0 || (ids && d_logp)) && (!d_entropy || entropy),
                 "mpcx_reveal_logprobs_grad: NULL pointer");
    MPCX_REQUIRE(ctx, "mpcx_reveal_logprobs_grad: the context is NULL");
    const LogitIn in{(const u64 *)a, (const u64 *)b, (const u64 *)c};
    hipLaunchKernelGGL(logprobs_grad_kernel, dim3((u32)rows), dim3(256), 0, ctx->stream, in, vocab, ldexpf(1.0f, -frac), ids,
                       per_row, d_logp, d_entropy, row_max, log_sum, entropy, grad, grad_words, ldexpf(1.0f, grad_frac));
    MPCX_LAUNCH_CHECK();
    return 0;
}

} // extern "C"
