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

// ---- opened logits.  A word x = a + b + c stands for the logit x 2^-frac; distances from a maximum are differences of
// words, exact before their one conversion to a float.
template <int SH> struct LogitIn {
    const u64 *a, *b, *c;
    __device__ i64 at(u64 i) const {
        u64 x = a[i];
        if (SH > 1) x += b[i];
        if (SH > 2) x += c[i];
        return (i64)x;
    }
    __device__ u64x2 at2(u64 i) const {
        u64x2 x = ld2(a + i);
        if (SH > 1) x += ld2(b + i);
        if (SH > 2) x += ld2(c + i);
        return x;
    }
};
// hi - lo >= 0 as a float, off by less than two half steps
__device__ inline float word_dist(i64 hi, i64 lo) {
    const u64 d = (u64)hi - (u64)lo;
    return fmaf((float)(u32)(d >> 32), 4294967296.0f, (float)(u32)d);
}
__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); } // v_exp_f32, within one step

__device__ inline i64 lane_word(i64 v, u32 lane) {
    const u32 lo = (u32)__builtin_amdgcn_readlane((int)(u32)v, (int)lane), hi = (u32)__builtin_amdgcn_readlane((int)((u64)v >> 32), (int)lane);
    return (i64)((u64)hi << 32 | lo);
}
__device__ inline i64 wave_max(i64 v) {
    for (u32 d = 32; d; d >>= 1) {
        const i64 o = (i64)__shfl_xor((long long)v, (int)d);
        v = o > v ? o : v;
    }
    return v;
}

// The likeliest `top` <= 32 entries a wavefront has seen, best first: entry l in lane l, in the order value descending,
// index ascending (all entries differ).  (tv, ti) is the last of them, the border that a new one has to beat.
struct TopEntry {
    i64 v;
    u32 i, pad;
};
__device__ inline bool top_better(i64 av, u32 ai, i64 bv, u32 bi) { return av > bv || (av == bv && ai < bi); }
constexpr u32 TOP_NONE = ~0u; // the index of an entry that is not there (with the lowest value: behind all others)
struct WaveTop {
    i64 v = INT64_MIN, tv = INT64_MIN;
    u32 i = TOP_NONE, ti = TOP_NONE;
    __device__ void border(u32 top) {
        tv = lane_word(v, top - 1);
        ti = (u32)__builtin_amdgcn_readlane((int)i, (int)top - 1);
    }
    // one candidate per lane; those that beat the border go in one after the other
    __device__ void insert(u32 top, bool valid, i64 x, u32 idx) {
        const u32 lane = threadIdx.x & 63;
        u64 mask = __ballot(valid && top_better(x, idx, tv, ti));
        while (mask) {
            const u32 src = (u32)__builtin_ctzll(mask);
            const i64 cv = lane_word(x, src);
            const u32 ci = (u32)__builtin_amdgcn_readlane((int)idx, (int)src);
            const u32 pos = (u32)__popcll(__ballot(top_better(v, i, cv, ci)));
            const i64 uv = (i64)__shfl_up((long long)v, 1);
            const u32 ui = (u32)__shfl_up((int)i, 1);
            if (lane > pos) v = uv, i = ui;
            if (lane == pos) v = cv, i = ci;
            border(top);
            mask &= mask - 1;
            mask &= __ballot(top_better(x, idx, tv, ti));
        }
    }
};
// The first tile of a wavefront: N candidates per lane at once.  A distance D is found by bisection such that at least
// `top` lanes hold something within D of the maximum; what lies within D (rarely more than a few above `top`) is
// gathered in LDS and sorted by counting, for each, how many are better.  Where more than 64 lie within D (many equal
// words), or lanes are few, the candidates are inserted one by one.
template <u32 N>
__device__ inline void top_first(WaveTop &t, u32 top, const i64 (&x)[N], const u32 (&idx)[N], const bool (&valid)[N], i64 lane_max,
                                 bool lane_any, TopEntry *buf) {
    const u32 lane = threadIdx.x & 63;
    const i64 m = wave_max(lane_any ? lane_max : INT64_MIN);
    const float near = lane_any ? word_dist(m, lane_max) : INFINITY;
    float lo = 0, hi = near;
    if ((u32)__popcll(__ballot(lane_any)) < top) {
        hi = INFINITY;
    } else {
        if (!lane_any) hi = 0;
        for (u32 d = 32; d; d >>= 1) hi = fmaxf(hi, __shfl_xor(hi, (int)d));
        for (u32 r = 0; r < 12; r++) {
            const float mid = 0.5f * (lo + hi);
            if ((u32)__popcll(__ballot(near <= mid)) >= top)
                hi = mid;
            else
                lo = mid;
        }
    }
    u32 count = 0;
    u32 slot[N];
#pragma unroll
    for (u32 k = 0; k < N; k++) {
        const u64 b = __ballot(valid[k] && word_dist(m, x[k]) <= hi);
        slot[k] = ((b >> lane) & 1) ? count + (u32)__popcll(b & ((1ull << lane) - 1)) : TOP_NONE;
        count += (u32)__popcll(b);
    }
    if (count > 64) {
#pragma unroll
        for (u32 k = 0; k < N; k++) t.insert(top, valid[k], x[k], idx[k]);
        return;
    }
#pragma unroll
    for (u32 k = 0; k < N; k++)
        if (slot[k] != TOP_NONE) buf[slot[k]] = TopEntry{x[k], idx[k], 0};
    prg_wave_sync();
    const i64 v = lane < count ? buf[lane].v : INT64_MIN;
    const u32 i = lane < count ? buf[lane].i : TOP_NONE;
    u32 rank = 0;
    for (u32 k = 0; k < count; k++) rank += top_better(buf[k].v, buf[k].i, v, i);
    prg_wave_sync();
    if (lane < count) buf[rank] = TopEntry{v, i, 0};
    prg_wave_sync();
    if (lane < count && lane < top) t.v = buf[lane].v, t.i = buf[lane].i;
    prg_wave_sync();
    t.border(top);
}
// The lists of the W wavefronts of a workgroup (in `lists`, `top` entries each) -> out[0 .. top): every entry counts the
// better ones.  Entries that are not there stay behind the rest.  All threads call it; ends with a barrier.
template <u32 W> __device__ inline void top_merge(const TopEntry *lists, TopEntry *out, u32 top) {
    const u32 tid = threadIdx.x, n = W * top;
    if (tid < top) out[tid] = TopEntry{INT64_MIN, TOP_NONE, 0};
    __syncthreads();
    if (tid < n) {
        const TopEntry e = lists[tid];
        u32 rank = 0;
        for (u32 k = 0; k < n; k++) rank += top_better(lists[k].v, lists[k].i, e.v, e.i);
        if (rank < top && e.i != TOP_NONE) out[rank] = e;
    }
    __syncthreads();
}

// max, sum of 2^-d and sum of d 2^-d, d = (max - x) in units of 1 / log2(e) 2^-frac, over some of a row's words
struct RowSums {
    i64 m = INT64_MIN;
    float S = 0, T = 0;
    __device__ void move_to(i64 to, float unit2) { // the same sums relative to a larger maximum
        const float d = word_dist(to, m) * unit2, f = exp2_fast(-d);
        T = (T + d * S) * f, S *= f, m = to;
    }
    __device__ void wave_join(float unit2) {
        move_to(wave_max(m), unit2);
        for (u32 d = 32; d; d >>= 1) S += __shfl_xor(S, (int)d), T += __shfl_xor(T, (int)d);
    }
};
struct RowPart {
    i64 m;
    float S, T;
};

struct LogprobArgs {
    u64 rows, vocab;
    u64 chunk;  // words of a row that one group of wavefronts reads
    u32 splits; // groups per row
    u32 top;
    float unit, unit2; // 2^-frac, 2^-frac log2(e)
    const i64 *ids;
    u64 per_row;
    float *logp, *entropy;
    i64 *top_ids;
    float *top_logp;
    i64 *row_max;
    float *log_sum;
    RowPart *parts;  // splits > 1: rows x splits, then
    TopEntry *lists; // rows x splits x top
};
// a row's outputs, by `n` threads (thread `t` of them); list: the row's sorted entries
template <int SH>
__device__ inline void logprobs_finish(const LogitIn<SH> &in, const LogprobArgs &A, u64 row, RowSums s, const TopEntry *list, u32 t, u32 n) {
    const float ls = logf(s.S);
    if (t == 0) {
        if (A.entropy) A.entropy[row] = ls + s.T / s.S * 0.69314718f;
        if (A.row_max) A.row_max[row] = s.m;
        if (A.log_sum) A.log_sum[row] = ls;
    }
    for (u64 k = t; k < A.per_row; k += n) {
        const u64 id = (u64)A.ids[row * A.per_row + k];
        A.logp[row * A.per_row + k] = id < A.vocab ? -(word_dist(s.m, in.at(row * A.vocab + id)) * A.unit + ls) : 0.0f;
    }
    if (t < A.top) {
        A.top_ids[row * A.top + t] = (i64)list[t].i;
        A.top_logp[row * A.top + t] = -(word_dist(s.m, list[t].v) * A.unit + ls);
    }
}

// W wavefronts of a workgroup of four read `chunk` words of a row, in tiles of 64 x 8 words each.  A lane keeps its own
// maximum and sums and moves them when a tile raises its maximum; nothing is exchanged between lanes before the end but
// the ballots that look for new entries of the top list.
template <u32 W, int SH> __global__ __launch_bounds__(256) void logprobs_kernel(LogitIn<SH> in, LogprobArgs A) {
    constexpr u32 U = 4, N = 2 * U, TILE = 64 * N;
    __shared__ TopEntry buf[4][64];
    __shared__ TopEntry merged[32];
    __shared__ RowPart ws[4];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const u64 group = W == 1 ? (u64)blockIdx.x * 4 + wave : blockIdx.x;
    const u64 row = group / A.splits, split = group % A.splits;
    if (W == 1 && row >= A.rows) return; // a wavefront of its own: no barrier follows
    const u64 base = row * A.vocab, j0 = split * A.chunk, j1 = j0 + A.chunk < A.vocab ? j0 + A.chunk : A.vocab;
    RowSums s;
    WaveTop top;
    bool first = true;
    for (u64 tile = j0 + (W == 1 ? 0 : wave) * TILE; tile < j1; tile += W * TILE) {
        i64 x[N];
        u32 idx[N];
        bool valid[N];
        if (tile + TILE <= j1) {
            u64x2 p[U];
#pragma unroll
            for (u32 u = 0; u < U; u++) p[u] = in.at2(base + tile + 128 * u + 2 * lane);
#pragma unroll
            for (u32 k = 0; k < N; k++) x[k] = (i64)(k & 1 ? p[k / 2].y : p[k / 2].x), valid[k] = true;
        } else {
#pragma unroll
            for (u32 k = 0; k < N; k++) {
                const u64 j = tile + 128 * (k / 2) + 2 * lane + (k & 1);
                valid[k] = j < j1;
                x[k] = valid[k] ? in.at(base + j) : INT64_MIN;
            }
        }
        i64 m = x[0];
        bool any = valid[0];
#pragma unroll
        for (u32 k = 0; k < N; k++) {
            m = x[k] > m ? x[k] : m;
            any |= valid[k];
            idx[k] = (u32)(tile + 128 * (k / 2) + 2 * lane + (k & 1));
        }
        if (m > s.m) s.move_to(m, A.unit2);
#pragma unroll
        for (u32 k = 0; k < N; k++) {
            const float d = word_dist(s.m, x[k]) * A.unit2, e = valid[k] ? exp2_fast(-d) : 0.0f;
            s.S += e, s.T = fmaf(d, e, s.T);
        }
        if (A.top) {
            if (first) {
                top_first<N>(top, A.top, x, idx, valid, m, any, buf[wave]);
                first = false;
            } else if (__ballot(m >= top.tv)) {
#pragma unroll
                for (u32 k = 0; k < N; k++) top.insert(A.top, valid[k], x[k], idx[k]);
            }
        }
    }
    s.wave_join(A.unit2);
    if (W == 1) {
        if (lane < A.top) buf[wave][lane] = TopEntry{top.v, top.i, 0};
        prg_wave_sync();
        logprobs_finish(in, A, row, s, buf[wave], lane, 64);
        return;
    }
    if (lane == 0) ws[wave] = RowPart{s.m, s.S, s.T};
    __syncthreads(); // every wavefront has left its own part of buf
    TopEntry *lists = &buf[0][0];
    if (lane < A.top) lists[wave * A.top + lane] = TopEntry{top.v, top.i, 0};
    for (u32 w = 0; w < 4; w++) {
        RowSums o;
        o.m = ws[w].m, o.S = ws[w].S, o.T = ws[w].T;
        if (w == 0) {
            s = o;
            continue;
        }
        if (o.m > s.m) s.move_to(o.m, A.unit2);
        else o.move_to(s.m, A.unit2);
        s.S += o.S, s.T += o.T;
    }
    __syncthreads();
    if (A.top) top_merge<4>(lists, merged, A.top);
    if (A.splits == 1) {
        logprobs_finish(in, A, row, s, merged, tid, 256);
    } else {
        if (tid == 0) A.parts[group] = RowPart{s.m, s.S, s.T};
        if (tid < A.top) A.lists[group * A.top + tid] = merged[tid];
    }
}
// joins the parts of a row: one workgroup per row
template <int SH> __global__ __launch_bounds__(256) void logprobs_join_kernel(LogitIn<SH> in, LogprobArgs A) {
    constexpr u32 N = 8;
    __shared__ TopEntry buf[4][64];
    __shared__ TopEntry merged[32];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const u64 row = blockIdx.x;
    const RowPart *parts = A.parts + row * A.splits;
    RowSums s;
    for (u32 k = lane; k < A.splits; k += 64) { // every wavefront for itself
        RowSums o;
        o.m = parts[k].m, o.S = parts[k].S, o.T = parts[k].T;
        if (o.m > s.m) s.move_to(o.m, A.unit2);
        else o.move_to(s.m, A.unit2);
        s.S += o.S, s.T += o.T;
    }
    s.wave_join(A.unit2);
    if (A.top) {
        const TopEntry *lists = A.lists + row * A.splits * A.top;
        const u32 n = A.splits * A.top;
        WaveTop top;
        bool first = true;
        for (u32 tile = wave * 64 * N; tile < n; tile += 4 * 64 * N) {
            i64 x[N], m = INT64_MIN;
            u32 idx[N];
            bool valid[N], any = false;
#pragma unroll
            for (u32 k = 0; k < N; k++) {
                const u32 j = tile + 64 * k + lane;
                const TopEntry e = j < n ? lists[j] : TopEntry{INT64_MIN, TOP_NONE, 0};
                x[k] = e.v, idx[k] = e.i, valid[k] = e.i != TOP_NONE, any |= valid[k];
                m = e.v > m ? e.v : m;
            }
            if (first) {
                top_first<N>(top, A.top, x, idx, valid, m, any, buf[wave]);
                first = false;
            } else if (__ballot(any && m >= top.tv)) {
#pragma unroll
                for (u32 k = 0; k < N; k++) top.insert(A.top, valid[k], x[k], idx[k]);
            }
        }
        __syncthreads();
        TopEntry *all = &buf[0][0];
        if (lane < A.top) all[wave * A.top + lane] = TopEntry{top.v, top.i, 0};
        __syncthreads();
        top_merge<4>(all, merged, A.top);
    }
    logprobs_finish(in, A, row, s, merged, tid, 256);
}

// The gradient: one workgroup per row
template <int SH>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(LogitIn<SH> in, u64 vocab, float unit, const i64 *__restrict__ ids,
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

constexpr u64 LP_GROUPS = 1024; // workgroups that fill the chip: four on each CU
constexpr u64 LP_CHUNK = 2048;  // words: one tile for each of four wavefronts
constexpr u64 LP_WAVE_ROW = 1024; // rows up to this length are read by one wavefront each
template <int SH> int logprobs_run(mpcx_ctx *ctx, LogitIn<SH> in, const LogprobArgs &A) {
    if (A.splits == 1 && A.vocab <= LP_WAVE_ROW)
        hipLaunchKernelGGL((logprobs_kernel<1, SH>), dim3((u32)ceil_div(A.rows, 4)), dim3(256), 0, ctx->stream, in, A);
    else
        hipLaunchKernelGGL((logprobs_kernel<4, SH>), dim3((u32)(A.rows * A.splits)), dim3(256), 0, ctx->stream, in, A);
    MPCX_LAUNCH_CHECK();
    if (A.splits > 1) {
        hipLaunchKernelGGL(logprobs_join_kernel<SH>, dim3((u32)A.rows), dim3(256), 0, ctx->stream, in, A);
        MPCX_LAUNCH_CHECK();
    }
    return 0;
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

// Groups that share a row: enough that the launch has LP_GROUPS workgroups of work, as long as each reads LP_CHUNK words.
static u64 logprob_chunk(u64 rows, u64 vocab) {
    u64 splits = rows >= LP_GROUPS ? 1 : LP_GROUPS / (rows ? rows : 1);
    if (splits > ceil_div(vocab, LP_CHUNK)) splits = ceil_div(vocab, LP_CHUNK);
    return ceil_div(ceil_div(vocab, splits ? splits : 1), 2048) * 2048;
}
uint64_t mpcx_reveal_logprobs_scratch(uint64_t rows, uint64_t vocab, uint64_t top) {
    const u64 splits = vocab ? ceil_div(vocab, logprob_chunk(rows, vocab)) : 1;
    return splits > 1 ? rows * splits * (sizeof(RowPart) + top * sizeof(TopEntry)) : 16;
}
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
    LogprobArgs A{};
    A.rows = rows, A.vocab = vocab, A.chunk = logprob_chunk(rows, vocab), A.splits = (u32)ceil_div(vocab, A.chunk), A.top = (u32)top;
    A.unit = ldexpf(1.0f, -frac), A.unit2 = ldexpf(1.44269504f, -frac);
    A.ids = ids, A.per_row = per_row, A.logp = logp, A.entropy = entropy, A.top_ids = top_ids, A.top_logp = top_logp;
    A.row_max = row_max, A.log_sum = log_sum;
    A.parts = (RowPart *)scratch, A.lists = (TopEntry *)(A.parts + rows * A.splits);
    return c ? logprobs_run<3>(ctx, {(const u64 *)a, (const u64 *)b, (const u64 *)c}, A)
         : b ? logprobs_run<2>(ctx, {(const u64 *)a, (const u64 *)b, nullptr}, A)
             : logprobs_run<1>(ctx, {(const u64 *)a, nullptr, nullptr}, A);
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
    auto run = [&](auto in) -> int {
        hipLaunchKernelGGL(logprobs_grad_kernel, dim3((u32)rows), dim3(256), 0, ctx->stream, in, vocab, ldexpf(1.0f, -frac), ids,
                           per_row, d_logp, d_entropy, row_max, log_sum, entropy, grad, grad_words, ldexpf(1.0f, grad_frac));
        MPCX_LAUNCH_CHECK();
        return 0;
    };
    return c ? run(LogitIn<3>{(const u64 *)a, (const u64 *)b, (const u64 *)c})
         : b ? run(LogitIn<2>{(const u64 *)a, (const u64 *)b, nullptr})
             : run(LogitIn<1>{(const u64 *)a, nullptr, nullptr});
}

} // extern "C"
