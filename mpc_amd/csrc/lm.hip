// Language-model operators on secret shares: lookup in a shared table and its gradient, the global norm of shared
// tensors and clipping, log probabilities of opened logits and their gradient (include/mpcx.h, "language models on
// shares").  Share arithmetic is exact mod 2^64, so sums may be taken in any order.
#include "mpcx_internal.h"
#include "prg_map.h"

namespace {

// a product of sizes that stays below 2^56 words (every byte count then fits 64 bits)
bool lm_fits(u64 a, u64 b) { return a == 0 || b <= (1ull << 56) / a; }
// Workgroups of one launch (a grid holds fewer than 2^32 threads); what is left over is reached by striding, or by
// another launch.
constexpr u64 LM_MAX_BLOCKS = 1ull << 22;
u64 lm_blocks(u64 n) {
    const u64 cap = LM_MAX_BLOCKS < MPCX_MAX_GRID ? LM_MAX_BLOCKS : MPCX_MAX_GRID;
    return n < cap ? n : cap;
}

// two neighbouring words by one 16-byte access; share arrays are 8-byte aligned only, which the hardware takes
typedef u64 u64x2 __attribute__((ext_vector_type(2)));
typedef u64x2 u64x2u __attribute__((aligned(8)));
__device__ inline u64x2 ld2(const u64 *p) { return *(const u64x2u *)p; }
// STREAM: the hint that the words are not read again soon, for calls that move more than the last-level cache holds
// (lookup of 16384 x 4096 words of two shares 301 -> 283 us, gradient of log probabilities of 2048 x 32768 387 -> 379)
template <bool STREAM = false> __device__ inline void st2(u64 *p, u64x2 v) {
    if (STREAM)
        __builtin_nontemporal_store(v, (u64x2u *)p);
    else
        *(u64x2u *)p = v;
}
constexpr u64 STREAM_BYTES = 256ull << 20;
// How a row of dim words is cut: 2^lg lanes (8 .. 2^max_lg, no more than a row needs) take 2 steps << lg words of it, `slices`
// such pieces.  In calls that stream, the pieces of an output row that does not begin on a 128-byte line are moved forward
// (`lines`) so that each of them does: a line that two wavefronts write a part of costs the memory more than a whole one.  The
// first piece then holds up to 15 words less -- a column of it may lie before the row, below 0, as a u64 beyond every column
// -- and the last one more, so this is done where it takes an eighth more pieces at most (two shares; lookup of 16384 x 4095:
// 290 us against 306, 65536 x 500 would go from one piece to two: 155 against 126; gradient of 15 tokens, 21447 rows of 3129:
// 194 us against 253).
constexpr u32 LINE_WORDS = 16;
struct RowCut {
    u32 lg;
    u64 slices;
    bool lines;
    RowCut() = default;
    RowCut(u64 dim, u32 max_lg, u32 steps, bool stream, const void *out) : lg(3), lines(false) {
        while (lg < max_lg && (2ull * steps << lg) < dim) lg++;
        const u64 width = 2ull * steps << lg, whole = ceil_div(dim, width), moved = ceil_div(dim + LINE_WORDS - 1, width);
        if (stream && ((u64)out % (8 * LINE_WORDS) || dim % LINE_WORDS)) lines = 8 * moved <= 9 * whole;
        slices = lines ? moved : whole;
    }
    // the first column of lane `lane` of slice `slice` of the row that is written at `row`
    __device__ u64 column(u64 slice, u32 lane, const u64 *row, u32 steps = 1) const {
        return 2 * ((slice * steps << lg) + lane) - (lines ? (u64)row / 8 % LINE_WORDS : 0);
    }
};
// the two words from p on, of which the row holds those that are asked for
__device__ inline u64x2 ld_part(const u64 *p, bool lo, bool hi) {
    if (lo && hi) return ld2(p);
    u64x2 v = {0, 0};
    if (lo) v.x = p[0];
    if (hi) v.y = p[1];
    return v;
}
template <bool STREAM> __device__ inline void st_part(u64 *p, u64x2 v, bool lo, bool hi) {
    if (lo && hi) return st2<STREAM>(p, v);
    if (lo) p[0] = v.x;
    if (hi) p[1] = v.y;
}

// ---- lookup: a copy of rows, bound by memory traffic (16384 rows of 4096 words of two shares, 6800 different ones: 1.5 GB
// in 275 us).  A row is copied by 2^lg lanes (8 .. 256) of a workgroup; a lane has two 16-byte loads under way, one of each
// share or two of the one (two of each: 280 us; one of a single share: 168 us against 127 for that half).
constexpr u32 emb_steps(bool two) { return two ? 1 : 2; }
template <bool TWO, bool STREAM>
__global__ __launch_bounds__(256) void embed_kernel(const u64 *__restrict__ T0, const u64 *__restrict__ T1, u64 vocab, u64 dim,
                                                    const i64 *__restrict__ ids, u64 n, u64 scale, int shift,
                                                    u64 *__restrict__ E0, u64 *__restrict__ E1, RowCut cut) {
    constexpr u32 EMB_STEPS = emb_steps(TWO);
    const u32 lg = cut.lg, lane = threadIdx.x & ((1u << lg) - 1), rows = 256u >> lg;
    for (u64 t = (u64)blockIdx.x * rows + (threadIdx.x >> lg); t < n; t += (u64)gridDim.x * rows) {
        const u64 v = (u64)ids[t];
        const bool ok = v < vocab;
        const u64 *r0 = T0 + v * dim, *r1 = TWO ? T1 + v * dim : nullptr;
        const u64 first = cut.column(blockIdx.y, lane, E0 + t * dim, EMB_STEPS);
        u64x2 a[EMB_STEPS], b[EMB_STEPS];
#pragma unroll
        for (u32 u = 0; u < EMB_STEPS; u++) {
            const u64 c = first + ((u64)(2 * u) << lg);
            const bool lo = ok && c < dim, hi = ok && c + 1 < dim;
            a[u] = ld_part(r0 + c, lo, hi);
            if (TWO) b[u] = ld_part(r1 + c, lo, hi);
        }
#pragma unroll
        for (u32 u = 0; u < EMB_STEPS; u++) {
            const u64 c = first + ((u64)(2 * u) << lg);
            const bool lo = c < dim, hi = c + 1 < dim;
            u64x2 x = a[u] * scale;
            if (!TWO) x.x = (u64)((i64)x.x >> shift), x.y = (u64)((i64)x.y >> shift);
            st_part<STREAM>(E0 + t * dim + c, x, lo, hi);
            if (TWO) st_part<STREAM>(E1 + t * dim + c, b[u] * scale, lo, hi);
        }
    }
}
// ---- gradient of the lookup.  Rows of G whose tokens are equal are added; every word of G is read once and every word of
// the table written once, so memory traffic is the bound.  A wavefront (or 2^lg lanes of it) owns 128 columns of a row of
// the table, a 16-byte piece of each share per lane, and adds NT tokens at a time, whose loads are under way
// together.  65536 tokens, 65536 rows of 1024 words of two shares (2.15 GB): 450 us, 410 of them in the additions (5.2 TB/s;
// a copy reaches 5.1); four pieces per lane take 490, atomic additions into the table 1300.
struct GradArgs {
    const u64 *G0, *G1;
    const i64 *ids;
    u64 n, vocab, dim, scale;
    int shift, accumulate;
    u64 *D0, *D1;
};
template <bool TWO> struct RowAcc {
    u64x2 a = 0, b = 0;
    // adds columns c and c + 1 of the rows row(i) of p0 / p1, i = i0, i0 + step, .. below i1, NT at a time, what is left NT / 2
    // at a time and so on
    template <u32 NT, class F>
    __device__ void add_rows(F row, const u64 *p0, const u64 *p1, u32 i0, u32 i1, u32 step, u64 c, u64 dim) {
        const bool lo = c < dim, hi = c + 1 < dim;
        u32 i = i0;
        for (; i + (NT - 1) * step < i1; i += NT * step) {
            u64 at[NT];
            u64x2 x[NT], y[NT];
#pragma unroll
            for (u32 q = 0; q < NT; q++) at[q] = row(i + q * step) + c;
#pragma unroll
            for (u32 q = 0; q < NT; q++) {
                x[q] = ld_part(p0 + at[q], lo, hi);
                if (TWO) y[q] = ld_part(p1 + at[q], lo, hi);
            }
#pragma unroll
            for (u32 q = 0; q < NT; q++) {
                a += x[q];
                if (TWO) b += y[q];
            }
        }
        if constexpr (NT > 1) add_rows<NT / 2>(row, p0, p1, i, i1, step, c, dim);
    }
    template <bool STREAM> __device__ static void put(u64 *p, u64x2 v, bool lo, bool hi, int accumulate) {
        if (accumulate) v += ld_part(p, lo, hi);
        st_part<STREAM>(p, v, lo, hi);
    }
    template <bool STREAM> __device__ void write(const GradArgs &A, u64 row, u64 c) const {
        const bool lo = c < A.dim, hi = c + 1 < A.dim;
        u64x2 x = a * A.scale;
        if (!TWO) x.x = (u64)((i64)x.x >> A.shift), x.y = (u64)((i64)x.y >> A.shift);
        put<STREAM>(A.D0 + row * A.dim + c, x, lo, hi, A.accumulate);
        if (TWO) put<STREAM>(A.D1 + row * A.dim + c, b * A.scale, lo, hi, A.accumulate);
    }
};
// the sums of WAVES wavefronts in the first one (one 16-byte piece of each share per lane); all threads call it
template <bool TWO, u32 WAVES> __device__ inline void join_waves(RowAcc<TWO> &acc, u64x2 *lds) {
    const u32 lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    if (wave) {
        lds[(wave - 1) * 64 + lane] = acc.a;
        if (TWO) lds[(WAVES - 1 + wave - 1) * 64 + lane] = acc.b;
    }
    __syncthreads();
    if (wave == 0)
        for (u32 w = 0; w < WAVES - 1; w++) {
            acc.a += lds[w * 64 + lane];
            if (TWO) acc.b += lds[(WAVES - 1 + w) * 64 + lane];
        }
}

// Few tokens: one launch.  A workgroup owns GRAD_ROWS rows of the table, 128 columns of them: it looks through all ids,
// sorts its own tokens by row in LDS, and adds them -- a row of few tokens by one wavefront, a row of many by all four.
// Taken up to GRAD_SMALL_N tokens (1000 rows of 256: 2048 tokens 12 us against 18 of the other form, 4096: 25 against 20),
// up to GRAD_SMALL_SCAN ids read by all workgroups together (8000 rows of 512: 500 tokens 17 us against 25, 2000: 23 against
// 26; of 1024: 2000 tokens 38 us against 32) and up to GRAD_SMALL_BLOCKS workgroups (64 tokens, 8000 rows of 1024: 25 us
// against 26; one token, 131072 rows of 64: 38 us against 23; 15 tokens, 21447 rows of 3129: 350 us against 190).
constexpr u32 GRAD_ROWS = 8, GRAD_SMALL_N = 2048, GRAD_ALONE = 8;
constexpr u64 GRAD_SMALL_SCAN = 1 << 23, GRAD_SMALL_BLOCKS = 8192;
template <bool TWO> __global__ __launch_bounds__(256) void embed_grad_small_kernel(GradArgs A) {
    __shared__ u16 list[GRAD_SMALL_N];
    __shared__ u32 cnt[GRAD_ROWS + 1], off[GRAD_ROWS + 1];
    __shared__ u64x2 lds[3 * (TWO ? 2 : 1) * 64];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = (u32)A.n;
    const u64 v0 = (u64)blockIdx.x * GRAD_ROWS;
    const u32 rows = (u32)(A.vocab - v0 < GRAD_ROWS ? A.vocab - v0 : GRAD_ROWS);
    constexpr u32 PER = GRAD_SMALL_N / 256;
    u32 mine[PER]; // rows of this workgroup that the thread's tokens belong to
#pragma unroll
    for (u32 q = 0; q < PER; q++) {
        const u32 t = 256 * q + tid;
        const u64 r = t < n ? (u64)A.ids[t] - v0 : GRAD_ROWS;
        mine[q] = r < rows ? (u32)r : GRAD_ROWS;
    }
    if (tid <= GRAD_ROWS) cnt[tid] = 0;
    __syncthreads();
#pragma unroll
    for (u32 q = 0; q < PER; q++)
        if (mine[q] < GRAD_ROWS) mine[q] |= atomicAdd(&cnt[mine[q]], 1u) << 8; // its place among the row's
    __syncthreads();
    if (tid <= GRAD_ROWS) {
        u32 s = 0;
#pragma unroll
        for (u32 r = 0; r < GRAD_ROWS; r++) s += r < tid ? cnt[r] : 0;
        off[tid] = s;
    }
    __syncthreads();
#pragma unroll
    for (u32 q = 0; q < PER; q++)
        if (mine[q] != GRAD_ROWS) list[off[mine[q] & 255] + (mine[q] >> 8)] = (u16)(256 * q + tid);
    __syncthreads();
    const u64 c0 = (u64)blockIdx.y * 128 + 2 * lane;
    auto row = [&](u32 i) { return (u64)list[i] * A.dim; };
    for (u32 r = wave; r < rows; r += 4) {
        const u32 k = off[r + 1] - off[r];
        if (k > GRAD_ALONE || (k == 0 && A.accumulate)) continue;
        RowAcc<TWO> acc;
        acc.template add_rows<4>(row, A.G0, A.G1, off[r], off[r + 1], 1, c0, A.dim);
        acc.template write<false>(A, v0 + r, c0);
    }
    for (u32 r = 0; r < rows; r++) {
        if (off[r + 1] - off[r] <= GRAD_ALONE) continue;
        RowAcc<TWO> acc;
        acc.template add_rows<8>(row, A.G0, A.G1, off[r] + wave, off[r + 1], 4, c0, A.dim);
        join_waves<TWO, 4>(acc, lds);
        if (wave == 0) acc.template write<false>(A, v0 + r, c0);
    }
}

// Many tokens: the tokens are put in the order of their rows first (a counting sort; the order inside a row is as it
// comes, sums mod 2^64 do not depend on it), then every row is added by one group of lanes.  A heavy row, of more than
// GRAD_CHUNK tokens, is added chunk by chunk: chunk k is the places [GRAD_CHUNK k, GRAD_CHUNK (k + 1)) of the order, which
// no heavy row lies inside of, so that it meets two at most; their sums go through scratch memory, and the workgroups of
// the chunk that a heavy row begins in add them up.
constexpr u32 GRAD_TOGETHER = 4, GRAD_CHUNK = 32;
struct GradWork {
    u32 *total; // places of the order: tokens inside the vocabulary
    u32 *count, *start, *rank;
    u32 *order, *row; // of each place: the token and its row
    u64 *partial;     // two sums of each chunk: dim words of each share
    __device__ void place(u32 at, u32 t, u32 v) const { order[at] = t, row[at] = v; }
};
// chunk k: its places, and the rows of the first and the last one
struct GradChunk {
    u32 p0, p1, va, vb;
    __device__ GradChunk(const GradWork &W, u32 total, u32 k) {
        p0 = k * GRAD_CHUNK, p1 = total - p0 < GRAD_CHUNK ? total : p0 + GRAD_CHUNK;
        va = W.row[p0], vb = W.row[p1 - 1];
    }
};
// The whole sort in one launch: a workgroup owns `rows` rows of the table and looks through all ids twice, counting its
// tokens in LDS (and those of the rows before, which gives its first place), then placing them.  Up to GRAD_SCAN_N tokens,
// where it comes level with the histogram in memory below, four launches (1000 rows of 256: 32768 tokens take 46 us in
// all either way, 49152 take 65 against 57; 32768 rows of 256: 74 against 76, 81 against 77).
constexpr u32 GRAD_SCAN_ROWS = 4096, GRAD_SCAN_THREADS = 1024;
constexpr u64 GRAD_SCAN_N = 32768;
__global__ __launch_bounds__(1024) void grad_scan_kernel(const i64 *__restrict__ ids, u32 n, u64 vocab, u32 rows, GradWork W) {
    __shared__ u32 cnt[GRAD_SCAN_ROWS], ws[16], wb[16];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const u64 v0 = (u64)blockIdx.x * rows;
    const u32 own = (u32)(vocab - v0 < rows ? vocab - v0 : rows);
    for (u32 r = tid; r < GRAD_SCAN_ROWS; r += GRAD_SCAN_THREADS) cnt[r] = 0;
    __syncthreads();
    u32 below = 0;
    auto look = [&](auto token) { // token(t, v) for every id, two by two
#pragma unroll 4
        for (u32 t = 2 * tid; t + 1 < n; t += 2 * GRAD_SCAN_THREADS) {
            const u64x2 v = ld2((const u64 *)ids + t);
            token(t, v.x), token(t + 1, v.y);
        }
        if (tid == 0 && (n & 1)) token(n - 1, (u64)ids[n - 1]);
    };
    look([&](u32, u64 v) {
        below += v < v0;
        if (v - v0 < own) atomicAdd(&cnt[v - v0], 1u);
    });
    __syncthreads();
    u32 c[4], s = 0; // four rows of a thread
#pragma unroll
    for (u32 k = 0; k < 4; k++) c[k] = cnt[4 * tid + k], s += c[k];
    u32 sum = s;
    for (u32 d = 1; d < 64; d <<= 1) {
        const u32 o = (u32)__shfl_up((int)sum, d);
        if (lane >= d) sum += o;
    }
    for (u32 d = 32; d; d >>= 1) below += (u32)__shfl_xor((int)below, d);
    if (lane == 63) ws[wave] = sum;
    if (lane == 0) wb[wave] = below;
    __syncthreads();
    u32 at = sum - s, mine = 0;
    for (u32 w = 0; w < 16; w++) {
        at += wb[w] + (w < wave ? ws[w] : 0);
        mine += ws[w];
    }
    if (tid == GRAD_SCAN_THREADS - 1 && v0 + own == vocab) *W.total = at + s;
#pragma unroll
    for (u32 k = 0; k < 4; k++) {
        const u32 r = 4 * tid + k;
        if (r < own) W.count[v0 + r] = c[k], W.start[v0 + r] = at;
        cnt[r] = at;
        at += c[k];
    }
    __syncthreads();
    if (mine)
        look([&](u32 t, u64 v) {
            if (v - v0 < own) W.place(atomicAdd(&cnt[v - v0], 1u), t, (u32)v);
        });
}
__global__ __launch_bounds__(256) void grad_clear_kernel(u32 *p, u64 n) {
    for (u64 i = (u64)blockIdx.x * 256 + threadIdx.x; i < n; i += (u64)gridDim.x * 256) p[i] = 0;
}
// count[v] = tokens of row v, rank[t] = place of token t among those of its row.  A workgroup first counts its own
// tokens in a hash table in LDS, then adds each row's number to memory once: the frequent tokens of a text would
// otherwise queue up at one address (65536 tokens, one in sixteen the same: 48 us).
constexpr u32 GRAD_TOKENS = 1024, GRAD_SLOTS = 2048; // per workgroup of 256: tokens, slots of its table
__global__ __launch_bounds__(256) void grad_count_kernel(const i64 *__restrict__ ids, u32 n, u64 vocab, GradWork W) {
    __shared__ u32 key[GRAD_SLOTS], num[GRAD_SLOTS];
    const u32 tid = threadIdx.x;
    for (u32 i = tid; i < GRAD_SLOTS; i += 256) key[i] = ~0u, num[i] = 0;
    __syncthreads();
    u32 slot[GRAD_TOKENS / 256], rank[GRAD_TOKENS / 256];
#pragma unroll
    for (u32 q = 0; q < GRAD_TOKENS / 256; q++) {
        const u32 t = blockIdx.x * GRAD_TOKENS + 256 * q + tid;
        const u64 v = t < n ? (u64)ids[t] : vocab;
        slot[q] = ~0u;
        if (v < vocab) {
            u32 h = (u32)v * 2654435761u >> 21; // the table has a free slot for every token
            for (;;) {
                const u32 k = atomicCAS(&key[h], ~0u, (u32)v);
                if (k == ~0u || k == (u32)v) break;
                h = (h + 1) & (GRAD_SLOTS - 1);
            }
            slot[q] = h;
            rank[q] = atomicAdd(&num[h], 1u);
        }
    }
    __syncthreads();
    for (u32 i = tid; i < GRAD_SLOTS; i += 256)
        if (num[i]) num[i] = atomicAdd(&W.count[key[i]], num[i]);
    __syncthreads();
#pragma unroll
    for (u32 q = 0; q < GRAD_TOKENS / 256; q++)
        if (slot[q] != ~0u) W.rank[blockIdx.x * GRAD_TOKENS + 256 * q + tid] = num[slot[q]] + rank[q];
}
// the rows' first places, in the order in which the workgroups come
__global__ __launch_bounds__(256) void grad_place_kernel(u32 vocab, GradWork W) {
    __shared__ u32 ws[4], at;
    const u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const u32 v = blockIdx.x * 256 + tid;
    const u32 c = v < vocab ? W.count[v] : 0;
    u32 s = c; // inclusive sum over the wavefront
    for (u32 d = 1; d < 64; d <<= 1) {
        const u32 o = (u32)__shfl_up((int)s, d);
        if (lane >= d) s += o;
    }
    if (lane == 63) ws[wave] = s;
    __syncthreads();
    if (tid == 0) {
        const u32 sum = ws[0] + ws[1] + ws[2] + ws[3];
        at = sum ? atomicAdd(W.total, sum) : 0;
    }
    __syncthreads();
    u32 first = at + s - c;
    for (u32 w = 0; w < wave; w++) first += ws[w];
    if (v < vocab) W.start[v] = first;
}
__global__ __launch_bounds__(256) void grad_order_kernel(const i64 *__restrict__ ids, u32 n, u64 vocab, GradWork W) {
    const u32 t = blockIdx.x * 256 + threadIdx.x;
    if (t >= n) return;
    const u64 v = (u64)ids[t];
    if (v < vocab) W.place(W.start[v] + W.rank[t], t, (u32)v);
}
// The first `heavy` workgroups add the chunks' parts of heavy rows into scratch memory, 128 columns per wavefront; the others
// one row of the table, 128 columns or less, per 2^lg lanes.  Where rows without tokens stay as they are and the tokens are
// fewer than the rows, the rows are found at the first of their places, else by looking at all of them (32768 rows of 1024,
// accumulated: 3000 tokens 33 us against 51, 131072 rows of 128: 65536 tokens 69 us against 72).
struct GradCut {
    u32 heavy, slices; // slices of 128 columns, of heavy rows
    bool by_place;
    RowCut row; // of the other rows
};
template <bool TWO, bool STREAM>
__global__ __launch_bounds__(256) void grad_rows_kernel(GradArgs A, GradWork W, GradCut cut) {
    RowAcc<TWO> acc;
    if (blockIdx.x < cut.heavy) {
        const u32 slices = cut.slices;
        const u32 total = *W.total;
        const u64 items = (u64)((total + GRAD_CHUNK - 1) / GRAD_CHUNK) * slices;
        for (u64 it = (u64)blockIdx.x * 4 + (threadIdx.x >> 6); it < items; it += (u64)cut.heavy * 4) {
            const u64 k = it / slices, c0 = (it % slices) * 128 + 2 * (threadIdx.x & 63);
            const GradChunk ch(W, total, (u32)k);
            for (u32 side = 0; side < (ch.va == ch.vb ? 1u : 2u); side++) {
                const u32 v = side ? ch.vb : ch.va, c = W.count[v], first = W.start[v];
                if (c <= GRAD_CHUNK) continue;
                const u32 i0 = first > ch.p0 ? first : ch.p0, i1 = first + c < ch.p1 ? first + c : ch.p1;
                acc = RowAcc<TWO>();
                acc.template add_rows<GRAD_TOGETHER>([&](u32 i) { return (u64)W.order[i] * A.dim; }, A.G0, A.G1, i0, i1, 1, c0, A.dim);
                u64 *p = W.partial + (2 * k + side) * 2 * A.dim + c0;
                st_part<false>(p, acc.a, c0 < A.dim, c0 + 1 < A.dim);
                if (TWO) st_part<false>(p + A.dim, acc.b, c0 < A.dim, c0 + 1 < A.dim);
            }
        }
        return;
    }
    const u32 lg = cut.row.lg;
    const u64 slices = cut.row.slices, n = cut.by_place ? *W.total : A.vocab, step = (u64)(gridDim.x - cut.heavy) * 256 >> lg;
    for (u64 item = ((u64)(blockIdx.x - cut.heavy) * 256 + threadIdx.x) >> lg; item < n * slices; item += step) {
        u64 v = item / slices;
        const u32 place = (u32)v;
        if (cut.by_place) v = W.row[place];
        const u32 c = W.count[v];
        if (c > GRAD_CHUNK || (c == 0 && A.accumulate)) continue;
        const u32 first = c ? W.start[v] : 0;
        if (cut.by_place && first != place) continue;
        const u64 c0 = cut.row.column(item % slices, threadIdx.x & ((1u << lg) - 1), A.D0 + v * A.dim);
        acc = RowAcc<TWO>();
        acc.template add_rows<GRAD_TOGETHER>([&](u32 i) { return (u64)W.order[first + i] * A.dim; }, A.G0, A.G1, 0, c, 1, c0, A.dim);
        acc.template write<STREAM>(A, v, c0);
    }
}
// 128 columns of the heavy rows that begin in eight chunks (one at most does in each): a wavefront looks at one chunk and
// adds the sums of its row when they are few; those of a longer row are shared out to all wavefronts.
constexpr u32 HEAVY_WAVES = 8, HEAVY_ALONE = 8;
template <bool TWO>
__global__ __launch_bounds__(64 * HEAVY_WAVES) void grad_heavy_kernel(GradArgs A, GradWork W, u32 slices, u64 items) {
    __shared__ u64x2 lds[(HEAVY_WAVES - 1) * (TWO ? 2 : 1) * 64];
    __shared__ u32 begin[HEAVY_WAVES], chunks[HEAVY_WAVES], rows[HEAVY_WAVES]; // the sum of the first chunk, how many, the row
    const u32 total = *W.total, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (u64 it = blockIdx.x; it < items; it += gridDim.x) { // items = slices for every HEAVY_WAVES chunks
        const u32 k = (u32)(it / slices) * HEAVY_WAVES + wave;
        const u64 c0 = (it % slices) * 128 + 2 * lane;
        u32 n = 0, b = 0, v = 0;
        if ((u64)k * GRAD_CHUNK < total) {
            const GradChunk ch(W, total, k);
            const u32 c = W.count[ch.vb], first = W.start[ch.vb];
            if (c > GRAD_CHUNK && first >= ch.p0) n = (first + c - 1) / GRAD_CHUNK - k + 1;
            b = 2 * k + (ch.va != ch.vb), v = ch.vb;
        }
        // the first chunk's sum is the one of its last row, every other chunk's that of its first row
        auto add = [&](RowAcc<TWO> &acc, u32 b, u32 i0, u32 n, u32 step) {
            acc.template add_rows<8>([&](u32 i) { return (u64)(i ? (b & ~1u) + 2 * i : b) * 2 * A.dim; }, W.partial,
                                     W.partial + A.dim, i0, n, step, c0, A.dim);
        };
        __syncthreads(); // the lists of the item before have been read
        if (lane == 0) begin[wave] = b, rows[wave] = v, chunks[wave] = n > HEAVY_ALONE ? n : 0;
        if (n && n <= HEAVY_ALONE) {
            RowAcc<TWO> acc;
            add(acc, b, 0, n, 1);
            acc.template write<false>(A, v, c0);
        }
        __syncthreads();
        for (u32 q = 0; q < HEAVY_WAVES; q++) {
            if (chunks[q] == 0) continue;
            RowAcc<TWO> acc;
            add(acc, begin[q], wave, chunks[q], HEAVY_WAVES);
            join_waves<TWO, HEAVY_WAVES>(acc, lds);
            if (wave == 0) acc.template write<false>(A, rows[q], c0);
        }
    }
}

// ---- many tensors in one launch.  The tensors of a call are cut into tiles; up to LM_TENSORS descriptors travel in the
// kernel's own arguments, so nothing is copied to the device and a captured call keeps its descriptors.  A workgroup
// finds the tensor of a tile by one comparison per lane and a population count.
constexpr u32 LM_TENSORS = 96;    // descriptors of 40 bytes: the arguments stay below 4 KiB
constexpr u64 LM_TILE = 1024;     // words
constexpr u32 LM_GRID = 1024;     // of the norm: four workgroups of four waves on each of 256 CUs (2048: 3 % slower)
struct TensorRef {
    const u64 *x0, *x1;
    u64 n, out, tile0; // words, first word in the call's output, first tile
};
struct TensorTable {
    TensorRef t[LM_TENSORS];
    u32 count;
    u64 tiles;
};
__device__ inline i64 lane_word(i64 v, u32 lane) {
    const u32 lo = (u32)__builtin_amdgcn_readlane((int)(u32)v, (int)lane), hi = (u32)__builtin_amdgcn_readlane((int)((u64)v >> 32), (int)lane);
    return (i64)((u64)hi << 32 | lo);
}
// the last of `count` descriptors that begins(k) holds for (it does for the first, and for none behind one without)
template <class F> __device__ inline u32 last_below(u32 count, F begins) {
    const u32 lane = threadIdx.x & 63, far = lane + 64 < LM_TENSORS ? lane + 64 : 0;
    const bool a = lane < count && begins(lane), b = lane + 64 < count && begins(far);
    const u32 k = (u32)(__popcll(__ballot(a)) + __popcll(__ballot(b))) - 1;
    return __builtin_amdgcn_readfirstlane(k);
}
__device__ inline u32 tensor_of(const TensorTable &tab, u64 tile) {
    return last_below(tab.count, [&](u32 k) { return tab.t[k].tile0 <= tile; });
}

// sum of x0 (x0 + 2 x1) = x0^2 + x0 x1 + x1 x0 over the tiles of a workgroup -> part[workgroup]: one 64-bit product for 16
// bytes read, bound by the reads (2e8 words in 293 tensors: 505-535 us in all, 6.0-6.3 TB/s)
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
// z = the sum of the partial sums + A[tA] - B[tB] (one word of each of two generator streams); 6700 partial sums: 11 us when
// a thread waits for each of its words
__global__ __launch_bounds__(1024) void sqnorm_join_kernel(const u64 *__restrict__ part, u64 parts, const PrgCk *__restrict__ ckA,
                                                          const PrgCk *__restrict__ ckB, u64 tA, u64 tB, u64 *__restrict__ z) {
    __shared__ u64 ws[16];
    const u32 tid = threadIdx.x, waves = blockDim.x / 64;
    u64 s = 0;
    for (u64 i = tid; i < parts; i += 8 * blockDim.x) {
        u64 p[8];
#pragma unroll
        for (u32 q = 0; q < 8; q++) p[q] = i + q * blockDim.x < parts ? part[i + q * blockDim.x] : 0;
#pragma unroll
        for (u32 q = 0; q < 8; q++) s += p[q];
    }
    if (tid == 0 || tid == 64) {
        PrgCursor g;
        g.open(tid ? ckB : ckA, tid ? tB : tA, true);
        const u64 w = g.next();
        s += tid ? 0 - w : w;
    }
    for (u32 d = 32; d; d >>= 1) s += __shfl_xor((unsigned long long)s, d);
    if ((tid & 63) == 0) ws[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) {
        for (u32 w = 1; w < waves; w++) s += ws[w];
        *z = s;
    }
}

// f to the nearest word, ties to even; beyond the range its ends, 0 for what is no number
__device__ inline i64 nearest_word(float f) {
    const float r = rintf(f);
    if (r >= 9223372036854775808.0f) return INT64_MAX;
    if (r <= -9223372036854775808.0f) return INT64_MIN;
    return r == r ? (i64)r : 0;
}

// the largest c in [0, 2^f] with c^2 S <= R^2: an estimate in 64-bit floats, off by one at most (c < 2^32), put right in
// 128-bit integers, so that all parties and all roundings agree on it
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
// y = (c x0) >> number (party 0).  A copy with a product, bound by memory traffic (2e8 words in 293 tensors: 575 us, 5.6
// TB/s), best with one small tile per workgroup (4096 words and a looping grid: 655 us).  Every workgroup forms the factor,
// which saves a launch.
__global__ __launch_bounds__(256) void clip_kernel(TensorTable tab, ClipArgs A, i64 *__restrict__ coef, u64 *__restrict__ Y) {
    const u32 tid = threadIdx.x;
    const u64 c = A.factor();
    if (blockIdx.x == 0 && tid == 0) *coef = (i64)c;
    const int sh = A.number;
    for (u64 tile = blockIdx.x; tile < tab.tiles; tile += gridDim.x) {
        const u32 k = tensor_of(tab, tile);
        const u64 at = (tile - tab.t[k].tile0) * LM_TILE, n = tab.t[k].n - at;
        const u64 *x0 = tab.t[k].x0 + at;
        u64 *y = Y + tab.t[k].out + at;
        if (n >= LM_TILE) {
#pragma unroll
            for (u32 u = 0; u < LM_TILE / 512; u++) {
                const u32 i = 512 * u + 2 * tid;
                const u64x2 a = ld2(x0 + i) * c;
                st2(y + i, u64x2{(u64)((i64)a.x >> sh), (u64)((i64)a.y >> sh)});
            }
        } else {
            for (u64 i = tid; i < n; i += 256) y[i] = (u64)((i64)(x0[i] * c) >> sh);
        }
    }
}
// y = ((c (x0 + x1)) >> number) - w (party 1), w the stream's words, consumed where they are regenerated: 24 bytes of traffic
// a word, the bound of long tensors of whole runs (2^26 words in 1, 4 or 16 tensors: 310 us, 5.2 TB/s).  Tensors of any length
// cost more, 2e8 words in 293 take 1.52 ms (3.2 TB/s): the runs of 16 words that a visit reads lie across lines (the counters
// show up to twice the reads, and a fifth more writes), and launches that begin between two checkpoints of the stream discard
// up to 63 words a lane.  The 32 words of a lane's 16 visits
// are asked for before the stream's are generated, which hides their way from memory (90 tensors of 5000 words: 25 us against
// 33).  A wavefront (4096 words) that lies in one tensor finds it once; another goes, at every visit, from tensor to tensor.
// Scaling all tensors by one launch and masking them by a second takes 542 us for 16 tensors, 30 for 90 of 5000 words, and 26
// for 90 of 100 words, where this takes 41.
struct ClipMasked {
    struct wavefront;
    TensorTable tab;
    const i64 *coef;
    int number;
    u64 *y;
    struct Part { // of the launch's words: those below `end`, x0 and x1 at the launch's word 0
        u64 end;
        const u64 *x0, *x1;
    };
    struct Wave {
        const ClipMasked &f;
        Part near, far; // the lane's two tensors
        Part one;       // the tensor of all words; x0 NULL: there are several
        u64 c;
        __device__ static Part of_lane(const Part &p, u32 lane) {
            return Part{(u64)lane_word((i64)p.end, lane), (const u64 *)lane_word((i64)p.x0, lane), (const u64 *)lane_word((i64)p.x1, lane)};
        }
        __device__ Part part(u64 at) const {
            const u32 k = (u32)(__popcll(__ballot(near.end <= at)) + __popcll(__ballot(far.end <= at)));
            return k < 64 ? of_lane(near, k) : of_lane(far, k - 64);
        }
        struct Ask {
            u64 a[PRG_VISITS], b[PRG_VISITS];
        };
        __device__ Ask ask(u64 rel, u64 count) const {
            Ask s;
#pragma unroll
            for (u32 k = 0; k < PRG_VISITS; k++, rel += PRG_VISIT_STEP) {
                Part p = one;
                if (!one.x0) {
                    const u64 todo = __ballot(rel < count);
                    for (u64 left = todo; left;) { // a lane's word lies behind those of the lanes before it
                        const u32 first = (u32)__builtin_ctzll(left);
                        const Part t = part((u64)lane_word((i64)rel, first));
                        if ((threadIdx.x & 63) >= first) p = t;
                        left = todo & ~__ballot(rel < t.end);
                    }
                }
                s.a[k] = s.b[k] = 0;
                if (rel < count) s.a[k] = p.x0[rel], s.b[k] = p.x1[rel];
            }
            return s;
        }
        __device__ void put(u64 rel, const u64 (&w)[PRG_VISITS], const Ask &s, u64 count) const {
#pragma unroll
            for (u32 k = 0; k < PRG_VISITS; k++, rel += PRG_VISIT_STEP)
                if (rel < count) f.y[rel] = (u64)((i64)((s.a[k] + s.b[k]) * c) >> f.number) - w[k];
        }
    };
    __device__ Part part_of(u32 k) const {
        if (k >= tab.count) return Part{~0ull, nullptr, nullptr};
        const TensorRef &t = tab.t[k];
        return Part{t.out + t.n, t.x0 - t.out, t.x1 - t.out};
    }
    __device__ Wave wave(u64 first, u64 end) const {
        const u32 lane = threadIdx.x & 63;
        Wave w{*this, part_of(lane), part_of(lane + 64), Part{0, nullptr, nullptr}, (u64)*coef};
        if (first >= end) return w;
        const Part p = w.part(first);
        if (end <= p.end) w.one = p;
        return w;
    }
};
static_assert(sizeof(ClipMasked) <= 4096 - 64, "a kernel's arguments");
__global__ void clip_factor_kernel(ClipArgs A, i64 *coef) { *coef = (i64)A.factor(); }

// ---- opened logits.  A word x = a + b + c stands for the logit x 2^-frac; distances from a maximum are differences of
// words, exact before their one conversion to a float.
template <int SH> struct LogitIn {
    const u64 *a, *b, *c;
    void skip(u64 n) { a += n, b = b ? b + n : b, c = c ? c + n : c; }
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

__device__ inline i64 wave_max(i64 v) {
    for (u32 d = 32; d; d >>= 1) {
        const i64 o = (i64)__shfl_xor((long long)v, (int)d);
        v = o > v ? o : v;
    }
    return v;
}

// The likeliest `top` <= 32 entries that a wavefront has seen, in the order value descending, index ascending (all entries
// differ): up to 64 candidates in LDS in any order, and a border (tv, ti) that a new one has to beat.  When the 64 places
// are full the candidates are sorted -- every one counts the better ones, from LDS -- and the first `top` stay; a sort
// costs what a handful of one-by-one insertions would, and most tiles bring no candidate at all.
struct TopEntry {
    i64 v;
    u32 i, pad;
};
constexpr u32 TOP_NONE = ~0u; // the index of an entry that is not there (with the lowest value: behind all others)
__device__ inline bool top_better(i64 av, u32 ai, i64 bv, u32 bi) { return av > bv || (av == bv && ai < bi); }
struct WaveTop {
    TopEntry *buf; // 64 entries
    u32 top, count = 0;
    i64 tv = INT64_MIN;
    u32 ti = TOP_NONE;
    __device__ WaveTop(TopEntry *b, u32 t) : buf(b), top(t) {}
    __device__ void sort() {
        const u32 lane = threadIdx.x & 63;
        const TopEntry e = lane < count ? buf[lane] : TopEntry{INT64_MIN, TOP_NONE, 0};
        u32 rank = 0;
#pragma unroll 8
        for (u32 k = 0; k < count; k++) rank += top_better(buf[k].v, buf[k].i, e.v, e.i);
        prg_wave_sync();
        if (lane < count) buf[rank] = e;
        prg_wave_sync();
        if (count < top) return;
        count = top;
        tv = lane_word(buf[top - 1].v, 0), ti = (u32)__builtin_amdgcn_readfirstlane((int)buf[top - 1].i);
    }
    // at most one candidate per lane, and room for them
    __device__ void append(bool in, i64 x, u32 idx) {
        const u64 b = __ballot(in);
        if (in) buf[count + (u32)__popcll(b & ((1ull << (threadIdx.x & 63)) - 1))] = TopEntry{x, idx, 0};
        count += (u32)__popcll(b);
        prg_wave_sync();
    }
    // N candidates per lane
    template <u32 N> __device__ void add(const i64 (&x)[N], const u32 (&idx)[N], const bool (&valid)[N]) {
        const u32 lane = threadIdx.x & 63;
        u32 left = 0, n = 0;
#pragma unroll
        for (u32 k = 0; k < N; k++) {
            const bool in = valid[k] && top_better(x[k], idx[k], tv, ti);
            left |= (u32)in << k;
            n += (u32)__popcll(__ballot(in));
        }
#pragma unroll 1
        while (n) {
            if (count + n > 64) sort();
            n = 0;
#pragma unroll
            for (u32 k = 0; k < N; k++) {
                const bool in = (left >> k & 1) && top_better(x[k], idx[k], tv, ti);
                const u64 b = __ballot(in);
                const u32 at = count + (u32)__popcll(b & ((1ull << lane) - 1)), c = (u32)__popcll(b), room = 64 - count;
                if (in && at < 64) {
                    buf[at] = TopEntry{x[k], idx[k], 0};
                    left &= ~(1u << k);
                }
                count += c < room ? c : room;
                n += c < room ? 0 : c - room;
            }
            prg_wave_sync();
        }
    }
};
// A distance such that at least `top` of the K values of 64 lanes lie within it, and hardly more than TOP_SLACK others
// (values below 0 are not there; infinity when there are not enough): a bisection that counts with ballots.  `guess` is
// tried first -- sixteen in the exponent, so that rows whose masked words lie far away do not take the range.
constexpr u32 TOP_SLACK = 8;
template <u32 K> __device__ inline float top_border(const float (&near)[K], u32 top, float guess) {
    auto within = [&](float d) {
        u32 n = 0;
#pragma unroll
        for (u32 k = 0; k < K; k++) n += (u32)__popcll(__ballot(near[k] >= 0 && near[k] <= d));
        return n;
    };
    float lo = 0, hi = guess;
    if (within(guess) < top) {
        if (within(INFINITY) < top) return INFINITY;
        lo = guess, hi = 0;
#pragma unroll
        for (u32 k = 0; k < K; k++) hi = fmaxf(hi, near[k]);
        for (u32 d = 32; d; d >>= 1) hi = fmaxf(hi, __shfl_xor(hi, (int)d));
    }
    for (u32 r = 0; r < 16; r++) {
        const float mid = 0.5f * (lo + hi);
        const u32 n = within(mid);
        if (n >= top) hi = mid;
        else lo = mid;
        if (n >= top && n <= top + TOP_SLACK) break;
    }
    return hi;
}
// The first tile of a wavefront: only what lies within the border distance of the lanes' N / 2 pair maxima is a candidate
// (rarely more than a few above `top`).
template <u32 N>
__device__ inline void top_first(WaveTop &t, const i64 (&x)[N], const u32 (&idx)[N], const bool (&valid)[N], i64 lane_max, float guess) {
    const i64 m = wave_max(lane_max);
    float near[N / 2];
#pragma unroll
    for (u32 k = 0; k < N / 2; k++) {
        const i64 best = valid[2 * k + 1] && x[2 * k + 1] > x[2 * k] ? x[2 * k + 1] : x[2 * k];
        near[k] = valid[2 * k] ? word_dist(m, best) : -1.0f;
    }
    const float border = top_border<N / 2>(near, t.top, guess);
    bool in[N];
    u32 at[N], n = 0;
#pragma unroll
    for (u32 k = 0; k < N; k++) {
        in[k] = valid[k] && word_dist(m, x[k]) <= border;
        const u64 b = __ballot(in[k]);
        at[k] = n + (u32)__popcll(b & ((1ull << (threadIdx.x & 63)) - 1));
        n += (u32)__popcll(b);
    }
    if (n > 64) { // many equal words
        t.add(x, idx, in);
        return;
    }
#pragma unroll
    for (u32 k = 0; k < N; k++)
        if (in[k]) t.buf[at[k]] = TopEntry{x[k], idx[k], 0};
    t.count = n;
    prg_wave_sync();
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
#pragma unroll 8
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
    template <class P> __device__ void join(const P &part, float unit2) {
        RowSums o;
        o.m = part.m, o.S = part.S, o.T = part.T;
        if (o.m > m) move_to(o.m, unit2);
        else o.move_to(m, unit2);
        S += o.S, T += o.T;
    }
    __device__ void wave_join(float unit2) {
        move_to(wave_max(m), unit2);
        for (u32 d = 32; d; d >>= 1) S += __shfl_xor(S, (int)d), T += __shfl_xor(T, (int)d);
    }
};
struct RowPart { // of one wavefront; S = 0: it has read no words
    i64 m;
    float S, T;
};
constexpr u32 LIST = 32; // entries of a part's list, in any order; those that are not there have the index TOP_NONE

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
    RowPart *parts;  // splits > 1: rows x splits x 4 wavefronts, then
    TopEntry *lists; // LIST entries for each
};
// a row's outputs, by `n` threads (thread `t` of them); list: the row's sorted entries; at_first: the word of the thread's
// first id, where that has been read (first_id inside the vocabulary)
template <int SH>
__device__ inline void logprobs_finish(const LogitIn<SH> &in, const LogprobArgs &A, u64 row, RowSums s, const TopEntry *list, u32 t, u32 n,
                                       u64 first_id = ~0ull, i64 at_first = 0) {
    const float ls = logf(s.S);
    if (t == 0) {
        if (A.entropy) A.entropy[row] = ls + s.T / s.S * 0.69314718f;
        if (A.row_max) A.row_max[row] = s.m;
        if (A.log_sum) A.log_sum[row] = ls;
    }
    for (u64 k = t; k < A.per_row; k += n) {
        const u64 id = (u64)A.ids[row * A.per_row + k];
        const i64 x = id >= A.vocab ? 0 : k == t && first_id == id ? at_first : in.at(row * A.vocab + id);
        A.logp[row * A.per_row + k] = id < A.vocab ? -(word_dist(s.m, x) * A.unit + ls) : 0.0f;
    }
    if (t < A.top) {
        A.top_ids[row * A.top + t] = (i64)list[t].i;
        A.top_logp[row * A.top + t] = -(word_dist(s.m, list[t].v) * A.unit + ls);
    }
}

// One pass over the logits: maximum, sum of exponentials, entropy sum and top list together, bound by the reads (4096 rows of
// 32771 words of three shares, 3.2 GB: 539 us, 6.0 TB/s; about 30 vector instructions a word).  W wavefronts of a workgroup
// of four read `chunk` words of a row, in tiles of 64 x 8 words each.  A lane keeps its own maximum and sums and moves
// them when a tile raises its maximum; nothing is exchanged between lanes before the end but the ballots that look for new
// entries of the top list.  SPLIT: several workgroups read a row, and every wavefront leaves its own part for
// logprobs_join_kernel.
template <u32 W, bool SPLIT, int SH> __global__ __launch_bounds__(256, W == 1 ? 5 : 1) void logprobs_kernel(LogitIn<SH> in, LogprobArgs A) {
    constexpr u32 U = 4, N = 2 * U, TILE = 64 * N;
    __shared__ TopEntry buf[4][64];
    __shared__ TopEntry merged[32];
    __shared__ RowPart ws[4];
    const u32 tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const u64 group = W == 1 ? (u64)blockIdx.x * 4 + wave : blockIdx.x;
    const u64 row = SPLIT ? group / A.splits : group, split = SPLIT ? group % A.splits : 0;
    if (W == 1 && row >= A.rows) return; // a wavefront of its own: no barrier follows
    const u64 base = row * A.vocab, j0 = split * A.chunk, j1 = j0 + A.chunk < A.vocab ? j0 + A.chunk : A.vocab;
    RowSums s;
    WaveTop top(buf[wave], A.top);
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
            const u32 left = (u32)(j1 - tile);
#pragma unroll
            for (u32 u = 0; u < U; u++) {
                const u32 j = 128 * u + 2 * lane;
                u64x2 p = {1ull << 63, 1ull << 63}; // the lowest word
                if (j + 1 < left) p = in.at2(base + tile + j);
                else if (j < left) p.x = (u64)in.at(base + tile + j);
                x[2 * u] = (i64)p.x, x[2 * u + 1] = (i64)p.y, valid[2 * u] = j < left, valid[2 * u + 1] = j + 1 < left;
            }
        }
        i64 m = x[0];
#pragma unroll
        for (u32 k = 0; k < N; k++) {
            m = x[k] > m ? x[k] : m;
            idx[k] = (u32)(tile + 128 * (k / 2) + 2 * lane + (k & 1));
        }
        if (m > s.m) s.move_to(m, A.unit2);
        float S = 0, T = 0; // of the tile: a lane's sums take one step of rounding a tile, not one a word
#pragma unroll
        for (u32 k = 0; k < N; k++) {
            const float d = word_dist(s.m, x[k]) * A.unit2, e = valid[k] ? exp2_fast(-d) : 0.0f;
            S += e, T = fmaf(d, e, T);
        }
        s.S += S, s.T += T;
        if (A.top) {
            if (first && j1 - tile > 64) {
                top_first<N>(top, x, idx, valid, m, 16.0f / A.unit);
            } else if (__ballot(m >= top.tv)) {
                if (top.count > A.top) top.sort(); // for a border that is up to date
                // the border's entry has a lower index than this tile's words, so equal words do not beat it; and a lane
                // hardly ever has two that do
                u32 over = 0;
#pragma unroll
                for (u32 k = 0; k < N; k++) over |= (u32)(valid[k] && x[k] > top.tv) << k;
                const u64 lanes = __ballot(over);
                if (__ballot(over & (over - 1)) || top.count + (u32)__popcll(lanes) > 64 || top.ti == TOP_NONE) {
                    top.add(x, idx, valid);
                } else if (lanes) {
                    const u32 k = (u32)__builtin_ctz(over | 256);
                    top.append(over, m, (u32)tile + 128 * (k / 2) + 2 * lane + (k & 1));
                }
            }
            first = false;
        }
    }
    s.wave_join(A.unit2);
    if (A.top && (!SPLIT || top.count > LIST)) top.sort();
    if (SPLIT) {
        const u64 part = group * 4 + wave;
        if (lane == 0) A.parts[part] = RowPart{s.m, s.S, s.T};
        if (A.top) {
            if (lane < LIST) A.lists[part * LIST + lane] = lane < top.count ? top.buf[lane] : TopEntry{INT64_MIN, TOP_NONE, 0};
        }
        return;
    }
    if (W == 1) {
        logprobs_finish(in, A, row, s, buf[wave], lane, 64);
        return;
    }
    if (lane == 0) ws[wave] = RowPart{s.m, s.S, s.T};
    const TopEntry mine = lane < top.count ? top.buf[lane] : TopEntry{INT64_MIN, TOP_NONE, 0};
    __syncthreads(); // every wavefront has left its own part of buf
    TopEntry *lists = &buf[0][0];
    if (lane < A.top) lists[wave * A.top + lane] = mine;
    s = RowSums();
    for (u32 w = 0; w < 4; w++) s.join(ws[w], A.unit2);
    __syncthreads();
    if (A.top) top_merge<4>(lists, merged, A.top);
    logprobs_finish(in, A, row, s, merged, tid, 256);
}
constexpr u32 JOIN_THREADS = 512; // 256 / 512 / 1024: 9.4 / 8.2 / 8.1 us for one row of 131072 with 20 alternatives
// Joins the parts of a row: one workgroup per row.  What counts is the time of one such call (one row of 131072 with 20
// alternatives: 13.5 us in all, 6.3 of them in the pass, 8.2 here, of which a launch and two trips to memory are 5), so parts
// and lists are asked for together and every wavefront forms the maximum and the border (from the lanes' maxima over four
// interleaved sets of parts each) for itself; its entries within the border go to LDS, and after the one barrier the first
// wavefront sorts them.
template <int SH> __global__ __launch_bounds__(JOIN_THREADS) void logprobs_join_kernel(LogitIn<SH> in, LogprobArgs A) {
    constexpr u32 K = 4, THREADS = JOIN_THREADS, E = 8192 / THREADS;
    __shared__ TopEntry buf[64];
    __shared__ u32 count;
    const u32 tid = threadIdx.x, lane = tid & 63;
    const u64 row = blockIdx.x;
    const u32 n = A.splits * 4, slots = A.top ? n * LIST : 0;
    const RowPart *parts = A.parts + row * n;
    const TopEntry *lists = A.lists + row * n * LIST;
    const u64 id = tid < A.per_row ? (u64)A.ids[row * A.per_row + tid] : A.vocab; // asked for early, used at the end
    TopEntry e[E];
#pragma unroll
    for (u32 k = 0; k < E; k++) {
        const u32 j = k * THREADS + tid;
        e[k] = j < slots ? lists[j] : TopEntry{INT64_MIN, TOP_NONE, 0};
    }
    RowSums s;
    i64 best[K];
#pragma unroll
    for (u32 k = 0; k < K; k++) best[k] = INT64_MIN;
    u32 any = 0;
    for (u32 p0 = 0; p0 < n; p0 += 64 * K) {
        RowPart o[K];
#pragma unroll
        for (u32 k = 0; k < K; k++) {
            const u32 p = p0 + 64 * k + lane;
            o[k] = p < n ? parts[p] : RowPart{INT64_MIN, 0.0f, 0.0f};
        }
#pragma unroll
        for (u32 k = 0; k < K; k++) {
            s.join(o[k], A.unit2);
            if (o[k].S > 0.0f) any |= 1u << k, best[k] = o[k].m > best[k] ? o[k].m : best[k];
        }
    }
    if (tid == 0) count = 0;
    const i64 at_id = id < A.vocab ? in.at(row * A.vocab + id) : 0;
    s.wave_join(A.unit2);
    float border = 0;
    if (A.top) {
        float near[K];
#pragma unroll
        for (u32 k = 0; k < K; k++) near[k] = (any >> k & 1) ? word_dist(s.m, best[k]) : -1.0f;
        border = top_border<K>(near, A.top, 16.0f / A.unit);
    }
    __syncthreads();
    for (u32 j0 = 0; j0 < slots; j0 += E * THREADS) {
        if (j0) {
#pragma unroll
            for (u32 k = 0; k < E; k++) {
                const u32 j = j0 + k * THREADS + tid;
                e[k] = j < slots ? lists[j] : TopEntry{INT64_MIN, TOP_NONE, 0};
            }
        }
#pragma unroll
        for (u32 k = 0; k < E; k++)
            if (e[k].i != TOP_NONE && word_dist(s.m, e[k].v) <= border) {
                const u32 at = atomicAdd(&count, 1u);
                if (at < 64) buf[at] = e[k];
            }
    }
    __syncthreads();
    if (tid < 64 && A.top) {
        WaveTop top(buf, A.top);
        if (count <= 64) {
            top.count = count;
        } else { // many equal words: all lists, one after the other
            for (u32 j = lane; j - lane < slots; j += 64) {
                const TopEntry q = j < slots ? lists[j] : TopEntry{INT64_MIN, TOP_NONE, 0};
                const i64 x[1] = {q.v};
                const u32 idx[1] = {q.i};
                const bool valid[1] = {q.i != TOP_NONE};
                top.add(x, idx, valid);
            }
        }
        top.sort();
    }
    logprobs_finish(in, A, row, s, buf, tid, THREADS, id, at_id);
}

// The gradient: reads the logits once and writes its floats or words, bound by that traffic (2048 rows of 32768 words of
// three shares into floats, 1.9 GB: 331 us, 5.7 TB/s; into ring words, 2.1 GB: 371 us, 5.8 TB/s).  TPR threads (a workgroup, or
// one wavefront of it for short rows) take `chunk` words of a row, 16 bytes of each share per load and GRAD_PAIRS of them
// together; the words of the given ids are written again at the end with their own terms added, so that the pass itself knows
// no ids and every word is rounded once; MANY: ids beyond a few dozen a row.
constexpr u32 GRAD_PAIRS = 4;
struct LogprobGradArgs {
    u64 rows, vocab, chunk;
    u32 splits;
    float unit, words; // 2^-frac, 2^grad_frac
    const i64 *ids;
    u64 per_row;
    const float *d_logp, *d_entropy;
    const i64 *row_max;
    const float *log_sum, *entropy;
    float *grad;
    i64 *grad_words;
};
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef f32x2 f32x2u __attribute__((aligned(4)));
constexpr u64 LP_GRAD_CHUNK = 512 * GRAD_PAIRS; // words of a row that a workgroup takes: one tile, see below
constexpr u64 LP_GRAD_WAVE_ROW = 768;           // longest row that one wavefront takes
// The sums of d_logp of equal ids, for rows of many ids: a wavefront goes once through the row's ids, in their order, and
// adds to a word of LDS for each of its words of the row.  64 ids at a time: where no two of them are the same (every lane
// leaves its number at its id's word, and finds it there) the lanes add together, else one after the other.
template <u32 WORDS> struct IdSums {
    float sum[WORDS];
    u32 lane_of[WORDS]; // the last lane that came by; NO_ID: no id at all
    static constexpr u32 NO_ID = ~0u;
    __device__ void clear(u32 t, u32 n) {
        for (u32 i = t; i < WORDS; i += n) sum[i] = 0, lane_of[i] = NO_ID;
    }
    __device__ void add(const i64 *ids, const float *dl, u64 count, u64 j0, u64 j1) {
        const u32 lane = threadIdx.x & 63;
        u64 next = lane < count ? (u64)ids[lane] : j1;
        float next_w = lane < count ? dl[lane] : 0.0f;
        for (u64 k0 = 0; k0 < count; k0 += 64) {
            const u64 id = next, k = k0 + 64 + lane;
            const float w = next_w;
            next = k < count ? (u64)ids[k] : j1, next_w = k < count ? dl[k] : 0.0f; // the next 64 are on their way
            const bool in = id >= j0 && id < j1;
            const u32 at = in ? (u32)(id - j0) : 0;
            if (in) lane_of[at] = lane;
            prg_wave_sync();
            if (__ballot(in && lane_of[at] != lane) == 0) {
                if (in) sum[at] += w;
            } else {
                for (u64 todo = __ballot(in); todo; todo &= todo - 1) {
                    if (lane == (u32)__builtin_ctzll(todo)) sum[at] += w;
                    prg_wave_sync();
                }
            }
            prg_wave_sync();
        }
    }
};
template <int SH, bool STREAM, u32 TPR, bool MANY = false>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(LogitIn<SH> in, LogprobGradArgs A) {
    __shared__ float ws[4];
    constexpr u32 WORDS = MANY ? (TPR == 64 ? LP_GRAD_WAVE_ROW : LP_GRAD_CHUNK) : 1;
    __shared__ IdSums<WORDS> sums[MANY ? 256 / TPR : 1];
    const u32 tid = threadIdx.x % TPR;
    const u64 group = (u64)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const u64 row = group / A.splits, split = group % A.splits, base = row * A.vocab;
    if (row >= A.rows) return; // TPR = 64: no barrier follows
    const u64 j0 = split * A.chunk, j1 = j0 + A.chunk < A.vocab ? j0 + A.chunk : A.vocab;
    const i64 m = A.row_max[row];
    const float ls = A.log_sum[row], h = A.d_entropy ? A.d_entropy[row] : 0.0f, H = A.d_entropy ? A.entropy[row] : 0.0f;
    const i64 *ids = A.ids + row * A.per_row;
    const float *dl = A.d_logp + row * A.per_row;
    float w = 0;
    for (u64 t = tid; t < A.per_row; t += TPR)
        if ((u64)ids[t] < A.vocab) w += dl[t];
    if (A.per_row > 1) {
        for (u32 d = 32; d; d >>= 1) w += __shfl_xor(w, (int)d);
        if (TPR > 64) {
            if ((tid & 63) == 0) ws[tid >> 6] = w;
            __syncthreads();
            w = ws[0] + ws[1] + ws[2] + ws[3];
        }
    } else if (A.per_row) {
        w = (u64)ids[0] < A.vocab ? dl[0] : 0.0f;
    }
    // - p w - h p (ln p + H); 0 where p is, whatever h ln p comes to
    auto part = [&](u64 x) {
        const float lp = -(word_dist(m, (i64)x) * A.unit + ls), p = expf(lp);
        return p == 0.0f ? 0.0f : -p * (w + h * (lp + H));
    };
    auto put1 = [&](u64 at, float g) {
        if (A.grad) A.grad[at] = g;
        if (A.grad_words) A.grad_words[at] = nearest_word(g * A.words);
    };
    auto put2 = [&](u64 at, u64x2 x) {
        const f32x2 g = {part(x.x), part(x.y)};
        if (A.grad) {
            if (STREAM) __builtin_nontemporal_store(g, (f32x2u *)(A.grad + at));
            else *(f32x2u *)(A.grad + at) = g;
        }
        if (A.grad_words) st2<STREAM>((u64 *)A.grad_words + at, u64x2{(u64)nearest_word(g.x * A.words), (u64)nearest_word(g.y * A.words)});
    };
    u64 tile = j0;
    for (; TPR > 64 && tile + 512 * GRAD_PAIRS <= j1; tile += 512 * GRAD_PAIRS) {
        const u64 at = base + tile + 2 * tid;
        u64x2 x[GRAD_PAIRS];
#pragma unroll
        for (u32 k = 0; k < GRAD_PAIRS; k++) x[k] = in.at2(at + 512 * k);
#pragma unroll
        for (u32 k = 0; k < GRAD_PAIRS; k++) put2(at + 512 * k, x[k]);
    }
    for (u64 j = tile + 2 * tid; j < j1; j += 2 * TPR) {
        if (j + 1 < j1) put2(base + j, in.at2(base + j));
        else put1(base + j, part((u64)in.at(base + j)));
    }
    if (A.per_row == 0) return;
    // a word of an id is written by another lane now: the stores above have to be done
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (TPR > 64) __syncthreads();
    else prg_wave_sync();
    if constexpr (MANY) {
        auto &mine = sums[threadIdx.x / TPR];
        mine.clear(tid, TPR);
        if (TPR > 64) __syncthreads();
        else prg_wave_sync();
        if (tid < 64) mine.add(ids, dl, A.per_row, j0, j1);
        if (TPR > 64) __syncthreads();
        for (u32 i = tid; i < j1 - j0; i += TPR)
            if (mine.lane_of[i] != mine.NO_ID) put1(base + j0 + i, mine.sum[i] + part((u64)in.at(base + j0 + i)));
        return;
    }
    for (u64 t = tid; t < A.per_row; t += TPR) {
        const u64 id = (u64)ids[t];
        if (id < j0 || id >= j1) continue;
        float g = 0; // equal ids write the same value
        for (u64 k = 0; k < A.per_row; k++)
            if ((u64)ids[k] == id) g += dl[k];
        g += part((u64)in.at(base + id));
        put1(base + id, g);
    }
}

// How a call is cut.  Fewer than LP_ROWS rows: a row is split over workgroups, LP_GROUPS of them in all (four on each CU),
// as long as each has LP_CHUNK words, one tile for each of its wavefronts (one row of 131072, 20 alternatives: 14 us, with
// 4096 words 19; 64 rows of 32000: 20 us, with 512 groups 33; 300 rows of 20000: 39 us against 31 unsplit, of 200000: 281
// against 289).  A row of up to 1024 words, or of up to LP_WAVE_ROW where the rows fill the chip, is read by one wavefront,
// others by four (300 rows of 500: 7.4 us against 8.8, of 1000: 9.7 against 8.8; 1024 rows of 1000: 10.6 against 11.2, of
// 1500: 14.8 against 12.8; 8192 rows of 500: 26 against 75, of 1500: 53 against 97; 2048 rows of 1500: 18.6 against 26, of
// 8000: 74 against 78, of 16000: 137 against 140).
constexpr u64 LP_ROWS = 256, LP_GROUPS = 1024, LP_CHUNK = 2048, LP_WAVE_ROW = 8192;
bool lp_one_wave(u64 rows, u64 vocab) { return vocab <= 1024 || (vocab <= LP_WAVE_ROW && rows >= 2048); }
// LP_GRAD_CHUNK, one tile: 2048 rows of 32768 words of three shares take 331 us with 2048 words (5.7 TB/s), 344 with 4096, 372
// with whole rows.  LP_GRAD_WAVE_ROW: 8192 rows of 500 21 us against 27 of a workgroup, of 1000 38 against 38.
// LP_GRAD_MANY: rows of more ids collect them in LDS (IdSums); up to it every id looks through the row's ids by itself, whose
// work grows with their square.  512 rows of 32768: 16 ids 37 us either way, 32 43 looking against 37, 256 264 against 49, 1024
// 3.7 ms against 87 us; 512 rows of 700: 32 ids 10.7 us against 11.6, 64 15.7 against 14.0; as many ids as words, 512 rows of
// 32768: 1.46 ms collected.
constexpr u64 LP_GRAD_MANY = 32;
template <int SH> int logprobs_run(mpcx_ctx *ctx, LogitIn<SH> in, LogprobArgs A) {
    const u64 all = A.rows;
    for (u64 r0 = 0; r0 < all; r0 += LM_MAX_BLOCKS) { // rows of one launch; more than one launch: nothing is split
        A.rows = all - r0 < LM_MAX_BLOCKS ? all - r0 : LM_MAX_BLOCKS;
        if (A.splits > 1)
            hipLaunchKernelGGL((logprobs_kernel<4, true, SH>), dim3((u32)(A.rows * A.splits)), dim3(256), 0, ctx->stream, in, A);
        else if (lp_one_wave(all, A.vocab))
            hipLaunchKernelGGL((logprobs_kernel<1, false, SH>), dim3((u32)ceil_div(A.rows, 4)), dim3(256), 0, ctx->stream, in, A);
        else
            hipLaunchKernelGGL((logprobs_kernel<4, false, SH>), dim3((u32)A.rows), dim3(256), 0, ctx->stream, in, A);
        MPCX_LAUNCH_CHECK();
        if (A.splits > 1) {
            hipLaunchKernelGGL(logprobs_join_kernel<SH>, dim3((u32)A.rows), dim3(JOIN_THREADS), 0, ctx->stream, in, A);
            MPCX_LAUNCH_CHECK();
        }
        in.skip(A.rows * A.vocab);
        auto skip = [&](auto *&p, u64 n) { p = p ? p + n : p; };
        skip(A.ids, A.rows * A.per_row), skip(A.logp, A.rows * A.per_row), skip(A.entropy, A.rows), skip(A.row_max, A.rows);
        skip(A.log_sum, A.rows), skip(A.top_ids, A.rows * A.top), skip(A.top_logp, A.rows * A.top);
    }
    return 0;
}

// scratch memory of the many-token form, in 8-byte words from its start
struct GradLayout {
    u64 total, count, start, rank, order, row, partial, words, rows, n;
    bool scan() const { return n <= GRAD_SCAN_N && rows <= GRAD_SCAN_ROWS; } // sorted by one launch, `rows` rows a workgroup
    GradLayout(u64 n_, u64 vocab, u64 dim) : rows(ceil_div(vocab, 256) < GRAD_ROWS ? GRAD_ROWS : ceil_div(vocab, 256)), n(n_) {
        u64 at = 0;
        auto take = [&](u64 &where, u64 bytes) { where = at, at += ceil_div(bytes, 16) * 2; };
        take(total, 16);
        take(count, 4 * vocab); // right behind the total: cleared together
        take(start, 4 * vocab);
        take(rank, scan() ? 0 : 4 * n);
        take(order, 4 * n);
        take(row, 4 * n);
        take(partial, n > GRAD_CHUNK ? ceil_div(n, GRAD_CHUNK) * 4 * dim * 8 : 0);
        words = at;
    }
};
template <bool TWO> int embed_grad_run(mpcx_ctx *ctx, const GradArgs &A, void *scratch) {
    const u64 slices = ceil_div(A.dim, 128);
    const u64 small_blocks = ceil_div(A.vocab, GRAD_ROWS) * slices;
    if (A.n <= GRAD_SMALL_N && A.n * small_blocks <= GRAD_SMALL_SCAN && small_blocks <= GRAD_SMALL_BLOCKS) {
        hipLaunchKernelGGL(embed_grad_small_kernel<TWO>, dim3((u32)ceil_div(A.vocab, GRAD_ROWS), (u32)slices), dim3(256), 0,
                           ctx->stream, A);
        MPCX_LAUNCH_CHECK();
        return 0;
    }
    const GradLayout L(A.n, A.vocab, A.dim);
    u64 *w = (u64 *)scratch;
    const GradWork W{(u32 *)(w + L.total), (u32 *)(w + L.count), (u32 *)(w + L.start), (u32 *)(w + L.rank), (u32 *)(w + L.order),
                     (u32 *)(w + L.row), w + L.partial};
    const u32 n = (u32)A.n;
    const u32 heavy_blocks = n <= GRAD_CHUNK ? 0 : A.n > A.vocab ? 1024 : 512; // otherwise no row is heavy
    const bool stream = (A.n + A.vocab) * A.dim * (TWO ? 16 : 8) > STREAM_BYTES;
    GradCut cut{};
    cut.heavy = heavy_blocks, cut.slices = (u32)slices, cut.by_place = A.accumulate && A.n < A.vocab;
    cut.row = RowCut(A.dim, 6, 1, stream, A.D0);
    const u64 blocks = heavy_blocks + lm_blocks(ceil_div((cut.by_place ? A.n : A.vocab) * cut.row.slices, 256u >> cut.row.lg));
    const u64 heavy_items = ceil_div(ceil_div(n, GRAD_CHUNK), HEAVY_WAVES) * slices;
    MPCX_REQUIRE(slices < (1ull << 32), "mpcx_ring_embed_grad: rows of %llu words", (unsigned long long)A.dim);
    if (L.scan()) {
        hipLaunchKernelGGL(grad_scan_kernel, dim3((u32)ceil_div(A.vocab, L.rows)), dim3(GRAD_SCAN_THREADS), 0, ctx->stream, A.ids, n,
                           A.vocab, (u32)L.rows, W);
    } else {
        const u32 vb = (u32)ceil_div(A.vocab, 256);
        hipLaunchKernelGGL(grad_clear_kernel, dim3(vb), dim3(256), 0, ctx->stream, W.total, 4 + A.vocab);
        if (n) hipLaunchKernelGGL(grad_count_kernel, dim3((u32)ceil_div(n, GRAD_TOKENS)), dim3(256), 0, ctx->stream, A.ids, n, A.vocab, W);
        hipLaunchKernelGGL(grad_place_kernel, dim3(vb), dim3(256), 0, ctx->stream, (u32)A.vocab, W);
        if (n) hipLaunchKernelGGL(grad_order_kernel, dim3((u32)ceil_div(n, 256)), dim3(256), 0, ctx->stream, A.ids, n, A.vocab, W);
    }
    if (blocks)
        hipLaunchKernelGGL((stream ? grad_rows_kernel<TWO, true> : grad_rows_kernel<TWO, false>), dim3((u32)blocks), dim3(256), 0,
                           ctx->stream, A, W, cut);
    if (heavy_blocks)
        hipLaunchKernelGGL(grad_heavy_kernel<TWO>, dim3((u32)lm_blocks(heavy_items)), dim3(64 * HEAVY_WAVES), 0, ctx->stream, A, W,
                           (u32)slices, heavy_items);
    MPCX_LAUNCH_CHECK();
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
    const bool stream = n * dim * (T1 ? 32 : 16) > STREAM_BYTES;
    const RowCut cut(dim, 8, emb_steps(T1), stream, E0);
    MPCX_REQUIRE(cut.slices < 65536, "mpcx_ring_embed: rows of %llu words", (unsigned long long)dim);
    const dim3 grid((u32)lm_blocks(ceil_div(n, 256u >> cut.lg)), (u32)cut.slices), block(256);
    const auto kernel = T1 ? (stream ? embed_kernel<true, true> : embed_kernel<true, false>)
                           : (stream ? embed_kernel<false, true> : embed_kernel<false, false>);
    hipLaunchKernelGGL(kernel, grid, block, 0, ctx->stream, (const u64 *)T0, (const u64 *)T1, vocab, dim, ids, n, (u64)scale, shift,
                       (u64 *)E0, (u64 *)E1, cut);
    MPCX_LAUNCH_CHECK();
    return 0;
}

uint64_t mpcx_ring_embed_grad_scratch(uint64_t n, uint64_t vocab, uint64_t dim) { return 8 * GradLayout(n, vocab, dim).words; }
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
    const GradArgs A{(const u64 *)G0, (const u64 *)G1, ids, n, vocab, dim, (u64)scale, shift, accumulate, (u64 *)dT0, (u64 *)dT1};
    return dT1 ? embed_grad_run<true>(ctx, A, scratch) : embed_grad_run<false>(ctx, A, scratch);
}

// the next tensors of a call, from tensor `i` on, as one launch's table; advances i and out
static TensorTable tensor_table(const int64_t *const *X0, const int64_t *const *X1, const uint64_t *lens, u64 count, u64 &i,
                                u64 &out) {
    TensorTable tab;
    tab.count = 0, tab.tiles = 0;
    for (; i < count && tab.count < LM_TENSORS; i++) {
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
        const TensorTable tab = tensor_table(X0, X1, lens, count, i, out);
        if (tab.count == 0) continue;
        const u32 grid = tensor_grid(tab);
        hipLaunchKernelGGL(sqnorm_kernel, dim3(grid), dim3(256), 0, ctx->stream, tab, part + parts);
        MPCX_LAUNCH_CHECK();
        parts += grid;
    }
    hipLaunchKernelGGL(sqnorm_join_kernel, dim3(1), dim3(parts <= 2048 ? 256 : 1024), 0, ctx->stream, part, parts, ckA, ckB, tA, tB, (u64 *)z0);
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
        const u64 first = out;
        TensorTable tab = tensor_table(X0, party == 1 ? X1 : nullptr, lens, count, i, out);
        if (tab.count == 0) continue;
        if (party == 1) {
            for (u32 k = 0; k < tab.count; k++) tab.t[k].out -= first;
            MPCX_TRY(prg_map1(ctx, seed12, PRG_POP_T0 + pop12 + first, out - first, ClipMasked{tab, coef, number, Y + first}));
        } else {
            hipLaunchKernelGGL(clip_kernel, dim3((u32)lm_blocks(tab.tiles)), dim3(256), 0, ctx->stream, tab, A, coef, Y);
            MPCX_LAUNCH_CHECK();
        }
    }
    return 0;
}

// words of a row that one workgroup reads
static u64 logprob_chunk(u64 rows, u64 vocab) {
    u64 splits = rows >= LP_ROWS ? 1 : LP_GROUPS / (rows ? rows : 1);
    if (splits > ceil_div(vocab, LP_CHUNK)) splits = ceil_div(vocab, LP_CHUNK);
    return ceil_div(ceil_div(vocab, splits ? splits : 1), 2048) * 2048;
}
uint64_t mpcx_reveal_logprobs_scratch(uint64_t rows, uint64_t vocab, uint64_t top) {
    if (vocab >= (1ull << 31)) return 16; // the call refuses it
    const u64 splits = vocab ? ceil_div(vocab, logprob_chunk(rows, vocab)) : 1;
    return splits > 1 ? rows * splits * 4 * (sizeof(RowPart) + (top ? LIST * sizeof(TopEntry) : 0)) : 16;
}
int mpcx_reveal_logprobs(mpcx_ctx *ctx, const int64_t *a, const int64_t *b, const int64_t *c, uint64_t rows, uint64_t vocab,
                         int frac, const int64_t *ids, uint64_t per_row, uint64_t top, void *scratch, float *logp,
                         float *entropy, int64_t *top_ids, float *top_logp, int64_t *row_max, float *log_sum) {
    MPCX_REQUIRE((vocab >= 1 || rows == 0) && vocab < (1ull << 31), "mpcx_reveal_logprobs: vocabulary of %llu", (unsigned long long)vocab);
    MPCX_REQUIRE(lm_fits(rows, vocab) && lm_fits(rows, per_row), "mpcx_reveal_logprobs: sizes too large");
    MPCX_REQUIRE(frac >= 0 && frac <= 62, "mpcx_reveal_logprobs: %d fractional bits", frac);
    MPCX_REQUIRE(top <= 32 && (top <= vocab || rows == 0), "mpcx_reveal_logprobs: %llu alternatives", (unsigned long long)top);
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
    A.parts = (RowPart *)scratch, A.lists = (TopEntry *)(A.parts + rows * A.splits * 4);
    return c ? logprobs_run<3>(ctx, {(const u64 *)a, (const u64 *)b, (const u64 *)c}, A)
         : b ? logprobs_run<2>(ctx, {(const u64 *)a, (const u64 *)b, nullptr}, A)
             : logprobs_run<1>(ctx, {(const u64 *)a, nullptr, nullptr}, A);
}

int mpcx_reveal_logprobs_grad(mpcx_ctx *ctx, const int64_t *a, const int64_t *b, const int64_t *c, uint64_t rows,
                              uint64_t vocab, int frac, const int64_t *ids, uint64_t per_row, const float *d_logp,
                              const float *d_entropy, const int64_t *row_max, const float *log_sum, const float *entropy,
                              float *grad, int64_t *grad_words, int grad_frac) {
    MPCX_REQUIRE((vocab >= 1 || rows == 0) && vocab < (1ull << 31), "mpcx_reveal_logprobs_grad: vocabulary of %llu", (unsigned long long)vocab);
    MPCX_REQUIRE(lm_fits(rows, vocab) && lm_fits(rows, per_row), "mpcx_reveal_logprobs_grad: sizes too large");
    MPCX_REQUIRE(frac >= 0 && frac <= 62, "mpcx_reveal_logprobs_grad: %d fractional bits", frac);
    MPCX_REQUIRE(!grad_words || (grad_frac >= 0 && grad_frac <= 62), "mpcx_reveal_logprobs_grad: %d fractional bits", grad_frac);
    MPCX_REQUIRE(b || !c, "mpcx_reveal_logprobs_grad: the third share without the second");
    if (rows == 0) return 0;
    MPCX_REQUIRE(a && row_max && log_sum && (grad || grad_words) && (per_row == 0 || (ids && d_logp)) && (!d_entropy || entropy),
                 "mpcx_reveal_logprobs_grad: NULL pointer");
    MPCX_REQUIRE(ctx, "mpcx_reveal_logprobs_grad: the context is NULL");
    LogprobGradArgs A{};
    A.vocab = vocab, A.chunk = LP_GRAD_CHUNK, A.splits = (u32)ceil_div(vocab, A.chunk);
    A.unit = ldexpf(1.0f, -frac), A.words = ldexpf(1.0f, grad_words ? grad_frac : 0);
    A.ids = ids, A.per_row = per_row, A.d_logp = d_logp, A.d_entropy = d_entropy;
    A.row_max = row_max, A.log_sum = log_sum, A.entropy = entropy, A.grad = grad, A.grad_words = grad_words;
    const bool stream = rows * vocab * ((c ? 24 : b ? 16 : 8) + (grad ? 4 : 0) + (grad_words ? 8 : 0)) > STREAM_BYTES;
    const bool one_wave = A.splits == 1 && vocab <= LP_GRAD_WAVE_ROW;
    auto run = [&](auto kernel, auto in) -> int {
        const u64 batch = LM_MAX_BLOCKS / A.splits; // rows of one launch
        for (u64 r0 = 0; r0 < rows; r0 += batch) {
            const u64 now = rows - r0 < batch ? rows - r0 : batch;
            A.rows = now;
            hipLaunchKernelGGL(kernel, dim3((u32)ceil_div(now * A.splits, one_wave ? 4 : 1)), dim3(256), 0, ctx->stream, in, A);
            MPCX_LAUNCH_CHECK();
            in.skip(now * vocab);
            auto skip = [&](auto *&p, u64 n) { p = p ? p + n : p; };
            skip(A.ids, now * per_row), skip(A.d_logp, now * per_row), skip(A.d_entropy, now), skip(A.row_max, now);
            skip(A.log_sum, now), skip(A.entropy, now), skip(A.grad, now * vocab), skip(A.grad_words, now * vocab);
        }
        return 0;
    };
    const u64 *pa = (const u64 *)a, *pb = (const u64 *)b, *pc = (const u64 *)c;
    const bool many = per_row > LP_GRAD_MANY;
    auto pick = [&](auto in, auto whole, auto streaming, auto wave, auto many_whole, auto many_wave) {
        return run(many ? (one_wave ? many_wave : many_whole) : one_wave ? wave : stream ? streaming : whole, in);
    };
    if (c)
        return pick(LogitIn<3>{pa, pb, pc}, logprobs_grad_kernel<3, false, 256>, logprobs_grad_kernel<3, true, 256>,
                    logprobs_grad_kernel<3, false, 64>, logprobs_grad_kernel<3, false, 256, true>, logprobs_grad_kernel<3, false, 64, true>);
    if (b)
        return pick(LogitIn<2>{pa, pb, nullptr}, logprobs_grad_kernel<2, false, 256>, logprobs_grad_kernel<2, true, 256>,
                    logprobs_grad_kernel<2, false, 64>, logprobs_grad_kernel<2, false, 256, true>, logprobs_grad_kernel<2, false, 64, true>);
    return pick(LogitIn<1>{pa, nullptr, nullptr}, logprobs_grad_kernel<1, false, 256>, logprobs_grad_kernel<1, true, 256>,
                logprobs_grad_kernel<1, false, 64>, logprobs_grad_kernel<1, false, 256, true>, logprobs_grad_kernel<1, false, 64, true>);
}

} // extern "C"
