// Fused scaled-dot-product attention with a learned relative position bias, bf16, head_dim 64, on the packed projection
// qkv[b, S, 3*H*64], forward and backward.
//
//   s_ij = scale * <q_i, k_j> + T[bucket(j - i), h],   p = softmax_j(s),   o_i = sum_j p_ij v_j,   lse_i = log sum_j exp s_ij
//   ds_ij = p_ij (<do_i, v_j> - delta_i),  delta_i = <do_i, o_i>
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//   dT[u, h] = sum over the batch and all visible pairs with bucket(j - i) = u of ds_ij
//
// bucket() depends on the relative position only and is constant from distance R = the last bucket's first distance on, so
// a head's bias is a vector over the window [-R, R], which every block expands into LDS once.  The vector is kept divided
// by `scale` and handed to the QK matrix instructions as their initial accumulator: the bias costs LDS reads and no vector
// arithmetic.  The score layout is that of the kernels without a bias (each lane owns one query column in forward and dQ,
// one key column in dK / dV; consecutive registers are consecutive keys / queries, so a lane's window reads are runs of
// four consecutive words and the 32 columns of a half wave read 32 consecutive addresses).
//
// dT: ds_ij is summed along the diagonals j - i of a 32 x 32 score block in registers: the 63 diagonals fit the 64 lanes, the
// rows of the block are added one after the other to a vector that moves up by one lane between two rows (a DPP wave
// shift that rides on the addition), so that lane l always holds the diagonal (row) - l.  A row's 32 columns have to lie in
// lanes 0 .. 31 with zeros above: the swap of half waves delivers that for the two rows of an accumulator register at
// once.  That is 4 vector instructions a register, and no atomics: LDS float additions of the 16 registers cost 180 cycles
// each on this chip (the dQ kernel of [12, 512] x 16 heads took 274 us with them and 46 us without; 38 us by now).  The vector is
// added to the wave's own window in LDS; the block adds its four windows and sums the buckets' ranges, the dK / dV kernel adds the blocks, all in a
// fixed order: the same bits every time.
//
// Roundings.  Scores, statistics, sums and accumulators are float32.  Probabilities and score gradients are rounded to bf16 where they
// become operands of a matrix instruction (P before PV and dV, dS before dQ and dK), as in the kernels without a bias: a float32 or split
// operand would take three or more times the matrix work.  Each is off by 2^-8 of itself at most, independently of the
// others, so a result carries its own rounding to bf16 once more (norm-wise 1.7e-3 from the operands next to 1.7e-3 of the result's own:
// 2.2e-3 .. 2.4e-3 measured against float64).  The sum of weights adds the unrounded ones: rounded ones would shift lse, which backward takes for exact.  The table's
// gradient adds unrounded dS.
#include <atomic>

#include "common.h"
#include "attention_tile.h"

namespace {

constexpr float LN2 = 0.6931471805599453f;
constexpr int REL_MAX_SIDE = HAPMI_RELBIAS_MAX_SIDE;
constexpr int REL_MAX_REACH = HAPMI_RELBIAS_MAX_REACH;
// A 64 x 32 block of scores spans 95 diagonals: the window carries this many saturated entries on either side, and the
// offset of a block that lies wholly beyond the window is clamped so that it reads nothing else.
constexpr int MARGIN = 95;
// A bias at or below this hides the pair (the type's lowest value included).  float32 scores of that size are multiples of 8, and
// a log-sum-exp of them is good to 1e8 * 2^-22 = 24: up to here weights made from it stay inside the exponentials' range (2^34),
// further down they would not.
constexpr float HIDDEN = -1e8f;

struct RelArgs {
    const float *table;                       // [buckets, ld], column = head
    int64_t ld;
    int side, bidir, R;                       // buckets per side; R: first distance of the last bucket, or S - 1 if that is less; >= 1
    int starts[REL_MAX_SIDE];                 // first distance of every bucket of a side, starts[0] = 0; then INT32_MAX
    // has the starts' cache lines come with the kernel's other arguments: the search would wait for them later ([1, 128] x 4 heads: forward
    // 5.8 us for 6.2, dK / dV 7.8 for 8.2; in dQ, where other loads are under way meanwhile, no effect)
    __device__ __forceinline__ void touch() const { asm volatile("" ::"s"(starts[0]), "s"(starts[15]), "s"(starts[31]), "s"(starts[47]), "s"(starts[63])); }
    __device__ __forceinline__ int window() const { return 2 * R + 1 + 2 * MARGIN; }
    __device__ __forceinline__ int bucket(int d) const {      // of a side, for a distance
        int k = -1;
        for (int i = 0; i < side; i += 16) {                  // sixteen at a time: one wait for the scalar loads
#pragma unroll
            for (int j = 0; j < 16; ++j) k += d >= starts[i + j] ? 1 : 0;
        }
        return k;
    }
    // relative positions lo .. hi of the window that belong to bucket u (none: lo > hi)
    __device__ __forceinline__ void range(int u, int &lo, int &hi) const {
        int first = 0, next = R + MARGIN + 1;                 // distances of the bucket: first .. next - 1
        const int k = bidir && u >= side ? u - side : u;
        for (int i = 0; i < side; i += 16) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {                    // (starts[] is indexed by the loops only: scalar loads)
                if (i + j == k) first = starts[i + j];
                if (i + j == k + 1 && k + 1 < side) next = starts[i + j];
            }
        }
        if (next > R + MARGIN + 1) next = R + MARGIN + 1;
        if (bidir && u >= side) { lo = first < 1 ? 1 : first; hi = next - 1; }
        else { lo = -(next - 1); hi = first == 0 ? (bidir || next < 1 ? 0 : R + MARGIN) : -first; }
        if (first >= next) { lo = 1; hi = 0; }
    }
    // the head's bias / scale over the window; REV: entry i belongs to relative position -(i - R - MARGIN); CAUSAL: keys behind
    // the query are hidden
    template <bool REV, bool CAUSAL> __device__ __forceinline__ void expand(float *win, int head, float scale) const {
        auto put = [&](int i, float t, bool hidden) { win[i] = t <= HIDDEN || hidden ? -INFINITY : t / scale; };
        const int mid = R + MARGIN, same = bidir ? 0 : bucket(0);
        for (int d = threadIdx.x; d <= mid; d += AT_THREADS) {              // both positions at a distance: one search, both loads at once
            const int k = bucket(d < R ? d : R), before = k, after = bidir ? (d > 0 ? k + side : k) : same;
            const float tb = table[(int64_t)before * ld + head], ta = table[(int64_t)after * ld + head];
            put(REV ? mid + d : mid - d, tb, false);
            if (d > 0) put(REV ? mid - d : mid + d, ta, CAUSAL);
        }
    }
    // word of the window that the lane's row 0 of a block of ROWS x 32 scores reads; D = first row - first column
    template <int ROWS> __device__ __forceinline__ int at(int D, int c, int h) const {
        D = D < -R - (ROWS - 1) ? -R - (ROWS - 1) : (D > R + 31 ? R + 31 : D);
        return D + R + MARGIN + 4 * h - c;
    }
};

// A [64 rows][64 d] tile global -> LDS like DirectTileLoader's, for the many tiles of a kernel that lie wholly inside the
// operand: the lane's byte offsets inside a tile never change, the tile's first row is a scalar base, and a transfer costs no
// vector arithmetic.  A tile that ends inside repeats the operand's last row.
struct TileStream {
    static constexpr int LOADS = 2;                           // wave instructions a tile: rows 0 .. 31 and 32 .. 63
    int off, ld;
    __device__ __forceinline__ static int row(int tid) { return (tid >> 6) * 8 + ((tid & 63) >> 3); }
    __device__ __forceinline__ static int chunk(int tid) { return ((tid & 7) ^ aswz(row(tid))) * 16; }        // (32 rows on the same)
    __device__ __forceinline__ TileStream(int ld_) : off(row(threadIdx.x) * ld_ * 2 + chunk(threadIdx.x)), ld(ld_) {}
    __device__ __forceinline__ void issue(const bf16_t *base, int rows_left, char *lds_tile) const {
        typedef __attribute__((address_space(3))) char lds_char;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t lds_addr = (uint32_t)(uintptr_t)(lds_char *)lds_tile + wave * 1024;
        int o[LOADS] = {off, off};
        const bf16_t *from[LOADS] = {base, base + 32 * ld};
        if (__builtin_expect(rows_left < TILE, 0)) {
            int tid = threadIdx.x;
            asm volatile("" : "+v"(tid));                     // (nothing of this is kept in registers over the whole tiles)
            from[1] = base;
#pragma unroll
            for (int i = 0; i < LOADS; ++i)
                o[i] = (row(tid) + i * 32 < rows_left ? row(tid) + i * 32 : rows_left - 1) * ld * 2 + chunk(tid);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                         :
                         : "s"(lds_addr + i * 4096), "v"(o[i]), "s"(from[i])
                         : "memory");
    }
};

// The wave's own 32 rows of 64, the operand that stays in its registers, come through LDS as well: a transfer reads whole 128-byte
// rows, where a fragment read from memory touches 32 bytes of 32 rows.  The wave waits for its transfers (vmcnt) and needs no
// barrier.  Rows from `rows` on repeat the last one, and are replaced by zeros when they are read.
__device__ __forceinline__ void issue_own_rows(const bf16_t *first_row, int ld, int rows, char *lds) {
    typedef __attribute__((address_space(3))) char lds_char;
    if (rows <= 0) return;
    const int lane = threadIdx.x & 63;
    const uint32_t lds_addr = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_char *)lds);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 3);
        const int off = (r < rows ? r : rows - 1) * ld * 2 + ((lane & 7) ^ aswz(r)) * 16;
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(lds_addr + i * 1024), "v"(off), "s"(first_row)
                     : "memory");
    }
}
__device__ __forceinline__ void own_frags(const char *lds, int c, int h, int rows, frag_t (&f)[4]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) f[s] = frag_rowk(lds, c, s, h);
    if (rows >= 32) return;
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const u32x4 bits = __builtin_bit_cast(u32x4, f[s].v);
        f[s].v = __builtin_bit_cast(bf16x8, c < rows ? bits : (u32x4)(0u));
    }
}

// A wave adds to its window of ds sums by load, add and store, and a word that one lane adds to belongs to another lane in the next
// addition: the order of the accesses counts although no thread meets its own word again.  The wave's LDS accesses are carried out
// in their order; this keeps the compiler from moving a load above the store before it.
__device__ __forceinline__ void window_order() { asm volatile("" ::: "memory"); }

// the same in all lanes, in a scalar register
__device__ __forceinline__ float uniform(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }

// initial accumulator of a 32 x 32 score block: rows of the block are runs of four words
__device__ __forceinline__ f32x16 bias_tile(const float *w) {
    f32x16 a;
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[g * 4 + e] = w[g * 8 + e];
    return a;
}

// sums of a 32 x 32 block along its diagonals: lane l gets the sum over (row, column) with row - column = 31 - l
__device__ __forceinline__ float diagonal_sums(const f32x16 &x) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    float y = 0.f;
    auto step = [&](uint32_t row) {                           // one more row: up by one lane, zero into lane 0
        const int up = __builtin_amdgcn_update_dpp(0, __float_as_int(y), 0x138, 0xf, 0xf, true);   // wave_shr:1
        y = __int_as_float(up) + __uint_as_float(row);
    };
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        u32x2 rows[4];                                        // .x: row 8 g + e, .y: row 8 g + 4 + e, in lanes 0 .. 31
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[g * 4 + e]), 0u, false, false);
            rows[e].x = r[0];
            rows[e].y = r[1];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) step(rows[e].x);
#pragma unroll
        for (int e = 0; e < 4; ++e) step(rows[e].y);
    }
    return y;
}

__device__ __forceinline__ float both_halves_max(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A wave's 32 rows of 64 results, held as accumulators of the transposed product (lane (c, h): row c, register i of half u: column
// u * 32 + acc_row(i, h)), to memory by whole 128-byte rows: through 4 KB of LDS of the wave's own, so that no barrier is needed.
// Stored from the registers, 8 bytes a lane, it takes 8 instructions that touch 32 rows each: the forward, dQ and dK / dV
// kernels of [12, 512] x 16 heads took 25.1, 44.2 and 41.6 us then, and 24.1, 43.4 and 38.8 us this way.
template <typename F> __device__ __forceinline__ void store_rows(char *lds, bf16_t *first_row, int ld, int rows, F value) {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));                            // (no address of this is worth a register before)
    const int c = lane & 31, h = lane >> 5;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            bf16x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (bf16_t)value(u, g * 4 + e);
            *(bf16x4 *)(lds + c * 128 + ((u * 4 + g) ^ (c & 7)) * 16 + h * 8) = o;
        }
    asm volatile("" ::: "memory");                            // (a wave's LDS accesses are carried out in their order)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 3);
        const bf16x8 o = *(const bf16x8 *)(lds + r * 128 + ((lane & 7) ^ (r & 7)) * 16);
        if (r < rows) *(bf16x8 *)(first_row + (int64_t)r * ld + (lane & 7) * 8) = o;
    }
}

// Which 128-row block of which (batch, head) a thread block takes.  Blocks are dealt round-robin over the 8 XCDs in the order
// of their linear index; the row blocks of one (batch, head) stream the same tiles, so they go to one XCD, next to each
// other in time.  Neighbouring heads go to different XCDs: in a padded batch they have the same length, and a long sample
// would otherwise land on one XCD (dK / dV of lengths 334 .. 1001 in [6, 1001] x 12 heads: 62 us with a contiguous eighth of the heads on
// each XCD, 44 us so).  Causal: the row blocks with the most work start first (BlockOrder), which keeps a head on its XCD too.
template <bool CAUSAL> struct Order {
    int blk, bh;
    __device__ __forceinline__ Order(bool work_grows_with_index) {
        if (CAUSAL) {
            blk = BlockOrder<true>::row_block(work_grows_with_index);
            bh = BlockOrder<true>::batch_head();
        } else {
            const int gx = (int)gridDim.x, l = (int)(blockIdx.y * gridDim.x + blockIdx.x), even = (int)gridDim.y / 8 * 8;
            const int turn = l < even * gx ? l / 8 : l;
            blk = turn % gx;
            bh = l < even * gx ? turn / gx * 8 + l % 8 : turn / gx;
        }
    }
};

__device__ __forceinline__ int row_length(const int32_t *lengths, int b, int S) {
    if (!lengths) return S;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > S ? S : n);
}

// ---------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------
// One pass over the keys with a running maximum and sum; a wave holds 32 queries, a block of four waves 128, and the 64-key
// tiles pass through three LDS stages, so that a transfer has two tiles' arithmetic to arrive in.  Three blocks a CU: all 768
// of the encoder shape are resident at once (two blocks where the bias window takes the room, which is given out in pieces of 1280 bytes:
// R above 480, encoder shape 28 -> 30.4 us; with dropout above 96).
// A score costs a multiply-add, an exponential (two multiply-adds' time, measured: 3.8 ns a wave instruction for 2.0 with four waves a
// SIMD), an addition, half a maximum and half a conversion, 20 cycles of the vector pipe, against 16 of the matrix pipe; masks, window
// reads, the running maximum and the operands' addresses come on top.
// [12, 512] x 16 heads: 24 us, 0.54 PFLOP/s, vector pipe 58 % and matrix pipe 28 % of the cycles (8 us of it fixed: launch, prologue,
// results), with dropout 30 us; [6, 1001] x 12 heads of 334 .. 1001 tokens: 28 us; [1, 8192] x 16 heads, causal: 164 .. 185 us as
// the power limit lets it, 0.80 PFLOP/s of the visible half, vector pipe 70 %, matrix pipe 41 %, HBM 67 + 17 MB.
// Without effect or worse: four parallel chains for the maximum, products pinned between the exponentials (184 for 177 us), no
// maximum unless a sum of weights gets large (198 us: the test stands between the exponentials and the products), the next tile's
// scores between this one's exponentials with two waves a SIMD (0 to 5 % slower even where the card is half empty).
template <bool CAUSAL, bool DROP>
__global__ __launch_bounds__(AT_THREADS, 3) void relbias_fwd_kernel(const RelArgs rel, const bf16_t *qkv, bf16_t *out, float *lse,
                                                               const int32_t *lengths, int S, int H, float scale,
                                                               const uint32_t *keep_rows, float keep_scale) {
    constexpr int NST = 3;                                    // one tile is multiplied while two are on their way
    __shared__ __attribute__((aligned(16))) char Ks3[NST][TILE_BYTES];
    __shared__ __attribute__((aligned(16))) char Vs3[NST][TILE_BYTES];
    __shared__ __attribute__((aligned(16))) uint32_t keep_s[DROP ? NST : 1][AT_THREADS];
    extern __shared__ __attribute__((aligned(16))) float win[];
    rel.touch();
    const TransposedReader tr;
    const int W = rel.window();
    const int E = H * HD, ld = 3 * E;
    const Order<CAUSAL> order(true);
    const int blk = order.blk, bh = order.bh;
    const int b = bh / H, hh = bh % H;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int n = row_length(lengths, b, S);
    const int qw = blk * 128 + wave * 32, q = qw + c;
    const bf16_t *Q = qkv + (int64_t)b * S * ld + hh * HD;
    const bf16_t *K = Q + E, *V = Q + 2 * E;

    const int q_blk_end = blk * 128 + 128;
    const int kv_end = blk * 128 >= n ? 0 : ((CAUSAL && q_blk_end < n) ? q_blk_end : n);
    f32x16 ot[2] = {zero16(), zero16()};
    float m = -INFINITY, lsum = 0.f;                          // running maximum in units of log 2
    if (kv_end > 0) {
        const TileStream ldr(ld);
        const float sl2 = uniform(scale * LOG2E);
        constexpr int PER_TILE = 2 * TileStream::LOADS + (DROP ? 1 : 0);
        static_assert(2 * TileStream::LOADS == 4, "the waits below are written for four (five) transfers per tile");
        const int n_kt = (S + TILE - 1) / TILE;
        const uint32_t *keep_row = DROP ? keep_rows + ((int64_t)bh * S + (q < S ? q : S - 1)) * n_kt * 2 + h : nullptr;
        auto issue_tile = [&](int kv0, int bufi) {
            ldr.issue(K + (int64_t)kv0 * ld, n - kv0, Ks3[bufi]);
            ldr.issue(V + (int64_t)kv0 * ld, n - kv0, Vs3[bufi]);
            if constexpr (DROP) issue_word(keep_row + (kv0 / TILE) * 2, &keep_s[bufi][0]);
        };
        // the queries come through the third stage, which takes its first tile behind the loop's first barrier
        char *own = (wave < 2 ? Ks3[2] : Vs3[2]) + (wave & 1) * 4096;
        issue_own_rows(Q + (int64_t)qw * ld, ld, n - qw, own);
        issue_tile(0, 0);
        rel.expand<false, CAUSAL>(win, hh, scale);            // published by the first barrier of the loop
        __builtin_amdgcn_s_waitcnt(0x0F70);                   // vmcnt(0): queries and first tile have landed
        if (TILE < kv_end) issue_tile(TILE, 1);
        frag_t qf[4];
        own_frags(own, c, h, n - qw, qf);
        int buf = 0;
        for (int kv0 = 0; kv0 < kv_end; kv0 += TILE) {
            if (kv0 + TILE < kv_end) __builtin_amdgcn_s_waitcnt(0x0070 | 0x0F00 | PER_TILE);   // vmcnt: only the next tile may be outstanding
            else __builtin_amdgcn_s_waitcnt(0x0F70);                                           // vmcnt(0)
            __syncthreads();
            if (kv0 + 2 * TILE < kv_end) issue_tile(kv0 + 2 * TILE, buf == 0 ? 2 : buf - 1);
            const char *Ks = Ks3[buf], *Vs = Vs3[buf];
            buf = buf == NST - 1 ? 0 : buf + 1;
            if (CAUSAL && kv0 > qw + 31) continue;            // the wave's queries see none of the tile's keys
            uint32_t keep = 0xffffffffu;
            if constexpr (DROP) keep = keep_s[buf == 0 ? NST - 1 : buf - 1][threadIdx.x];
            const bool whole = kv0 + TILE <= n;
            const bool far_hi = kv0 - qw - 31 >= rel.R, far_lo = kv0 - qw + 63 <= -rel.R;
            // all fragment reads of a group are issued before its first MFMA waits for one, and those of V before the
            // softmax arithmetic, which hides them
            frag_t kf[2][4], vf[2][4];
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int t = 0; t < 2; ++t) kf[t][s] = frag_rowk(Ks, t * 32 + c, s, h);
            f32x16 st[2];
            float shift = 0.f;                                // bias of a tile beyond the window, in units of log 2
            if (whole && (far_hi || far_lo)) {
                shift = win[far_hi ? W - 1 : 0] * sl2;
                __builtin_amdgcn_sched_barrier(0);
                st[0] = zero16();
                st[1] = zero16();
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int t = 0; t < 2; ++t) st[t] = mma(kf[t][s], qf[s], st[t]);
            } else {
                const float *w = win + rel.at<64>(kv0 - qw, c, h);
                st[0] = bias_tile(w);
                st[1] = bias_tile(w + 32);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int t = 0; t < 2; ++t) st[t] = mma(kf[t][s], qf[s], st[t]);
                if (__builtin_expect(!whole, 0)) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (kv0 + t * 32 + acc_row(r, h) >= n) st[t][r] = -INFINITY;
                }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int u = 0; u < 2; ++u) vf[u][s] = tr.frag(Vs, u * 32, s);
            __builtin_amdgcn_sched_barrier(0);
            float mx = st[0][0];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, st[t][r]);
            mx = both_halves_max(mx);
            // The subtracted maximum only has to keep the exponentials in range: it moves when some query's has grown by more than
            // 2^8 (or was -inf), and the accumulators are rescaled then.  Probabilities stay below 2^8 until then, which costs no
            // precision: both roundings are relative.
            const float m_tile = fmaf(mx, sl2, shift);
            if (__builtin_amdgcn_ballot_w64(m_tile > m + 8.f)) {
                const float m_new = fmaxf(m, m_tile), alpha = __builtin_amdgcn_exp2f(m - (m_new == -INFINITY ? 0.f : m_new));
                m = m_new;
                lsum *= alpha;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 16; ++r) ot[u][r] *= alpha;
            }
            const float off = shift - (m == -INFINITY ? 0.f : m);
            float psum = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(st[t][r], sl2, off));
                    st[t][r] = p;
                    psum += p;
                }
            lsum += psum;
            if constexpr (DROP) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int r = 0; r < 16; ++r) st[t][r] = (keep & (1u << (t * 16 + r))) ? st[t][r] : 0.f;
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const frag_t pb = acc_to_b(st[s >> 1], s & 1);
#pragma unroll
                for (int u = 0; u < 2; ++u) ot[u] = mma(vf[u][s], pb, ot[u]);
            }
        }
    }
    const float l = lsum + __shfl_xor(lsum, 32, 64);
    const bool seen = q < n && l > 0.f;                       // a padded query, or one that sees nothing: zeros, lse = -inf
    const float inv = seen ? (DROP ? keep_scale : 1.f) / l : 0.f;
    __syncthreads();                                          // everybody is done with the tiles
    store_rows(Ks3[0] + wave * 4096, out + ((int64_t)b * S + qw) * E + hh * HD, E, S - qw,
               [&](int u, int i) { return l != l ? l : (seen ? ot[u][i] * inv : 0.f); });
    if (q < S && h == 0) lse[((int64_t)b * H + hh) * S + q] = q < n ? m * LN2 + logf(l) : -INFINITY;
}

// ---------------------------------------------------------------------------------------------
// dQ and the bias gradient: lanes own query columns, kv tiles are streamed
// ---------------------------------------------------------------------------------------------
// 13 matrix products and about 80 vector instructions a lane for a 32 x 32 block of scores, 64 more where it touches the bias
// window (the diagonal sums).  Three waves a SIMD hide each other's latencies; where the launch does not fill the card, two
// that also work on the next block's scores are faster (AHEAD; ahead_holds has both sides).  [12, 512] x 16 heads: 38 us,
// matrix pipe 28 %, vector pipe 51 %, HBM 64 + 14 MB, a quarter of the time before the first tile and behind the last one;
// [2, 4096] x 16 heads, causal: 137 .. 142 us, matrix pipe 44 %, vector pipe 61 %.
// The plain form with the full mask needs one register more than the 168 of three waves a SIMD: 8 bytes a lane go to scratch.
__host__ __device__ __forceinline__ int round4(int n) { return (n + 3) & ~3; }
// a window, and the waves' sums, whose room their dO rows pass through first
__host__ __device__ __forceinline__ int dq_lds_words(int W) { return round4(W) + (W > 1024 ? 4 * round4(W) : 4096); }

template <bool CAUSAL, bool DROP, bool AHEAD>
__global__ __launch_bounds__(AT_THREADS, AHEAD ? 2 : 3) void relbias_bwd_dq_kernel(const RelArgs rel, const bf16_t *qkv, const bf16_t *out,
                                                                  const bf16_t *dout, const float *lse, float *delta,
                                                                  bf16_t *dqkv, float *part, const int32_t *lengths, int S,
                                                                  int H, float scale, const uint32_t *keep_rows,
                                                                  float keep_scale) {
    static_assert(!(DROP && AHEAD), "the mask keeps delta out of the products");
    constexpr int NST = AHEAD ? 3 : 2;
    __shared__ __attribute__((aligned(16))) char Kst[NST][TILE_BYTES];
    __shared__ __attribute__((aligned(16))) char Vst[NST][TILE_BYTES];
    __shared__ int ranges[2 * REL_MAX_SIDE][2];               // the buckets' first and last relative position in the window
    extern __shared__ __attribute__((aligned(16))) float win[];             // the bias window, then the four waves' windows of ds sums
    const TransposedReader tr;
    const int W = rel.window();
    const int E = H * HD, ld = 3 * E;
    const Order<CAUSAL> order(true);
    const int blk = order.blk, bh = order.bh;
    const int b = bh / H, hh = bh % H;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int n = row_length(lengths, b, S);
    const int qw = blk * 128 + wave * 32, q = qw + c;
    const bool qok = q < n;
    const bf16_t *Q = qkv + (int64_t)b * S * ld + hh * HD;
    const bf16_t *K = Q + E, *V = Q + 2 * E;
    const bf16_t *dO = dout + (int64_t)b * S * E + hh * HD;
    const int q_blk_end = blk * 128 + 128;
    const int kv_end = blk * 128 >= n ? 0 : ((CAUSAL && q_blk_end < n) ? q_blk_end : n);
    const int WS = round4(W), n_buckets = rel.side << rel.bidir;
    float *sums = win + WS, *own = sums + wave * WS;
    auto set_ranges = [&]() {
        if ((int)threadIdx.x < n_buckets) rel.range(threadIdx.x, ranges[threadIdx.x][0], ranges[threadIdx.x][1]);
    };
    auto clear_own = [&]() {
        for (int i = lane * 4; i < WS; i += 256) *(f32x4 *)(own + i) = (f32x4)(0.f);
    };
    f32x16 dqt[2] = {zero16(), zero16()};
    float far_sum[2] = {0.f, 0.f};                            // blocks wholly before / behind the window
    if (kv_end > 0) {
        const TileStream ldr(ld);
        // queries through the second stage, dO through the room of the ds sums
        char *own_q = (wave < 2 ? Kst[1] : Vst[1]) + (wave & 1) * 4096, *own_do = (char *)sums + wave * 4096;
        issue_own_rows(Q + (int64_t)qw * ld, ld, n - qw, own_q);
        issue_own_rows(dO + (int64_t)qw * E, E, n - qw, own_do);
        ldr.issue(K, n, Kst[0]);
        ldr.issue(V, n, Vst[0]);
        const float lse_q = qok ? lse[((int64_t)b * H + hh) * S + q] : -INFINITY;
        const bf16_t *O = out + ((int64_t)b * S + qw) * E + hh * HD;
        frag_t of[4];                                         // row i * 8 + lane / 8, columns 8 (lane % 8) ..
#pragma unroll
        for (int i = 0; i < 4; ++i) of[i] = load_row_frag(O + (int64_t)(i * 8 + (lane >> 3)) * E + (lane & 7) * 8, qw + i * 8 + (lane >> 3) < n, 0, 0);
        set_ranges();
        rel.expand<false, CAUSAL>(win, hh, scale);            // published by the loop's first barrier
        __builtin_amdgcn_s_waitcnt(0x0F70);                   // vmcnt(0): queries, dO and the first tile have landed
        frag_t qf[4], dof[4];
        own_frags(own_q, c, h, n - qw, qf);
        own_frags(own_do, c, h, n - qw, dof);
        float delta_q = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = i * 8 + (lane >> 3);
            const frag_t dr = *(const frag_t *)(own_do + r * ROW_BYTES + (((lane & 7) ^ aswz(r)) << 4));
            float v = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v += (float)of[i].v[e] * (float)dr.v[e];
            v = qw + r < n ? group_sum(v, 3) : 0.f;
            if (qw + r < n && (lane & 7) == 0) delta[((int64_t)b * H + hh) * S + qw + r] = v;
            const float mine = __shfl(v, (c & 7) * 8, 64);    // rows 8 i .. + 7 to their columns
            if (c >> 3 == i) delta_q = mine;
        }
        __syncthreads();                                      // everybody has read its dO: the room is the sums' now
        clear_own();
        // ds is kept without its factor `scale`; a query that sees nothing (lse = -inf) has p = 0
        const float sl2 = uniform(scale * LOG2E), nl = lse_q == -INFINITY ? -INFINITY : -lse_q * LOG2E;
        if constexpr (AHEAD) {
            // One block's score products stand between the vector instructions of the block before it; dP's accumulators start from
            // -delta, the scores' from the bias.
            __syncthreads();                                  // the window and the first tile are there
            auto fetch = [&](int kv0, int bufi) {
                ldr.issue(K + (int64_t)kv0 * ld, n - kv0, Kst[bufi]);
                ldr.issue(V + (int64_t)kv0 * ld, n - kv0, Vst[bufi]);
            };
            if (TILE < kv_end) fetch(TILE, 1);
            int buf = 0, nbuf = 1;
            f32x16 minus_delta, sc0, dp0, sc1, dp1;
#pragma unroll
            for (int r = 0; r < 16; ++r) minus_delta[r] = -delta_q;
            frag_t ka[4], va[4];
            auto read_frag = [&](int bufi, int t, int s) {
                ka[s] = frag_rowk(Kst[bufi], t * 32 + c, s, h);
                va[s] = frag_rowk(Vst[bufi], t * 32 + c, s, h);
            };
            // first reads for the scores of block (nb, nt) of the tile at nk0
            auto prepare = [&](f32x16 &xs, int nb, int nt, int nk0) {
                xs = bias_tile(win + rel.at<32>(nk0 + nt * 32 - qw, c, h));
                read_frag(nb, nt, 0);
                read_frag(nb, nt, 1);
                __builtin_amdgcn_sched_barrier(0);
            };
            // dS, dQ and the table's sums of block (cbuf, t) at key k0, whose scores and dP - delta are in (sc, dp), and the scores of
            // block (nb, nt) into (xs, xd).  Behind the last block that is some old tile's data, whose result nobody uses.
            auto block = [&](f32x16 &sc, f32x16 &dp, f32x16 &xs, f32x16 &xd, int cbuf, int t, int k0, int nb, int nt) {
                const char *Ks = Kst[cbuf];
                if (__builtin_expect(k0 + 32 > n, 0)) {                            // keys behind the end
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (k0 + acc_row(r, h) >= n) sc[r] = -INFINITY;
                }
                auto score = [&](int r) { dp[r] *= __builtin_amdgcn_exp2f(fmaf(sc[r], sl2, nl)); };
                auto next_scores = [&](int s) { xs = mma(ka[s], qf[s], xs); };
                frag_t kt[2];
#pragma unroll
                for (int r = 0; r < 4; ++r) score(r);
                next_scores(0);
                score(4);
                score(5);
                xd = mma(va[0], dof[0], minus_delta);
                score(6);
                score(7);
                frag_t db = acc_to_b(dp, 0);
#pragma unroll
                for (int u = 0; u < 2; ++u) kt[u] = tr.frag(Ks, u * 32, t * 2);
                read_frag(nb, nt, 2);
                next_scores(1);
                score(8);
                score(9);
                xd = mma(va[1], dof[1], xd);
                read_frag(nb, nt, 3);
                score(10);
                dqt[0] = mma(kt[0], db, dqt[0]);
                score(11);
                kt[0] = tr.frag(Ks, 0, t * 2 + 1);
                dqt[1] = mma(kt[1], db, dqt[1]);
                score(12);
                kt[1] = tr.frag(Ks, 32, t * 2 + 1);
                next_scores(2);
                score(13);
                xd = mma(va[2], dof[2], xd);
                score(14);
                score(15);
                db = acc_to_b(dp, 1);
                next_scores(3);
                xd = mma(va[3], dof[3], xd);
#pragma unroll
                for (int u = 0; u < 2; ++u) dqt[u] = mma(kt[u], db, dqt[u]);
                const int D = k0 - qw;
                const bool far_hi = D - 31 >= rel.R, far_lo = D + 31 <= -rel.R;
                if (far_hi || far_lo) {
                    float sum = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) sum += dp[r];
                    far_sum[far_hi ? 1 : 0] += sum;
                } else {
                    const float sums_of_lane = diagonal_sums(dp);
                    window_order();
                    own[rel.at<32>(D, 0, 0) + 31 - lane] += sums_of_lane;
                    window_order();
                }
            };
            sc0 = bias_tile(win + rel.at<32>(-qw, c, h));
            dp0 = minus_delta;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                read_frag(0, 0, s);
                sc0 = mma(ka[s], qf[s], sc0);
                dp0 = mma(va[s], dof[s], dp0);
            }
            prepare(sc1, 0, 1, 0);
            for (int kv0 = 0; kv0 < kv_end; kv0 += TILE) {
                block(sc0, dp0, sc1, dp1, buf, 0, kv0, buf, 1);
                const int fbuf = nbuf == NST - 1 ? 0 : nbuf + 1;
                __builtin_amdgcn_s_waitcnt(0x0F70);           // vmcnt(0): the next tile has landed
                __syncthreads();                              // for everybody, and everybody is done with the tile before this one
                if (kv0 + 2 * TILE < kv_end) fetch(kv0 + 2 * TILE, fbuf);
                prepare(sc0, nbuf, 0, kv0 + TILE);
                block(sc1, dp1, sc0, dp0, buf, 1, kv0 + 32, nbuf, 0);
                prepare(sc1, nbuf, 1, kv0 + TILE);
                buf = nbuf;
                nbuf = fbuf;
            }
        } else {
            // dP - delta in the matrix pipe: a product of ones (every key row) and -delta_q cut into three bf16 terms, which hold all 24
            // bits of it; one matrix instruction a block in place of 16 subtractions a lane
            frag_t ones, minus_delta;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                ones.v[e] = (bf16_t)1.f;
                minus_delta.v[e] = (bf16_t)0.f;
            }
            if (h == 0) {
                float rest = -delta_q;
#pragma unroll
                for (int e = 0; e < 3; ++e) {
                    minus_delta.v[e] = (bf16_t)rest;
                    rest -= (float)minus_delta.v[e];
                }
            }
            const uint32_t *keep_row = DROP ? keep_rows + ((int64_t)bh * S + (q < S ? q : S - 1)) * ((S + TILE - 1) / TILE) * 2 + h : nullptr;
            uint32_t keep = 0xffffffffu, keep_next = 0xffffffffu;
            if constexpr (DROP) keep_next = keep_row[0];
            int buf = 0;
            for (int kv0 = 0; kv0 < kv_end; kv0 += TILE) {
                __builtin_amdgcn_s_waitcnt(0x0F70);               // vmcnt(0): the tile has landed
                __syncthreads();                                  // for everybody, and everybody is done with the other buffer
                if constexpr (DROP) keep = keep_next;
                if (kv0 + TILE < kv_end) {
                    const int nx = kv0 + TILE;
                    ldr.issue(K + (int64_t)nx * ld, n - nx, Kst[buf ^ 1]);
                    ldr.issue(V + (int64_t)nx * ld, n - nx, Vst[buf ^ 1]);
                    if constexpr (DROP) keep_next = keep_row[(nx / TILE) * 2];
                }
                const char *Ks = Kst[buf], *Vs = Vst[buf];
                buf ^= 1;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int k0 = kv0 + t * 32, D = k0 - qw;
                    if (qw >= n || k0 >= n || (CAUSAL && D > 31)) continue;        // nothing here that any query sees
                    const bool whole = k0 + 32 <= n;
                    const bool far_hi = D - 31 >= rel.R, far_lo = D + 31 <= -rel.R;
                    f32x16 st, dp = zero16();
                    frag_t db[2];
                    frag_t kf[4], vf[4];
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        kf[s] = frag_rowk(Ks, t * 32 + c, s, h);
                        vf[s] = frag_rowk(Vs, t * 32 + c, s, h);
                    }
                    auto products = [&]() {                       // every group of reads is issued before the arithmetic that hides it
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int s = 0; s < 4; ++s) {
                            st = mma(kf[s], qf[s], st);
                            dp = mma(vf[s], dof[s], dp);
                        }
                        if constexpr (DROP) {                     // (the mask is applied before delta is subtracted)
#pragma unroll
                            for (int r = 0; r < 16; ++r) dp[r] = ((keep & (1u << (t * 16 + r))) ? dp[r] * keep_scale : 0.f) - delta_q;
                        } else {
                            dp = mma(ones, minus_delta, dp);
                        }
                    };
                    if (whole && (far_hi || far_lo)) {            // one bucket for the whole block
                        st = zero16();
                        products();
                        const float off = nl + win[far_hi ? W - 1 : 0] * sl2;
                        float sum = 0.f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            dp[r] *= __builtin_amdgcn_exp2f(fmaf(st[r], sl2, off));
                            sum += dp[r];
                        }
                        far_sum[far_hi ? 1 : 0] += sum;
                        db[0] = acc_to_b(dp, 0);
                        db[1] = acc_to_b(dp, 1);
                    } else {
                        const int at = rel.at<32>(D, c, h);
                        st = bias_tile(win + at);
                        products();
                        if (__builtin_expect(!whole, 0)) {
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                if (k0 + acc_row(r, h) >= n) st[r] = -INFINITY;
                        }
#pragma unroll
                        for (int r = 0; r < 16; ++r) dp[r] *= __builtin_amdgcn_exp2f(fmaf(st[r], sl2, nl));
                        db[0] = acc_to_b(dp, 0);
                        db[1] = acc_to_b(dp, 1);
                        asm volatile("" : "+v"(db[0].v), "+v"(db[1].v));      // rounded here: the sums below then need no copies of dp
                        // lane l of the sums: diagonal (last row) - l; `at` is row 0's word of column c
                        const float sums_of_lane = diagonal_sums(dp);
                        window_order();
                        own[at - 4 * h + c + 31 - lane] += sums_of_lane;
                        window_order();
                    }
#pragma unroll
                    for (int sp = 0; sp < 2; ++sp) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) dqt[u] = mma(tr.frag(Ks, u * 32, t * 2 + sp), db[sp], dqt[u]);
                    }
                }
            }
        }
        const float lo = group_sum(far_sum[0], 6), hi = group_sum(far_sum[1], 6);
        window_order();
        if (lane == 0) {
            own[0] += lo;
            own[W - 1] += hi;
        }
    }
    if (kv_end == 0) {
        clear_own();
        set_ranges();
    }
    // the block's bucket sums: window words over the four waves, then every bucket's range by a group of eight lanes
    __syncthreads();                                          // (everybody is done with the tiles, too)
    store_rows(Kst[0] + wave * 4096, dqkv + ((int64_t)b * S + qw) * ld + hh * HD, ld, S - qw,
               [&](int u, int i) { return qok ? dqt[u][i] * scale : 0.f; });
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));                            // addresses below are not worth registers in the loop above
    for (int i = tid * 4; i < WS; i += AT_THREADS * 4)
        *(f32x4 *)(win + i) = ((*(const f32x4 *)(sums + i) + *(const f32x4 *)(sums + WS + i)) + *(const f32x4 *)(sums + 2 * WS + i)) +
                              *(const f32x4 *)(sums + 3 * WS + i);
    __syncthreads();
    float *mine = part + ((int64_t)bh * ((S + 127) / 128) + blk) * n_buckets;
    for (int u = tid >> 3; u < n_buckets; u += AT_THREADS / 8) {
        const int lo = ranges[u][0] + rel.R + MARGIN, hi = ranges[u][1] + rel.R + MARGIN;
        float v = 0.f;
        for (int i = lo + (tid & 7); i <= hi; i += 32) {          // four reads under way at once
            float w4[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w4[j] = i + j * 8 <= hi ? win[i + j * 8] : 0.f;
            v += (w4[0] + w4[1]) + (w4[2] + w4[3]);
        }
        v = group_sum(v, 3);
        if ((tid & 7) == 0) mine[u] = v;
    }
}

// dT[u, head] (+)= the dQ blocks' sums part[b][H][row blocks][buckets], in order, by one block of the dK / dV kernel for each
// head: AT_THREADS / buckets threads share a bucket, each over every so many-th block, their sums added in order.
__device__ __forceinline__ void table_gradient(const float *part, float *dtable, int64_t ldd, int n_buckets, int b, int H, int head, int row_blocks,
                                              int accumulate, float *red) {
    const int u = threadIdx.x % n_buckets, run = threadIdx.x / n_buckets, runs = AT_THREADS / n_buckets;
    if (run < runs) {
        float v = 0.f;
        const int items = b * row_blocks;                     // (b H <= 65535 and row_blocks < 2^17: fits)
#pragma unroll 8
        for (int i = run; i < items; i += runs) v += part[(((int64_t)(i / row_blocks) * H + head) * row_blocks + i % row_blocks) * n_buckets + u];
        red[threadIdx.x] = v;
    }
    __syncthreads();
    if (run == 0) {
        float v = 0.f;
        for (int i = 0; i < runs; ++i) v += red[i * n_buckets + u];
        float *d = dtable + (int64_t)u * ldd + head;
        *d = accumulate ? *d + v : v;
    }
}

// ---------------------------------------------------------------------------------------------
// dK, dV: lanes own kv columns, query tiles are streamed
// ---------------------------------------------------------------------------------------------
// A wave works on one 32 x 32 block of scores at a time: 8 matrix products for the scores and dP, 80 vector instructions a
// lane for P and dS, 8 products for dV and dK.  Two waves fit a SIMD, so the wave itself has to keep the matrix pipe fed:
// the score products of the NEXT block and the first half of this block's dV / dK products stand one by one between the
// instructions of this block, and three tiles are kept in LDS because the next block may be the next tile's.  Everything that
// would be a branch a block is data: causally hidden pairs are -inf in the bias window, queries beyond the end carry
// lse = +inf, and dP starts from -delta.  Plain blocks with three waves a SIMD instead: 36.9 us for 37.3 on [12, 512] x 16 heads,
// but 29.0 for 25.2 us on [8, 512] and 88 for 74 us on [2, 2048].  What it spends adds up rather than overlaps (leaving out the
// matrix products 108 of 182 us on [4, 2048], the LDS reads 138, the exponentials 178).  [12, 512] x 16 heads: 38 us, 0.68
// PFLOP/s, matrix pipe 34 %, vector pipe 40 %, LDS 39 %, HBM 51 + 25 MB; [2, 4096] x 16 heads, causal: 153 .. 167 us, matrix
// pipe 47 %, vector pipe 46 %, LDS 49 %.
template <bool CAUSAL, bool DROP>
__global__ __launch_bounds__(AT_THREADS, 2) void relbias_bwd_dkv_kernel(const RelArgs rel, const bf16_t *qkv, const bf16_t *dout,
                                                                   const float *lse, const float *delta, bf16_t *dqkv,
                                                                   const int32_t *lengths, int S, int H, float scale,
                                                                   const uint32_t *keep_cols, float keep_scale, const float *part,
                                                                   float *dtable, int64_t ldd, int n_buckets, int batch, int accumulate) {
    constexpr int NST = 3;
    __shared__ __attribute__((aligned(16))) char Qs3[NST][TILE_BYTES];
    __shared__ __attribute__((aligned(16))) char dOs3[NST][TILE_BYTES];
    __shared__ __attribute__((aligned(16))) float lse_s[NST][TILE], delta_s[NST][TILE];
    extern __shared__ __attribute__((aligned(16))) float win[];
    rel.touch();
    const TransposedReader tr;
    const int E = H * HD, ld = 3 * E;
    const Order<CAUSAL> order(false);
    const int blk = order.blk, bh = order.bh;
    const int b = bh / H, hh = bh % H;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int n = row_length(lengths, b, S);
    const int kvw = blk * 128 + wave * 32, kv = kvw + c;
    const bool kok = kv < n;
    const bf16_t *Q = qkv + (int64_t)b * S * ld + hh * HD;
    const bf16_t *K = Q + E, *V = Q + 2 * E;
    const bf16_t *dO = dout + (int64_t)b * S * E + hh * HD;
    const float *lse_b = lse + ((int64_t)b * H + hh) * S, *delta_b = delta + ((int64_t)b * H + hh) * S;
    f32x16 dvt[2] = {zero16(), zero16()}, dkt[2] = {zero16(), zero16()};
    if (blk * 128 < n) {
        const TileStream lq(ld), ldo(E);
        const float sl2 = uniform(scale * LOG2E);
        const int q_begin = CAUSAL ? blk * 128 : 0;           // causal: earlier queries see none of the block's keys
        typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
        const u32x2 *keep_col = DROP ? (const u32x2 *)(keep_cols + ((int64_t)bh * S + (kv < S ? kv : S - 1)) * (2 * ((S + TILE - 1) / TILE))) : nullptr;
        u32x2 keep2 = {0u, 0u}, keep2_next = keep2;
        // a query's log-sum-exp times log2 e (+inf where it sees nothing: p = 0) and its -delta (with dropout +delta, which
        // then is subtracted behind the mask)
        float l_next = 0.f, d_next = 0.f;
        auto fetch = [&](int q0, int bufi) {
            lq.issue(Q + (int64_t)q0 * ld, n - q0, Qs3[bufi]);
            ldo.issue(dO + (int64_t)q0 * E, n - q0, dOs3[bufi]);
            if constexpr (DROP) keep2_next = keep_col[q0 / TILE];
            if (threadIdx.x < TILE) {
                const int qq = q0 + threadIdx.x;
                l_next = qq < n ? lse_b[qq] : -INFINITY;
                d_next = qq < n ? delta_b[qq] : 0.f;
            }
        };
        auto stage = [&](int bufi) {
            if (threadIdx.x < TILE) {
                lse_s[bufi][threadIdx.x] = l_next == -INFINITY ? INFINITY : l_next * LOG2E;
                delta_s[bufi][threadIdx.x] = DROP ? d_next : -d_next;
            }
        };
        // keys and values through the stages that take no tile before the barrier below
        issue_own_rows(K + (int64_t)kvw * ld, ld, n - kvw, Qs3[1] + wave * 4096);
        issue_own_rows(V + (int64_t)kvw * ld, ld, n - kvw, dOs3[1] + wave * 4096);
        fetch(q_begin, 0);
        rel.expand<true, CAUSAL>(win, hh, scale);
        stage(0);
        if constexpr (DROP) keep2 = keep2_next;
        __builtin_amdgcn_s_waitcnt(0x0F70);                   // vmcnt(0): keys, values and the first tile have landed
        frag_t kf[4], vf[4];
        own_frags(Qs3[1] + wave * 4096, c, h, n - kvw, kf);
        own_frags(dOs3[1] + wave * 4096, c, h, n - kvw, vf);
        __syncthreads();
        int buf = 0, nbuf = 1;
        if (q_begin + TILE < n) fetch(q_begin + TILE, 1);

        // sixteen row values of a lane's block, in register order
        auto row_values = [&](const float *rows, int t) {
            f32x16 y;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 r4 = *(const f32x4 *)(rows + t * 32 + g * 8 + h * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[g * 4 + e] = r4[e];
            }
            return y;
        };
        if constexpr (DROP) {
            // The mask keeps delta out of the products and needs the keep words, and the look-ahead below then spills (backward of
            // [12, 512] x 16 heads with dropout: 134 us with it, 102 us with these plain blocks when that was tried, 88 us by now).
            for (int q0 = q_begin; q0 < n; q0 += TILE) {
                const char *Qs = Qs3[buf], *dOs = dOs3[buf];
#pragma unroll 1
                for (int t = 0; t < 2; ++t) {
                    if (kvw >= n || q0 + t * 32 >= n || (CAUSAL && q0 + t * 32 + 31 < kvw)) continue;
                    f32x16 sc = bias_tile(win + rel.at<32>(q0 + t * 32 - kvw, c, h)), dp = zero16();
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        sc = mma(frag_rowk(Qs, t * 32 + c, s, h), kf[s], sc);
                        dp = mma(frag_rowk(dOs, t * 32 + c, s, h), vf[s], dp);
                    }
                    const uint32_t keep = t ? keep2.y : keep2.x;
                    const f32x16 l = row_values(lse_s[buf], t), d = row_values(delta_s[buf], t);
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float p = __builtin_amdgcn_exp2f(fmaf(sc[r], sl2, -l[r]));
                        const bool kp = keep & (1u << acc_row(r, h));
                        dp[r] = p * ((kp ? dp[r] * keep_scale : 0.f) - d[r]);
                        sc[r] = kp ? p * keep_scale : 0.f;
                    }
#pragma unroll
                    for (int sp = 0; sp < 2; ++sp) {
                        const frag_t pb = acc_to_b(sc, sp), db = acc_to_b(dp, sp);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            dvt[u] = mma(tr.frag(dOs, u * 32, t * 2 + sp), pb, dvt[u]);
                            dkt[u] = mma(tr.frag(Qs, u * 32, t * 2 + sp), db, dkt[u]);
                        }
                    }
                }
                const int fbuf = nbuf == NST - 1 ? 0 : nbuf + 1;
                if (q0 + TILE < n) {
                    stage(nbuf);
                    keep2 = keep2_next;
                }
                __builtin_amdgcn_s_waitcnt(0x0F70);           // vmcnt(0): the next tile has landed
                __syncthreads();                              // for everybody, and everybody is done with the tile before this one
                if (q0 + 2 * TILE < n) fetch(q0 + 2 * TILE, fbuf);
                buf = nbuf;
                nbuf = fbuf;
            }
        } else {
            f32x16 sc0, dp0, sc1, dp1;
            frag_t qa[4], da[4];
            auto read_frag = [&](int bufi, int t, int s) {
                qa[s] = frag_rowk(Qs3[bufi], t * 32 + c, s, h);
                da[s] = frag_rowk(dOs3[bufi], t * 32 + c, s, h);
            };
            // a block's accumulators before its products: the bias, -delta
            auto read_start = [&](int bufi, int t, int q0, f32x16 &x, f32x16 &y) {
                x = bias_tile(win + rel.at<32>(q0 + t * 32 - kvw, c, h));
                y = row_values(delta_s[bufi], t);
            };
            // P, dS, dV, dK of block (cbuf, t) whose scores and dP - delta are in (sc, dp), and the scores of block (nb, nt) of the
            // query tile at nq0 into (xs, xd).  Behind the last block that is some old tile's data, whose result nobody uses.
            f32x4 l4, l4n;                                        // log-sum-exps of the four rows being worked on, and of the next four
            auto stats = [&](int cbuf, int t, int g) { return *(const f32x4 *)(lse_s[cbuf] + t * 32 + h * 4 + g * 8); };
            // first reads for block (cbuf, t) and for the scores of block (nb, nt), issued behind the products of the block before
            auto prepare = [&](f32x16 &xs, f32x16 &xd, int cbuf, int t, int nb, int nt, int nq0) {
                l4 = stats(cbuf, t, 0);
                l4n = stats(cbuf, t, 1);
                read_start(nb, nt, nq0, xs, xd);
                read_frag(nb, nt, 0);
                read_frag(nb, nt, 1);
                __builtin_amdgcn_sched_barrier(0);
            };
            auto block = [&](f32x16 &sc, f32x16 &dp, f32x16 &xs, f32x16 &xd, int cbuf, int t, int nb, int nt) {
                const char *Qs = Qs3[cbuf], *dOs = dOs3[cbuf];
                auto score = [&](int r) {                         // P and dS of score register r
                    const float p = __builtin_amdgcn_exp2f(fmaf(sc[r], sl2, -l4[r & 3]));
                    dp[r] = p * dp[r];
                    sc[r] = p;
                };
                auto next_scores = [&](int s) { xs = mma(qa[s], kf[s], xs); };
                auto next_dp = [&](int s) { xd = mma(da[s], vf[s], xd); };
#pragma unroll
                for (int r = 0; r < 4; ++r) score(r);
                l4 = l4n;
                l4n = stats(cbuf, t, 2);
                next_scores(0);
                score(4);
                score(5);
                next_dp(0);
                score(6);
                score(7);
                frag_t pb = acc_to_b(sc, 0), db = acc_to_b(dp, 0), dt[2], qt[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    dt[u] = tr.frag(dOs, u * 32, t * 2);
                    qt[u] = tr.frag(Qs, u * 32, t * 2);
                }
                l4 = l4n;
                l4n = stats(cbuf, t, 3);
                read_frag(nb, nt, 2);
                next_scores(1);
                score(8);
                next_dp(1);
                score(9);
                read_frag(nb, nt, 3);
                dvt[0] = mma(dt[0], pb, dvt[0]);
                score(10);
                dkt[0] = mma(qt[0], db, dkt[0]);
                dt[0] = tr.frag(dOs, 0, t * 2 + 1);
                qt[0] = tr.frag(Qs, 0, t * 2 + 1);
                score(11);
                l4 = l4n;
                next_scores(2);
                score(12);
                dvt[1] = mma(dt[1], pb, dvt[1]);
                score(13);
                dkt[1] = mma(qt[1], db, dkt[1]);
                dt[1] = tr.frag(dOs, 32, t * 2 + 1);
                qt[1] = tr.frag(Qs, 32, t * 2 + 1);
                score(14);
                next_dp(2);
                score(15);
                pb = acc_to_b(sc, 1);
                db = acc_to_b(dp, 1);
                next_scores(3);
                next_dp(3);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    dvt[u] = mma(dt[u], pb, dvt[u]);
                    dkt[u] = mma(qt[u], db, dkt[u]);
                }
            };
            read_start(0, 0, q_begin, sc0, dp0);
#pragma unroll
            for (int s = 0; s < 4; ++s) read_frag(0, 0, s);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                sc0 = mma(qa[s], kf[s], sc0);
                dp0 = mma(da[s], vf[s], dp0);
            }
            prepare(sc1, dp1, 0, 0, 0, 1, q_begin);
            for (int q0 = q_begin; q0 < n; q0 += TILE) {
                block(sc0, dp0, sc1, dp1, buf, 0, buf, 1);
                const int fbuf = nbuf == NST - 1 ? 0 : nbuf + 1;
                if (q0 + TILE < n) stage(nbuf);
                __builtin_amdgcn_s_waitcnt(0x0F70);               // vmcnt(0): the next tile has landed
                __syncthreads();                                  // for everybody, and everybody is done with the tile before this one
                if (q0 + 2 * TILE < n) fetch(q0 + 2 * TILE, fbuf);
                prepare(sc0, dp0, buf, 1, nbuf, 0, q0 + TILE);
                block(sc1, dp1, sc0, dp0, buf, 1, nbuf, 0);
                prepare(sc1, dp1, nbuf, 0, nbuf, 1, q0 + TILE);
                buf = nbuf;
                nbuf = fbuf;
            }
        }
    }
    __syncthreads();                                          // everybody is done with the tiles
    bf16_t *drow = dqkv + ((int64_t)b * S + kvw) * ld + hh * HD;
    store_rows(Qs3[0] + wave * 4096, drow + E, ld, S - kvw, [&](int u, int i) { return kok ? dkt[u][i] * scale : 0.f; });
    store_rows(dOs3[0] + wave * 4096, drow + 2 * E, ld, S - kvw, [&](int u, int i) { return kok ? dvt[u][i] : 0.f; });
    if (b == 0 && blk == (int)gridDim.x - 1) {                // (with the causal mask the block with the least work)
        __syncthreads();
        table_gradient(part, dtable, ldd, n_buckets, batch, H, hh, (int)gridDim.x, accumulate, win);
    }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
int window_of(int R) { return 2 * R + 1 + 2 * MARGIN; }

int check_rel(const char *name, const hapmi_relbias *r, int64_t S, int64_t H, RelArgs *a) {
    HAPMI_REQUIRE(r && r->starts_host, HAPMI_EINVAL, "%s: null bias description", name);
    const int sides = r->bidirectional ? 2 : 1;
    HAPMI_REQUIRE(r->n_buckets >= 2 && r->n_buckets % sides == 0, HAPMI_EINVAL, "%s: %d buckets: at least 2, and even for two sides", name,
                  r->n_buckets);
    a->side = r->n_buckets / sides;
    HAPMI_REQUIRE(a->side <= REL_MAX_SIDE, HAPMI_ELIMIT, "%s: %d buckets on a side, at most %d", name, a->side, REL_MAX_SIDE);
    HAPMI_REQUIRE(r->starts_host[0] == 0, HAPMI_EINVAL, "%s: the first bucket must start at distance 0", name);
    for (int i = 0; i < a->side; ++i) {
        a->starts[i] = r->starts_host[i];
        HAPMI_REQUIRE(i == 0 || a->starts[i] >= a->starts[i - 1], HAPMI_EINVAL, "%s: the buckets' first distances must not fall", name);
    }
    for (int i = a->side; i < REL_MAX_SIDE; ++i) a->starts[i] = INT32_MAX;
    const int last = a->starts[a->side - 1];
    HAPMI_REQUIRE(last <= REL_MAX_REACH, HAPMI_ELIMIT, "%s: the last bucket starts at distance %d, at most %d", name, last, REL_MAX_REACH);
    a->bidir = r->bidirectional ? 1 : 0;
    // no pair is further apart than S - 1: a shorter window serves (dQ of [1, 128] x 2 heads, 64 buckets to 1000: 15.2 us with the
    // whole reach, 12.4 so)
    a->R = (int)(last < S - 1 ? last : S - 1);
    if (a->R < 1) a->R = 1;
    a->table = r->table;
    a->ld = r->ld;
    HAPMI_REQUIRE(r->ld >= H, HAPMI_EINVAL, "%s: table rows of %lld for %lld heads", name, (long long)r->ld, (long long)H);
    return HAPMI_OK;
}

int check_shape(const char *name, int64_t b, int64_t S, int64_t H, float scale, float p) {
    HAPMI_REQUIRE(b >= 0 && S >= 1 && H >= 1, HAPMI_EINVAL, "%s: bad shape", name);
    HAPMI_REQUIRE(S < (1ll << 24) && H <= 4096 && b <= 65535 / H, HAPMI_ELIMIT, "%s: b * H above 65535, H above 4096 or S too long", name);
    HAPMI_REQUIRE(scale > 0.f && scale < INFINITY, HAPMI_EINVAL, "%s: scale = %g must be positive", name, (double)scale);
    // the window holds bias / scale in float32: 1e8 / 1e-20 is far inside its range, and 1e20 loses no bias above 1e-17
    HAPMI_REQUIRE(scale >= 1e-20f && scale <= 1e20f, HAPMI_ELIMIT, "%s: scale = %g must lie in [1e-20, 1e20]", name, (double)scale);
    HAPMI_REQUIRE(p >= 0.f && p < 1.f, HAPMI_EINVAL, "%s: p = %g must lie in [0, 1)", name, (double)p);
    return HAPMI_OK;
}

// Whether the blocks that fit the 256 CUs at once hold the whole launch: two on each, or one where the bias window and the waves' sums
// fill the LDS (R from 697 on).  Then a third wave a SIMD has nothing to work on, and the kernels that keep two busy with the next
// block's scores are ahead (dQ, two a CU for three: [2, 2048] x 16 heads, 512 blocks, 69.9 us for 74.7; [1, 4096] x 8 causal, 256
// blocks, 80.6 for 90.9; [8, 512] x 16, 512 blocks, 29.0 for 29.7), beyond it they are behind ([12, 512] x 16 heads, 768 blocks: 46.0
// for 41.8; [2, 4096] causal, 1024 blocks: 147 for 141; with one a CU, R = 729, whole backward of 512 blocks [2, 2048] x 16: 179 for
// 154, [1, 4096] x 16 causal: 192 for 190).  The plain kernels themselves drop from three blocks a CU to two above R = 352
// (encoder shape, whole backward: 78 -> 87 us).
// Of a padded batch two thirds of the blocks are taken to be there ([6, 1001] x 12 heads of 334 .. 1001 tokens, 576 blocks: 48.6 for
// 50.6): the lengths are not known here, and a nearly full batch of 513 .. 768 blocks gets the form that is a tenth slower for it.
bool ahead_holds(int64_t blocks, bool padded, int W) {
    const int64_t lds = 3 * 2 * TILE_BYTES + 2 * REL_MAX_SIDE * 2 * 4 + (int64_t)dq_lds_words(W) * 4;      // of one block
    return (padded ? blocks * 2 / 3 : blocks) <= (lds <= 160 * 1024 / 2 ? 2 : 1) * 256;
}

bool aligned(const void *p, uintptr_t n) { return (uintptr_t)p % n == 0; }

// a strided float32 [n][ld] matrix of H columns; a row stride beyond any memory counts as 2^40
HapmiSpan rows_span(const float *p, int64_t n, int64_t ld, int64_t H) {
    if (ld > 1ll << 40) ld = 1ll << 40;
    return {p, ((n - 1) * ld + H) * 4, H * 4, ld > H ? ld * 4 : 0};
}
int64_t keep_bytes(int64_t b, int64_t S, int64_t H) { return b * H * S * 2 * hapmi_cdiv(S, TILE) * 4; }

// More than 64 KiB of LDS a block has to be asked for, once per kernel and device (`asked`: a bit for every device); each time would
// cost the host as much as the checks of all operands.  Asking again is harmless: two threads may.
template <typename F> int allow_lds(const char *name, F kernel, size_t most, std::atomic<uint64_t> &asked) {
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (e == hipSuccess && (asked.load(std::memory_order_relaxed) & bit)) return HAPMI_OK;
    if (e == hipSuccess) e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)most);
    HAPMI_REQUIRE(e == hipSuccess, HAPMI_ELAUNCH, "%s: %s", name, hipGetErrorString(e));
    asked.fetch_or(bit, std::memory_order_relaxed);
    return HAPMI_OK;
}

}  // namespace

extern "C" int hapmi_attention_relbias_fwd(const void *qkv, const hapmi_relbias *bias_host, int causal, const int32_t *lengths, void *out,
                                           float *lse, int64_t b, int64_t S, int64_t H, float scale, const uint32_t *keep_rows,
                                           float p, hapmi_stream_t stream) {
    const char *name = "attention_relbias_fwd";
    RelArgs a;
    int rc = check_shape(name, b, S, H, scale, p);
    if (!rc) rc = check_rel(name, bias_host, S, H, &a);
    if (rc) return rc;
    if (b == 0) return HAPMI_OK;
    HAPMI_REQUIRE(qkv && out && lse && a.table, HAPMI_EINVAL, "%s: null pointer", name);
    HAPMI_REQUIRE(aligned(qkv, 16) && aligned(out, 16) && aligned(keep_rows, 8) && aligned(lse, 4) && aligned(a.table, 4) && aligned(lengths, 4),
                  HAPMI_EALIGN, "%s: qkv and out must be 16-byte aligned (keep words: 8)", name);
    const int64_t n = b * S * H;
    rc = hapmi_apart(name, {{out, n * 128}, {lse, n * 4}},
                     {{qkv, n * 384}, rows_span(a.table, bias_host->n_buckets, a.ld, H), {lengths, b * 4}, {keep_rows, keep_bytes(b, S, H)}});
    if (rc) return rc;
    const float ks = keep_rows ? 1.0f / (1.0f - p) : 1.0f;
    const size_t lds = (size_t)window_of(a.R) * 4;
    dim3 grid((unsigned)hapmi_cdiv(S, 128), (unsigned)(b * H)), block(AT_THREADS);
    auto go = [&](auto kernel) -> int {
        hipLaunchKernelGGL(kernel, grid, block, lds, (hipStream_t)stream, a, (const bf16_t *)qkv, (bf16_t *)out, lse, lengths, (int)S,
                           (int)H, scale, keep_rows, ks);
        HAPMI_CHECK_LAUNCH(name);
        return HAPMI_OK;
    };
    if (causal) return keep_rows ? go(relbias_fwd_kernel<true, true>) : go(relbias_fwd_kernel<true, false>);
    return keep_rows ? go(relbias_fwd_kernel<false, true>) : go(relbias_fwd_kernel<false, false>);
}

extern "C" int hapmi_attention_relbias_workspace_elems(const hapmi_relbias *bias_host, int64_t b, int64_t S, int64_t H, int64_t *elems_host) {
    const char *name = "attention_relbias_workspace_elems";
    RelArgs a;
    int rc = check_shape(name, b, S, H, 1.f, 0.f);
    if (!rc) rc = check_rel(name, bias_host, S, H, &a);
    if (rc) return rc;
    HAPMI_REQUIRE(elems_host, HAPMI_EINVAL, "%s: null pointer", name);
    *elems_host = b * H * hapmi_cdiv(S, 128) * bias_host->n_buckets;
    return HAPMI_OK;
}

extern "C" int hapmi_attention_relbias_bwd(const void *qkv, const hapmi_relbias *bias_host, int causal, const int32_t *lengths,
                                           const void *out, const void *dout, const float *lse, void *dqkv, float *dtable,
                                           int64_t ld_dtable, int accumulate, float *delta_ws, float *workspace,
                                           int64_t workspace_elems, int64_t b, int64_t S, int64_t H, float scale,
                                           const uint32_t *keep_rows, const uint32_t *keep_cols, float p, hapmi_stream_t stream) {
    const char *name = "attention_relbias_bwd";
    RelArgs a;
    int rc = check_shape(name, b, S, H, scale, p);
    if (!rc) rc = check_rel(name, bias_host, S, H, &a);
    if (rc) return rc;
    HAPMI_REQUIRE(b >= 1, HAPMI_EINVAL, "%s: empty batch (the table's gradient would stay unwritten)", name);
    HAPMI_REQUIRE(qkv && out && dout && lse && dqkv && dtable && delta_ws && workspace && a.table, HAPMI_EINVAL, "%s: null pointer", name);
    HAPMI_REQUIRE(aligned(qkv, 16) && aligned(out, 16) && aligned(dout, 16) && aligned(dqkv, 16) && aligned(keep_rows, 8) && aligned(keep_cols, 8) &&
                      aligned(lse, 4) && aligned(a.table, 4) && aligned(dtable, 4) && aligned(delta_ws, 4) && aligned(workspace, 4) &&
                      aligned(lengths, 4),
                  HAPMI_EALIGN, "%s: bf16 tensors must be 16-byte aligned (keep words: 8)", name);
    HAPMI_REQUIRE((keep_rows != nullptr) == (keep_cols != nullptr), HAPMI_EINVAL, "%s: keep_rows and keep_cols come together", name);
    HAPMI_REQUIRE(ld_dtable >= H, HAPMI_EINVAL, "%s: gradient rows of %lld for %lld heads", name, (long long)ld_dtable, (long long)H);
    const int W = window_of(a.R);
    const int64_t row_blocks = hapmi_cdiv(S, 128);
    const int64_t need = b * H * row_blocks * bias_host->n_buckets;
    HAPMI_REQUIRE(workspace_elems >= need, HAPMI_ELIMIT, "%s: workspace of %lld floats, %lld needed", name, (long long)workspace_elems, (long long)need);
    const int64_t n = b * S * H;
    rc = hapmi_apart(name, {{dqkv, n * 384}, rows_span(dtable, bias_host->n_buckets, ld_dtable, H), {delta_ws, n * 4}, {workspace, need * 4}},
                     {{qkv, n * 384}, rows_span(a.table, bias_host->n_buckets, a.ld, H), {out, n * 128}, {dout, n * 128}, {lse, n * 4}, {lengths, b * 4},
                      {keep_rows, keep_bytes(b, S, H)}, {keep_cols, keep_bytes(b, S, H)}});
    if (rc) return rc;
    const bool drop = keep_rows != nullptr;
    const float ks = drop ? 1.0f / (1.0f - p) : 1.0f;
    hipStream_t st = (hipStream_t)stream;
    dim3 grid((unsigned)row_blocks, (unsigned)(b * H)), block(AT_THREADS);
    static std::atomic<uint64_t> asked[6];                    // one for each of dQ's kernels
    auto dq = [&](auto kernel, int which) -> int {
        const size_t lds = (size_t)dq_lds_words(W) * 4;
        rc = allow_lds(name, kernel, (size_t)dq_lds_words(window_of(REL_MAX_REACH)) * 4, asked[which]);
        if (rc) return rc;
        hipLaunchKernelGGL(kernel, grid, block, lds, st, a, (const bf16_t *)qkv, (const bf16_t *)out, (const bf16_t *)dout, lse, delta_ws,
                           (bf16_t *)dqkv, workspace, lengths, (int)S, (int)H, scale, keep_rows, ks);
        HAPMI_CHECK_LAUNCH(name);
        return HAPMI_OK;
    };
    auto dkv = [&](auto kernel) -> int {
        hipLaunchKernelGGL(kernel, grid, block, (size_t)(W > AT_THREADS ? W : AT_THREADS) * 4, st, a, (const bf16_t *)qkv, (const bf16_t *)dout, lse,
                           (const float *)delta_ws, (bf16_t *)dqkv, lengths, (int)S, (int)H, scale, keep_cols, ks, (const float *)workspace, dtable,
                           ld_dtable, bias_host->n_buckets, (int)b, accumulate);
        HAPMI_CHECK_LAUNCH(name);
        return HAPMI_OK;
    };
    if (drop) rc = causal ? dq(relbias_bwd_dq_kernel<true, true, false>, 0) : dq(relbias_bwd_dq_kernel<false, true, false>, 1);
    else if (ahead_holds(row_blocks * b * H, lengths != nullptr, W)) rc = causal ? dq(relbias_bwd_dq_kernel<true, false, true>, 2) : dq(relbias_bwd_dq_kernel<false, false, true>, 3);
    else rc = causal ? dq(relbias_bwd_dq_kernel<true, false, false>, 4) : dq(relbias_bwd_dq_kernel<false, false, false>, 5);
    if (rc) return rc;
    if (causal) return drop ? dkv(relbias_bwd_dkv_kernel<true, true>) : dkv(relbias_bwd_dkv_kernel<true, false>);
    return drop ? dkv(relbias_bwd_dkv_kernel<false, true>) : dkv(relbias_bwd_dkv_kernel<false, false>);
}
