// Pieces shared by the fused attention kernels (head_dim 64, bf16): LDS tile layout and fragment readers, tile loaders,
// the order in which thread blocks take their work.
#pragma once
#include "common.h"
#include "tile.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;


constexpr int HD = 64;                 // head dimension (bf16: one 128-byte LDS row)
constexpr int TILE = 64;               // rows of the streamed operand per iteration
constexpr int AT_THREADS = 256;        // 4 waves, 32 rows of the stationary operand each
constexpr int TILE_BYTES = TILE * ROW_BYTES;

typedef Vec16<bf16_t> frag_t;

__device__ __forceinline__ int aswz(int row) { return (((row >> 1) & 1) << 2) | ((row >> 2) & 3); }

// standard operand fragment of k-step s: k = 16 s + 8 h .. + 8 of `row`
__device__ __forceinline__ frag_t frag_rowk(const char *tile, int row, int s, int h) {
    return *(const frag_t *)(tile + row * ROW_BYTES + ((((s << 1) | h) ^ aswz(row)) << 4));
}

// Fragment of the transposed tile in accumulator order: MFMA row = tile column col0 + lane % 32, slots j < 4 ->
// k = tile row 16 s + 4 h + j, slots j >= 4 -> tile row 16 s + 8 + 4 h + (j - 4).  Within a group of 16 lanes
// ds_read_b64_tr_b16 hands lane j the elements D[4 e + j / 4][j % 4], e = 0..3, of the 16 x 4 matrix whose row
// i is the 8 bytes at lane i's address: lane i points at tile row (first row + i / 4), columns 4 (i % 4) ...
struct TransposedReader {
    int base, cx;              // lane constants: byte offset of (row 4 h + i / 4, within-chunk part), swizzled chunk
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    __device__ __forceinline__ TransposedReader() {
        const int lane = threadIdx.x & 63, i = lane & 15, half = (lane >> 4) & 1, h = lane >> 5, q = i >> 2;
        const int col = 16 * half + 4 * (i & 3);                  // + col0 (0 or 32: chunk + 0 or 4)
        base = (4 * h + q) * ROW_BYTES + (col & 7) * 2;
        cx = (col >> 3) ^ ((((q >> 1) & 1) << 2) | h);            // aswz(16 s + 4 h + q) = ((q >> 1) & 1) << 2 | h
    }
    __device__ __forceinline__ frag_t frag(const char *tile, int col0, int s) const {
        union { v4s h[2]; bf16x8 v; } u;
        // second read: rows + 8, whose swizzle differs by 2 (aswz low bits = (row >> 2) & 3)
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(tile + base + 16 * s * ROW_BYTES + ((cx ^ (col0 >> 3)) << 4)));
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(tile + base + (16 * s + 8) * ROW_BYTES + ((cx ^ (col0 >> 3) ^ 2) << 4)));
        frag_t f;
        f.v = u.v;
        return f;
    }
};
// 8 rows (one k-step) of an accumulator tile as a B operand
__device__ __forceinline__ frag_t acc_to_b(const f32x16 &a, int sp) {
    frag_t f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f.v[j] = (bf16_t)a[sp * 8 + j];
    return f;
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = 0.f;
    return z;
}
__device__ __forceinline__ f32x16 mma(const frag_t &a, const frag_t &b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
// row index inside a 32-row accumulator tile held in register r by a lane of half h
__device__ __forceinline__ int acc_row(int r, int h) { return ((r >> 2) << 3) + (h << 2) + (r & 3); }

__device__ __forceinline__ frag_t load_row_frag(const bf16_t *row_ptr, bool valid, int s, int h) {
    frag_t f;
    if (valid) f = *(const frag_t *)(row_ptr + 16 * s + 8 * h);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f.v[j] = (bf16_t)0.f;
    }
    return f;
}

// One [64 rows][64 d] operand tile (memory [row][d], row stride ld) held as two 16-byte vectors per thread
// (rows 2 * (t / 8) and + 1, d chunk t % 8) on its way into the row-major LDS tile.  The thread's element offsets
// inside a tile and its LDS byte offsets are fixed for the kernel's lifetime; `base` (the tile's first element) is
// the same for every thread, so a load is one instruction on a scalar base and a constant vector offset, and
// full tiles skip the row checks.
struct PairLoader {
    frag_t v[2];
    int goff[2], soff[2];
    __device__ __forceinline__ PairLoader(int ld) {
        const int c8 = threadIdx.x & 7, r0 = (threadIdx.x >> 3) * 2;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            goff[i] = (r0 + i) * ld + c8 * 8;
            soff[i] = (r0 + i) * ROW_BYTES + ((c8 ^ aswz(r0 + i)) << 4);
        }
    }
    __device__ __forceinline__ void load(const bf16_t *base, int rows_left) {
        if (rows_left >= TILE) {
#pragma unroll
            for (int i = 0; i < 2; ++i) v[i] = *(const frag_t *)(base + goff[i]);
        } else {
            const int r0 = (threadIdx.x >> 3) * 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) v[i] = load_row_frag(base + goff[i], r0 + i < rows_left, 0, 0);
        }
    }
    __device__ __forceinline__ void store_rows(char *lds) const {
#pragma unroll
        for (int i = 0; i < 2; ++i) *(frag_t *)(lds + soff[i]) = v[i];
    }
};

// One [64 rows][64 d] operand tile global -> LDS without a stop in registers (global_load_lds_dwordx4: every wave
// instruction fills 1024 contiguous LDS bytes = 8 tile rows, lane l landing in row l / 8, 16-byte slot l % 8).  The
// tile's swizzle is applied on the global side: the lane fetches the chunk that belongs in its slot.  Rows beyond the
// operand's end repeat its last row (finite values; the callers give such keys a probability of zero), since a
// transfer cannot be zero-filled.  The transfers are asynchronous: the caller counts them with s_waitcnt vmcnt (a
// wave's loads complete in issue order) and publishes the tile with a barrier.
struct DirectTileLoader {
    static constexpr int LOADS = 2;                            // wave instructions per tile (64 rows / 4 waves / 8 rows)
    int row[LOADS], chunk[LOADS], ld;
    __device__ __forceinline__ DirectTileLoader(int ld_) : ld(ld_) {
        const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            row[i] = (i * 4 + wave) * 8 + (lane >> 3);
            chunk[i] = ((lane & 7) ^ aswz(row[i])) * 8;
        }
    }
    __device__ __forceinline__ void issue(const bf16_t *base, int rows_left, char *lds_tile) const {
        typedef __attribute__((address_space(3))) char lds_char;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = row[i] < rows_left ? row[i] : rows_left - 1;
            const bf16_t *src = base + r * ld + chunk[i];
            const uint32_t lds_addr = (uint32_t)(uintptr_t)(lds_char *)(lds_tile + (i * 4 + wave) * 1024);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                         :
                         : "s"(lds_addr), "v"(src)
                         : "memory");
        }
    }
};

// One 4-byte word per thread global -> LDS (global_load_lds_dword: a wave instruction fills 256 contiguous LDS bytes,
// lane l landing in word l), into the thread's own slot lds_words[threadIdx.x]; asynchronous like the tile transfers.
__device__ __forceinline__ void issue_word(const uint32_t *src, uint32_t *lds_words) {
    typedef __attribute__((address_space(3))) uint32_t lds_u32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t lds_addr = (uint32_t)(uintptr_t)(lds_u32 *)(lds_words + wave * 64);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds_addr), "v"(src) : "memory");
}

// Which 128-row block and which (batch, head) a thread block works on.  Without a mask every block does the same
// work and the grid is taken as it is.  With the causal mask the work grows with the query block (falls with
// the key block): the blocks are renumbered so that the hardware, which starts blocks in the order of their
// linear index, starts the longest ones first and the short ones fill the tail.
template <bool CAUSAL> struct BlockOrder {
    __device__ __forceinline__ static int linear() { return (int)(blockIdx.y * gridDim.x + blockIdx.x); }
    // Without a mask: blocks are dealt round-robin over the 8 XCDs (each with an L2 of its own) in the order of
    // their linear index.  The row blocks of one (batch, head) stream the same K / V (Q / dO) tiles, so they are
    // given to the same XCD, next to each other in time: work item w = (XCD) * (items per XCD) + (turn on that XCD),
    // row block = w % row blocks.  The tiles then come from that XCD's L2 for all but the first of the blocks.
    __device__ __forceinline__ static int work_item() {
        const int n = (int)(gridDim.x * gridDim.y), l = linear();
        return (n % 8 == 0) ? (l % 8) * (n / 8) + l / 8 : l;
    }
    __device__ __forceinline__ static int row_block(bool work_grows_with_index) {
        if (!CAUSAL) return work_item() % (int)gridDim.x;
        const int i = linear() / (int)gridDim.y;
        return work_grows_with_index ? (int)gridDim.x - 1 - i : i;
    }
    __device__ __forceinline__ static int batch_head() { return CAUSAL ? linear() % (int)gridDim.y : work_item() / (int)gridDim.x; }
};

}  // namespace
