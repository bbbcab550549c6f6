// Balance loss of a router with its per-expert counts, and its gradient, on the records of the top-2 / switch gates.
//
//   n_b = number of real tokens of row b, G = number of rows with n_b > 0, k = choices counted per token (1 or 2)
//   c_be = how many of the row's choices name expert e,  P_be = sum of the row's probabilities of e
//   loss = coef E / G * sum_b 1 / (k n_b^2) * sum_e c_be P_be         (1 * coef for a perfectly even routing)
//   dlogits_bse = p_bse (w_be - sum_e' p_bse' w_be'),  w_be = coef E c_be / (G k n_b^2)       (c is a count: no gradient)
//
// The gate's own gradient (softmax backward of the kept choices' gate gradients) has the same form, so one pass over the
// probabilities serves both.  Memory bound at large sizes and launch bound at small ones: forward is one pass and one
// small joining launch, backward one launch.  64 padded rows of 2048 tokens, 64 experts: counts 8 us, joining 5 us, backward
// 15 us (with the gate's gradient: the probabilities and records of all tokens, 37 MB, read and 34 MB written: 4.7 TB/s); 16 rows of 512 tokens, 16 experts: 4, 2.6 and 4.2 us, most of
// which a launch takes that does nothing.
#include "common.h"

namespace {

constexpr int BAL_THREADS = 256;
constexpr int BAL_MAX_E = 64;
constexpr int BAL_SMALL_WAVES = 16;                // waves of the block that does a small call alone
constexpr int BAL_BLOCKS = 512;                     // a row is cut into slabs until about this many blocks run

__device__ __forceinline__ int bal_length(const int32_t *lengths, int b, int S) {
    if (!lengths) return S;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > S ? S : n);
}

// number of rows with tokens, by the whole block (BAL_THREADS or more threads, `red` 16 floats of LDS)
__device__ __forceinline__ float bal_rows(const int32_t *lengths, int B, int S, float *red) {
    if (!lengths) return (float)B;
    float v = 0.f;
    for (int i = threadIdx.x; i < B; i += blockDim.x) v += bal_length(lengths, i, S) > 0 ? 1.f : 0.f;
    return block_sum(v, red);                       // whole numbers below 2^24: exact in any order
}

// one slab of one row: counts, kept counts and probability sums of every expert
template <int V>
__global__ __launch_bounds__(BAL_THREADS) void balance_count_kernel(const float *probs, const int32_t *index, const int32_t *slot,
                                                                  const int32_t *lengths, int32_t *counts, int32_t *kept, float *psum,
                                                                  int S, int E, int choices, int slab) {
    __shared__ int32_t cnt[2][BAL_MAX_E];
    __shared__ float red[BAL_THREADS * V];
    const int b = blockIdx.y, n = bal_length(lengths, b, S);
    const int s0 = blockIdx.x * slab, s1 = s0 + slab < n ? s0 + slab : n;
    for (int i = threadIdx.x; i < 2 * BAL_MAX_E; i += BAL_THREADS) cnt[i / BAL_MAX_E][i % BAL_MAX_E] = 0;
    __syncthreads();
    for (int s = s0 + (int)threadIdx.x; s < s1; s += BAL_THREADS) {
        const int64_t rec = ((int64_t)b * S + s) * 2;
        for (int k = 0; k < choices; ++k) {
            const int e = index[rec + k];
            if (e >= 0 && e < E) {                  // whole numbers: the order of these additions does not show
                atomicAdd(&cnt[0][e], 1);
                if (slot[rec + k] > 0) atomicAdd(&cnt[1][e], 1);
            }
        }
    }
    const int cols = E / V, per = BAL_THREADS / cols, c = threadIdx.x % cols, r = threadIdx.x / cols;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
    if (r < per) {
        const float *p = probs + (int64_t)b * S * E + c * V;
#pragma unroll 4
        for (int s = s0 + r; s < s1; s += per) {
            if (V == 4) {
                const f32x4 x = *(const f32x4 *)(p + (int64_t)s * E);
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] += x[i];
            } else {
                acc[0] += p[(int64_t)s * E];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) red[threadIdx.x * V + i] = acc[i];
    __syncthreads();
    if ((int)threadIdx.x < E) {
        float v = 0.f;
        for (int i = 0; i < per; ++i) v += red[i * E + threadIdx.x];
        const int64_t at = ((int64_t)b * gridDim.x + blockIdx.x) * E + threadIdx.x;
        counts[at] = cnt[0][threadIdx.x];
        kept[at] = cnt[1][threadIdx.x];
        psum[at] = v;
    }
}

// joins the slabs of every row (slabs == 1: counts, kept, psum are the first kernel's own outputs) and adds up the loss; a
// thread takes V experts of a row, the loads of eight slabs under way at once.  One compute unit's read rate bounds it (64 rows
// x 8 slabs of 64 experts: 6.2 us by one block), so the kept counts, which the loss does not need, are a second block's: 5.0 us
template <int V>
__global__ __launch_bounds__(1024) void balance_join_kernel(const int32_t *lengths, const int32_t *pcounts, const int32_t *pkept,
                                                          const float *ppsum, int32_t *counts, int32_t *kept, float *psum, float *loss,
                                                          int B, int S, int E, int slabs, float coef, int choices) {
    typedef int32_t iv __attribute__((ext_vector_type(V)));
    typedef float fv __attribute__((ext_vector_type(V)));
    __shared__ float red[2][16];
    float v = 0.f;
    if (blockIdx.x == 1) {                          // (launched with slabs > 1 only)
        for (int64_t i = (int64_t)threadIdx.x * V; i < (int64_t)B * E; i += 1024 * V) {
            const int b = (int)(i / E), e = (int)(i - (int64_t)b * E);
            const int64_t at = (int64_t)b * slabs * E + e;
            iv k = 0;
#pragma unroll 8
            for (int z = 0; z < slabs; ++z) k += *(const iv *)(pkept + at + z * E);
            *(iv *)(kept + i) = k;
        }
        return;
    }
    // the lengths are on their way while the slabs are loaded, and both sums meet at one barrier
    const int first = lengths && (int)threadIdx.x < B ? lengths[threadIdx.x] : 0;
    for (int64_t i = (int64_t)threadIdx.x * V; i < (int64_t)B * E; i += 1024 * V) {
        const int b = (int)(i / E), e = (int)(i - (int64_t)b * E);
        const int64_t at = (int64_t)b * slabs * E + e;
        const int n_b = lengths ? lengths[b] : S;
        iv c = 0;
        fv p = 0.f;
#pragma unroll 8
        for (int z = 0; z < slabs; ++z) {
            c += *(const iv *)(pcounts + at + z * E);
            p += *(const fv *)(ppsum + at + z * E);
        }
        if (slabs > 1) {
            *(iv *)(counts + i) = c;
            *(fv *)(psum + i) = p;
        }
        const float n = (float)(n_b < 0 ? 0 : (n_b > S ? S : n_b));
        if (n > 0.f) {
#pragma unroll
            for (int j = 0; j < V; ++j) v += (float)c[j] / n * (p[j] / n);
        }
    }
    float rows = first > 0 ? 1.f : 0.f;             // rows with tokens: whole numbers below 2^24, exact in any order
    if (lengths)
        for (int i = 1024 + (int)threadIdx.x; i < B; i += 1024) rows += lengths[i] > 0 ? 1.f : 0.f;
    v = wave_sum(v);
    rows = wave_sum(rows);
    if ((threadIdx.x & 63) == 0) {
        red[0][threadIdx.x >> 6] = v;
        red[1][threadIdx.x >> 6] = rows;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float t = 0.f, G = 0.f;
        for (int i = 0; i < 16; ++i) {
            t += red[0][i];
            G += red[1][i];
        }
        if (!lengths) G = (float)B;
        loss[0] = G > 0.f ? coef * (float)E / (G * (float)choices) * t : 0.f;
    }
}

// A small call in one launch: a block, whose waves take a row each in turn.  Lanes hold V experts of 64 V / E tokens at a time.
template <int V>
__global__ __launch_bounds__(BAL_SMALL_WAVES * 64) void balance_small_kernel(const float *probs, const int32_t *index, const int32_t *slot,
                                                                          const int32_t *lengths, int32_t *counts, int32_t *kept, float *psum,
                                                                          float *loss, int B, int S, int E, float coef, int choices) {
    __shared__ int32_t cnt[BAL_SMALL_WAVES][2][BAL_MAX_E];
    __shared__ float part[BAL_SMALL_WAVES][64 * V];
    __shared__ float red[2][BAL_SMALL_WAVES];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int cols = E / V, per = 64 / cols, c = lane % cols, r = lane / cols;
    float v = 0.f, rows = 0.f;
    for (int b = wave; b < B; b += BAL_SMALL_WAVES) {
        const int n = bal_length(lengths, b, S);
        cnt[wave][0][lane] = 0;                     // (a wave's LDS accesses are carried out in their order)
        cnt[wave][1][lane] = 0;
        asm volatile("" ::: "memory");
        for (int s0 = lane; s0 < n; s0 += 4 * 64) {
            int e[4][2], sl[4][2];                  // the records of four tokens are on their way at once
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int s = s0 + j * 64;
                const int64_t rec = ((int64_t)b * S + (s < n ? s : s0)) * 2;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const bool counts_here = s < n && k < choices;
                    e[j][k] = counts_here ? index[rec + k] : -1;
                    sl[j][k] = counts_here ? slot[rec + k] : 0;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (e[j][k] >= 0 && e[j][k] < E) {        // whole numbers: the order of these additions does not show
                        atomicAdd(&cnt[wave][0][e[j][k]], 1);
                        if (sl[j][k] > 0) atomicAdd(&cnt[wave][1][e[j][k]], 1);
                    }
        }
        float acc[V];
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
        if (r < per) {
            const float *p = probs + (int64_t)b * S * E + c * V;
#pragma unroll 8
            for (int s = r; s < n; s += per) {
                if (V == 4) {
                    const f32x4 x = *(const f32x4 *)(p + (int64_t)s * E);
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[i] += x[i];
                } else {
                    acc[0] += p[(int64_t)s * E];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) part[wave][lane * V + i] = acc[i];
        asm volatile("" ::: "memory");
        if (lane < E) {
            float sum = 0.f;
            for (int i = 0; i < per; ++i) sum += part[wave][i * E + lane];
            const int named = cnt[wave][0][lane];
            const int64_t at = (int64_t)b * E + lane;
            counts[at] = named;
            kept[at] = cnt[wave][1][lane];
            psum[at] = sum;
            if (n > 0) v += (float)named / (float)n * (sum / (float)n);
        }
        asm volatile("" ::: "memory");
        rows += n > 0 ? 1.f : 0.f;
    }
    v = wave_sum(v);
    if (lane == 0) {
        red[0][wave] = v;
        red[1][wave] = rows;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float t = 0.f, G = 0.f;
        for (int i = 0; i < BAL_SMALL_WAVES; ++i) {
            t += red[0][i];
            G += red[1][i];
        }
        loss[0] = G > 0.f ? coef * (float)E / (G * (float)choices) * t : 0.f;
    }
}

// a group of lanes per token, V experts a lane; BAL_TURNS tokens of a lane are loaded before the first one is worked on.  A token
// that does not count and that no gate gradient reaches gets zeros whatever its probabilities hold (0 * NaN would pass its padding
// on to the router's weights); without the gate's gradient they are not read.
constexpr int BAL_TURNS = 4;
template <int V>
__global__ __launch_bounds__(BAL_THREADS) void balance_bwd_kernel(const float *probs, const int32_t *index, const int32_t *slot,
                                                                const float *dgate, const int32_t *counts, const int32_t *lengths,
                                                                float *dlogits, int B, int S, int E, float coef, int choices,
                                                                int group_log2) {
    __shared__ float red[16];
    typedef int32_t i32x2 __attribute__((ext_vector_type(2)));
    const int b = blockIdx.y, n = bal_length(lengths, b, S);
    const int j = threadIdx.x & ((1 << group_log2) - 1), e0 = j * V, per = BAL_THREADS >> group_log2;
    const int s0 = blockIdx.x * per * BAL_TURNS + (int)(threadIdx.x >> group_log2);
    float p[BAL_TURNS][V], dg[BAL_TURNS][2];
    int at[BAL_TURNS][2];
#pragma unroll
    for (int t = 0; t < BAL_TURNS; ++t) {
        const int s = s0 + t * per;
        const int64_t tok = (int64_t)b * S + s;
#pragma unroll
        for (int i = 0; i < V; ++i) p[t][i] = 0.f;
        at[t][0] = at[t][1] = -1;
        dg[t][0] = dg[t][1] = 0.f;
        if (s >= (dgate ? S : n)) continue;
        if (V == 4) {
            if (e0 < E) {
                const f32x4 x = *(const f32x4 *)(probs + tok * E + e0);
#pragma unroll
                for (int i = 0; i < V; ++i) p[t][i] = x[i];
            }
        } else if (e0 < E) {
            p[t][0] = probs[tok * E + e0];
        }
        if (dgate) {
            const i32x2 ix = *(const i32x2 *)(index + tok * 2), sl = *(const i32x2 *)(slot + tok * 2);
            const f32x2 g = *(const f32x2 *)(dgate + tok * 2);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                at[t][k] = ix[k];
                dg[t][k] = sl[k] > 0 ? g[k] : 0.f;
            }
        }
    }
    const float G = bal_rows(lengths, B, S, red);
    float w[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
        w[i] = n > 0 && e0 + i < E ? coef * (float)E / (G * (float)choices) * ((float)counts[(int64_t)b * E + e0 + i] / (float)n / (float)n) : 0.f;
#pragma unroll
    for (int t = 0; t < BAL_TURNS; ++t) {
        const int s = s0 + t * per;
        const int64_t tok = (int64_t)b * S + s;
        float g[V], dot = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            g[i] = s < n ? w[i] : 0.f;
#pragma unroll
            for (int k = 0; k < 2; ++k) g[i] += at[t][k] == e0 + i ? dg[t][k] : 0.f;
            dot += p[t][i] * g[i];
        }
        dot = group_sum(dot, group_log2);
        if (s >= S || e0 >= E) continue;
        const bool none = s >= n && dg[t][0] == 0.f && dg[t][1] == 0.f;
        if (V == 4) {
            f32x4 x;
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = none ? 0.f : p[t][i] * (g[i] - dot);
            *(f32x4 *)(dlogits + tok * E + e0) = x;
        } else {
            dlogits[tok * E + e0] = none ? 0.f : p[t][0] * (g[0] - dot);
        }
    }
}

int bal_check(const char *name, int64_t B, int64_t S, int64_t E, int choices) {
    HAPMI_REQUIRE(B >= 0 && S >= 1 && E >= 1 && (choices == 1 || choices == 2), HAPMI_EINVAL, "%s: bad argument", name);
    HAPMI_REQUIRE(E <= BAL_MAX_E && B <= 65535 && S < (1ll << 24), HAPMI_ELIMIT, "%s: at most %d experts, 65535 rows and 2^24 - 1 tokens a row", name, BAL_MAX_E);
    return HAPMI_OK;
}

// Whether one block does it all: up to 256 KiB of probabilities (a compute unit reads about 100 GB/s), and few steps for a wave (a
// load of 64 V / E tokens; 64 tokens' records and their LDS additions count 16).  One launch against two, in a graph / called from the
// host: 4 rows of 64 tokens, 16 experts 3.9 against 5.8 / 8.0 against 10.9 us; 11 of 90, 33 experts 6.6 against 5.9 / 7.8 against
// 10.5; beyond the limits 16 of 128, 64 experts 7.9 against 6.2 / 8.0 against 11.4; 2 of 1024, 8 experts 10.8 against 7.3 / 10.8
// against 11.8; 16 of 512, 16 experts 13.1 against 6.3 / 13.1 against 11.5.
bool bal_small(int64_t B, int64_t S, int64_t E) {
    const int64_t per = 64 / (E % 4 == 0 ? E / 4 : E), loads = hapmi_cdiv(S, per), records = 16 * hapmi_cdiv(S, 64);
    return B * S * E <= 65536 && hapmi_cdiv(B, BAL_SMALL_WAVES) * (loads > records ? loads : records) <= 96;
}

// tokens a block takes: about 16 KiB of probabilities at least, whole rows once there are BAL_BLOCKS of them
int64_t bal_slab(int64_t B, int64_t S, int64_t E) {
    const int64_t least = hapmi_cdiv(4096, E);
    int64_t slabs = hapmi_cdiv(BAL_BLOCKS, B);
    if (slabs > hapmi_cdiv(S, least)) slabs = hapmi_cdiv(S, least);
    return hapmi_cdiv(S, slabs);
}

}  // namespace

extern "C" int hapmi_balance_workspace_elems(int64_t B, int64_t S, int64_t E, int64_t *elems_host) {
    const int rc = bal_check("balance_workspace_elems", B, S, E, 1);
    if (rc) return rc;
    HAPMI_REQUIRE(elems_host, HAPMI_EINVAL, "balance_workspace_elems: null pointer");
    const int64_t slabs = B && !bal_small(B, S, E) ? hapmi_cdiv(S, bal_slab(B, S, E)) : 1;
    *elems_host = slabs > 1 ? 3 * B * slabs * E : 0;
    return HAPMI_OK;
}

extern "C" int hapmi_balance_loss_fwd(const float *probs, const int32_t *index, const int32_t *slot, const int32_t *lengths, float *loss,
                                      int32_t *counts, int32_t *kept, float *prob_sum, int64_t B, int64_t S, int64_t E, float coef, int choices,
                                      float *workspace, int64_t workspace_elems, hapmi_stream_t stream) {
    const char *name = "balance_loss_fwd";
    const int rc = bal_check(name, B, S, E, choices);
    if (rc) return rc;
    HAPMI_REQUIRE(B >= 1, HAPMI_EINVAL, "%s: empty batch (the loss would stay unwritten)", name);
    HAPMI_REQUIRE(probs && index && slot && loss && counts && kept && prob_sum, HAPMI_EINVAL, "%s: null pointer", name);
    HAPMI_REQUIRE((uintptr_t)probs % 16 == 0, HAPMI_EALIGN, "%s: probs must be 16-byte aligned", name);
    const bool small = bal_small(B, S, E);
    const int64_t slab = small ? S : bal_slab(B, S, E), slabs = hapmi_cdiv(S, slab), n = B * slabs * E;
    HAPMI_REQUIRE(slabs == 1 || (workspace && workspace_elems >= 3 * n), HAPMI_ELIMIT, "%s: workspace of %lld floats, %lld needed", name,
                  (long long)(workspace ? workspace_elems : 0), (long long)(3 * n));
    const int64_t records = B * S * 2 * 4, sums = B * E * 4;
    const int rc2 = hapmi_apart(name, {{loss, 4}, {counts, sums}, {kept, sums}, {prob_sum, sums}, {slabs > 1 ? workspace : nullptr, 3 * n * 4}},
                                {{probs, B * S * E * 4}, {index, records}, {slot, records}, {lengths, B * 4}});
    if (rc2) return rc2;
    if (small) {
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(1), dim3(BAL_SMALL_WAVES * 64), 0, (hipStream_t)stream, probs, index, slot, lengths, counts, kept, prob_sum, loss,
                               (int)B, (int)S, (int)E, coef, choices);
        };
        if (E % 4 == 0) go(balance_small_kernel<4>);
        else go(balance_small_kernel<1>);
        HAPMI_CHECK_LAUNCH(name);
        return HAPMI_OK;
    }
    int32_t *pc = slabs > 1 ? (int32_t *)workspace : counts, *pk = slabs > 1 ? (int32_t *)workspace + n : kept;
    float *pp = slabs > 1 ? workspace + 2 * n : prob_sum;
    const dim3 grid((unsigned)slabs, (unsigned)B), block(BAL_THREADS);
    hipStream_t st = (hipStream_t)stream;
    if (E % 4 == 0) hipLaunchKernelGGL((balance_count_kernel<4>), grid, block, 0, st, probs, index, slot, lengths, pc, pk, pp, (int)S, (int)E, choices, (int)slab);
    else hipLaunchKernelGGL((balance_count_kernel<1>), grid, block, 0, st, probs, index, slot, lengths, pc, pk, pp, (int)S, (int)E, choices, (int)slab);
    HAPMI_CHECK_LAUNCH(name);
    const bool vec = E % 4 == 0 && ((uintptr_t)pc % 16 == 0 && (uintptr_t)pk % 16 == 0 && (uintptr_t)pp % 16 == 0 && (uintptr_t)counts % 16 == 0 &&
                                    (uintptr_t)kept % 16 == 0 && (uintptr_t)prob_sum % 16 == 0);
    auto join = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(slabs > 1 ? 2 : 1), dim3(1024), 0, st, lengths, (const int32_t *)pc, (const int32_t *)pk, (const float *)pp, counts, kept, prob_sum, loss,
                           (int)B, (int)S, (int)E, (int)slabs, coef, choices);
    };
    if (vec) join(balance_join_kernel<4>);
    else join(balance_join_kernel<1>);
    HAPMI_CHECK_LAUNCH(name);
    return HAPMI_OK;
}

extern "C" int hapmi_balance_loss_bwd(const float *probs, const int32_t *index, const int32_t *slot, const float *dgate, const int32_t *counts,
                                      const int32_t *lengths, float *dlogits, int64_t B, int64_t S, int64_t E, float coef, int choices,
                                      hapmi_stream_t stream) {
    const char *name = "balance_loss_bwd";
    const int rc = bal_check(name, B, S, E, choices);
    if (rc) return rc;
    if (B == 0) return HAPMI_OK;
    HAPMI_REQUIRE(probs && counts && dlogits && (!dgate || (index && slot)), HAPMI_EINVAL, "%s: null pointer", name);
    HAPMI_REQUIRE((uintptr_t)probs % 16 == 0 && (uintptr_t)dlogits % 16 == 0, HAPMI_EALIGN, "%s: probs and dlogits must be 16-byte aligned", name);
    const int V = E % 4 == 0 ? 4 : 1;
    int group_log2 = 0;
    while ((V << group_log2) < E) ++group_log2;
    HAPMI_REQUIRE(!dgate || ((uintptr_t)index % 8 == 0 && (uintptr_t)slot % 8 == 0 && (uintptr_t)dgate % 8 == 0), HAPMI_EALIGN,
                  "%s: index, slot and dgate must be 8-byte aligned", name);
    const int64_t records = B * S * 2 * 4;
    const int rc2 = hapmi_apart(name, {{dlogits, B * S * E * 4}},
                                {{probs, B * S * E * 4}, {index, records}, {slot, records}, {dgate, records}, {counts, B * E * 4}, {lengths, B * 4}});
    if (rc2) return rc2;
    const dim3 grid((unsigned)hapmi_cdiv(S, (BAL_THREADS >> group_log2) * BAL_TURNS), (unsigned)B), block(BAL_THREADS);
    if (V == 4) hipLaunchKernelGGL((balance_bwd_kernel<4>), grid, block, 0, (hipStream_t)stream, probs, index, slot, dgate, counts, lengths, dlogits, (int)B, (int)S, (int)E, coef, choices, group_log2);
    else hipLaunchKernelGGL((balance_bwd_kernel<1>), grid, block, 0, (hipStream_t)stream, probs, index, slot, dgate, counts, lengths, dlogits, (int)B, (int)S, (int)E, coef, choices, group_log2);
    HAPMI_CHECK_LAUNCH(name);
    return HAPMI_OK;
}
