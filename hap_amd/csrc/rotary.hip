// Norm of queries and keys per head and rotation by position, in one pass over the packed projection
// qkv[b, S, 3*H*D], forward and backward.
//
//   r = 1 / sqrt(mean_d x^2 + eps),  u = x r,  n = g u,  y = R(position) n
//   R turns the first `rot` dimensions of a head in pairs: (i, i + rot / 2), or neighbours (2 i, 2 i + 1):
//   (y0, y1) = (n0 cos - n1 sin, n0 sin + n1 cos); the angles' cosines and sines come from a table of positions.
//   dn = R^T dy,  dg = sum over tokens and heads of dn u,  dx = r (g dn - u mean_d(g dn u))
//
// Memory bound: forward reads and writes a row once, backward reads x and dy and writes dx.  A group of 1 .. 32 lanes
// holds one head of a token, every lane two 16-byte vectors chosen so that both halves of every rotated pair are its
// own: the rotation needs no exchange, the mean one butterfly over the group.  The lane takes the query and the key of
// its (token, head) together and reads the angles once for both.  bf16, 16 heads of 64: forward of [12, 512] 16.4 us, 75 MB at
// 4.6 TB/s; backward of [4, 8192] with both gains 113 us, 547 MB at 4.8 TB/s.  A copy of that size with one vector a thread and
// non-temporal accesses reaches 6.6 TB/s (a library copy 5.2), which the looping grid and cached accesses here do not.
#include "common.h"

namespace {

constexpr int QN_THREADS = 256;
constexpr int QN_MAX_DIM = 256;
// backward with gains: rows of up to this many blocks are one block's, which needs no second launch.  Two, 8 tokens of 16 heads of 64:
// 11.6 for 14.4 us from the host, 9.5 for 8.6 in a graph; four: 17.9 for 14.4 and 17.8 for 8.6
constexpr int QN_TURNS = 2;
constexpr int QN_MAX_BLOCKS = 768;                  // backward: blocks whose gain sums a second kernel adds; 3 a CU are resident

struct QnArgs {
    const float *q_gain, *k_gain;                   // [D] or NULL (ones)
    const float *angles;                            // [n_pos][rot / 2][cos, sin] or NULL
    const int32_t *positions;                       // [tokens] or NULL (position inside the sequence)
    int64_t rows;                                   // tokens * H
    int64_t n_pos;
    int S, H, D, rot, interleaved, group_log2;
    float eps;
};

// the lane's two vectors of a head (vector indices, b < 0: none) and where their angles lie in a table row
struct QnLane {
    int a, b;
    bool turn_a, turn_b;
};
template <typename T> __device__ __forceinline__ QnLane qn_lane(const QnArgs &p, int j) {
    constexpr int V = Vec16<T>::N;
    const int nv = p.D / V, rv = p.rot / V;
    QnLane l;
    if (!p.interleaved && j < rv / 2) {
        l.a = j; l.b = j + rv / 2;
        l.turn_a = l.turn_b = true;
    } else {
        l.a = p.interleaved ? 2 * j : rv + 2 * (j - rv / 2);
        l.b = l.a + 1;
        l.turn_a = p.interleaved && l.a < rv;
        l.turn_b = p.interleaved && l.b < rv;
    }
    if (l.a >= nv) l.a = -1;
    if (l.b >= nv) l.b = -1;
    return l;
}

template <int V> struct QnAngles { float c[V], s[V]; };

// angles of the lane's rotated pairs: half-split: V pairs (a[e], b[e]); neighbours: V / 2 pairs of a, then V / 2 of b
template <int V> __device__ __forceinline__ QnAngles<V> qn_angles(const QnArgs &p, const QnLane &l, const float *row) {
    QnAngles<V> w;
    if (!p.interleaved) {
        f32x4 t[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) t[i] = *(const f32x4 *)(row + l.a * V * 2 + i * 4);
#pragma unroll
        for (int e = 0; e < V; ++e) { w.c[e] = t[e / 2][(e & 1) * 2]; w.s[e] = t[e / 2][(e & 1) * 2 + 1]; }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) { w.c[e] = 1.f; w.s[e] = 0.f; }
        f32x4 t[V / 4];
        if (l.turn_a) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) t[i] = *(const f32x4 *)(row + l.a * V + i * 4);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) { w.c[e] = t[e / 2][(e & 1) * 2]; w.s[e] = t[e / 2][(e & 1) * 2 + 1]; }
        }
        if (l.turn_b) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) t[i] = *(const f32x4 *)(row + l.b * V + i * 4);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) { w.c[V / 2 + e] = t[e / 2][(e & 1) * 2]; w.s[V / 2 + e] = t[e / 2][(e & 1) * 2 + 1]; }
        }
    }
    return w;
}

// turns the lane's values (sign = -1: back)
template <int V>
__device__ __forceinline__ void qn_turn(const QnArgs &p, const QnLane &l, const QnAngles<V> &w, float sign, float (&a)[V], float (&b)[V]) {
    if (!p.interleaved) {
        if (l.turn_a) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float s = w.s[e] * sign, x0 = a[e], x1 = b[e];
                a[e] = x0 * w.c[e] - x1 * s;
                b[e] = x0 * s + x1 * w.c[e];
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            const float sa = w.s[e] * sign, sb = w.s[V / 2 + e] * sign;
            const float a0 = a[2 * e], a1 = a[2 * e + 1], b0 = b[2 * e], b1 = b[2 * e + 1];
            a[2 * e] = a0 * w.c[e] - a1 * sa;
            a[2 * e + 1] = a0 * sa + a1 * w.c[e];
            b[2 * e] = b0 * w.c[V / 2 + e] - b1 * sb;
            b[2 * e + 1] = b0 * sb + b1 * w.c[V / 2 + e];
        }
    }
}

template <typename T> struct QnPair {
    static constexpr int V = Vec16<T>::N;
    Vec16<T> a, b;
    __device__ __forceinline__ void load(const T *row, const QnLane &l) {
        if (l.a >= 0) a = *(const Vec16<T> *)(row + l.a * V);
        else {
#pragma unroll
            for (int e = 0; e < V; ++e) a.set(e, 0.f);
        }
        if (l.b >= 0) b = *(const Vec16<T> *)(row + l.b * V);
        else {
#pragma unroll
            for (int e = 0; e < V; ++e) b.set(e, 0.f);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            a.set(e, 0.f);
            b.set(e, 0.f);
        }
    }
    __device__ __forceinline__ void store(T *row, const QnLane &l) const {
        if (l.a >= 0) *(Vec16<T> *)(row + l.a * V) = a;
        if (l.b >= 0) *(Vec16<T> *)(row + l.b * V) = b;
    }
};

template <int V> __device__ __forceinline__ void qn_gain(const float *g, const QnLane &l, float (&ga)[V], float (&gb)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        ga[e] = g && l.a >= 0 ? g[l.a * V + e] : 1.f;
        gb[e] = g && l.b >= 0 ? g[l.b * V + e] : 1.f;
    }
}

// A position outside the table poisons the token's queries and keys in forward instead of reading beyond it, and leaves the
// token out of backward: no gradient for its queries and keys, nothing in the gains' (as an id outside an embedding table does).
__device__ __forceinline__ int64_t qn_position(const QnArgs &p, int64_t token, int S, bool &bad) {
    const int64_t pos = p.positions ? p.positions[token] : token % S;
    bad = pos < 0 || pos >= p.n_pos;
    return bad ? 0 : pos;
}

template <typename T>
__global__ __launch_bounds__(QN_THREADS) void qk_norm_rotary_fwd_kernel(const QnArgs p, const T *qkv, T *out) {
    constexpr int V = Vec16<T>::N;
    const int group = 1 << p.group_log2, j = threadIdx.x & (group - 1);
    const QnLane l = qn_lane<T>(p, j);
    const int E = p.H * p.D;
    float gq[2][V], gk[2][V];
    qn_gain<V>(p.q_gain, l, gq[0], gq[1]);
    qn_gain<V>(p.k_gain, l, gk[0], gk[1]);
    const int64_t step = (int64_t)gridDim.x * (QN_THREADS >> p.group_log2);
    // a wave's groups stay together: rows are tested per group, the butterfly below runs over whole groups only
    for (int64_t row = (int64_t)blockIdx.x * (QN_THREADS >> p.group_log2) + (threadIdx.x >> p.group_log2); row < p.rows; row += step) {
        const int64_t token = row / p.H, at = token * 3 * E + (row - token * p.H) * p.D;
        QnPair<T> x[2];
        x[0].load(qkv + at, l);
        x[1].load(qkv + at + E, l);
        if (out != qkv) {
            QnPair<T> v;
            v.load(qkv + at + 2 * E, l);
            v.store(out + at + 2 * E, l);
        }
        bool bad = false;
        QnAngles<V> w;
        if (p.rot) {
            const int64_t pos = qn_position(p, token, p.S, bad);
            if (l.turn_a || l.turn_b) w = qn_angles<V>(p, l, p.angles + pos * p.rot);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float a[V], b[V], sq = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                a[e] = x[t].a.get(e);
                b[e] = x[t].b.get(e);
                sq += a[e] * a[e] + b[e] * b[e];
            }
            sq = group_sum(sq, p.group_log2);
            const float r = bad ? NAN : 1.0f / sqrtf(sq / p.D + p.eps);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                a[e] *= r * (t ? gk : gq)[0][e];
                b[e] *= r * (t ? gk : gq)[1][e];
            }
            if (l.turn_a || l.turn_b) qn_turn<V>(p, l, w, 1.f, a, b);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[t].a.set(e, a[e]);
                x[t].b.set(e, b[e]);
            }
            x[t].store(out + at + t * E, l);
        }
    }
}

template <typename T, bool GAINS>
__global__ __launch_bounds__(QN_THREADS, 3) void qk_norm_rotary_bwd_kernel(const QnArgs p, const T *dout, const T *qkv, T *dqkv, float *part,
                                                                          float *dq_gain, float *dk_gain, int accumulate) {
    constexpr int V = Vec16<T>::N;
    __shared__ __attribute__((aligned(16))) float red[GAINS ? QN_THREADS * 4 * V : 1];      // 2 D sums a group, and D <= 2 V a lane
    __shared__ __attribute__((aligned(16))) float gains[2][QN_MAX_DIM];     // read again for every row: 32 registers less a lane
    for (int i = threadIdx.x; i < p.D; i += QN_THREADS) {
        gains[0][i] = p.q_gain ? p.q_gain[i] : 1.f;
        gains[1][i] = p.k_gain ? p.k_gain[i] : 1.f;
    }
    __syncthreads();
    const int group = 1 << p.group_log2;
    const int E = p.H * p.D;
    float acc[2][2][V];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[t][0][e] = acc[t][1][e] = 0.f;
    const int64_t step = (int64_t)gridDim.x * (QN_THREADS >> p.group_log2);
    for (int64_t row = (int64_t)blockIdx.x * (QN_THREADS >> p.group_log2) + (threadIdx.x >> p.group_log2); row < p.rows; row += step) {
        int heads = p.H, S = p.S, tid = threadIdx.x;          // (reciprocals, the lane's part and its addresses are made for every
        asm volatile("" : "+s"(heads), "+s"(S), "+v"(tid));   // row: kept over the loop they cost spills)
        const QnLane m = qn_lane<T>(p, tid & (group - 1));
        const int64_t token = row / heads, at = token * 3 * E + (row - token * heads) * p.D;
        QnPair<T> x[2], d[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            x[t].load(qkv + at + t * E, m);
            d[t].load(dout + at + t * E, m);
        }
        if (dqkv != dout) {
            QnPair<T> v;
            v.load(dout + at + 2 * E, m);
            v.store(dqkv + at + 2 * E, m);
        }
        bool bad = false;
        QnAngles<V> w;
        if (p.rot) {
            const int64_t pos = qn_position(p, token, S, bad);
            if (m.turn_a || m.turn_b) w = qn_angles<V>(p, m, p.angles + pos * p.rot);
        }
        if (__builtin_expect(bad, 0)) {                       // (its rows may hold anything: zeros in their place, and r = 0 below)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                x[t].clear();
                d[t].clear();
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float a[V], b[V], da[V], db[V], sq = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                a[e] = x[t].a.get(e);
                b[e] = x[t].b.get(e);
                da[e] = d[t].a.get(e);
                db[e] = d[t].b.get(e);
                sq += a[e] * a[e] + b[e] * b[e];
            }
            sq = group_sum(sq, p.group_log2);
            const float r = bad ? 0.f : 1.0f / sqrtf(sq / p.D + p.eps);
            if (m.turn_a || m.turn_b) qn_turn<V>(p, m, w, -1.f, da, db);
            asm volatile("" ::: "memory");                    // (the gains are not to be hoisted into registers)
            const int ga = (m.a < 0 ? 0 : m.a) * V, gb = (m.b < 0 ? 0 : m.b) * V;
            float dot = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                a[e] *= r;
                b[e] *= r;
                if (GAINS) {
                    acc[t][0][e] += da[e] * a[e];
                    acc[t][1][e] += db[e] * b[e];
                }
                da[e] *= gains[t][ga + e];
                db[e] *= gains[t][gb + e];
                dot += da[e] * a[e] + db[e] * b[e];
            }
            dot = group_sum(dot, p.group_log2) / p.D;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                x[t].a.set(e, r * (da[e] - a[e] * dot));
                x[t].b.set(e, r * (db[e] - b[e] * dot));
            }
            x[t].store(dqkv + at + t * E, m);
        }
    }
    if (!GAINS) return;
    // gain sums over the block's groups, in their order: a row of 2 D sums for each of them (exchanges between lanes, 1 .. 6 for each of
    // the lane's 32 values, took 6 us of a block's time: 14.9 us for 8.6 at 32 tokens of 16 heads of 64, 117 for 113 at [4, 8192])
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const QnLane l = qn_lane<T>(p, tid & (group - 1));
    float *own = red + (tid >> p.group_log2) * 2 * p.D;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int vec = k ? l.b : l.a;
            if (vec < 0) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) own[t * p.D + vec * V + e] = acc[t][k][e];
        }
    __syncthreads();
    const int groups = QN_THREADS >> p.group_log2;
    for (int i = threadIdx.x; i < 2 * p.D; i += QN_THREADS) {
        float v = 0.f;
#pragma unroll 8
        for (int r = 0; r < groups; ++r) v += red[r * 2 * p.D + i];
        if (gridDim.x > 1) part[(int64_t)blockIdx.x * 2 * p.D + i] = v;
        else if (float *g = i < p.D ? dq_gain : dk_gain) {              // nothing to join
            g += i < p.D ? i : i - p.D;
            *g = accumulate ? *g + v : v;
        }
    }
}

// gradient of both gains: the blocks' sums part[blocks][2 D], 32 columns a block, 32 runs of block indices a column
__global__ __launch_bounds__(1024) void qk_gain_sum_kernel(const float *part, int blocks, int D, float *dq_gain, float *dk_gain, int accumulate) {
    __shared__ float red[32][33];
    const int c = threadIdx.x & 31, run = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
    float v = 0.f;
    if (col < 2 * D) {
        const int per = (blocks + 31) / 32, end = (run + 1) * per < blocks ? (run + 1) * per : blocks;
#pragma unroll 8
        for (int i = run * per; i < end; ++i) v += part[(int64_t)i * 2 * D + col];
    }
    red[run][c] = v;
    __syncthreads();
    if (run == 0 && col < 2 * D) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += red[i][c];
        float *g = col < D ? dq_gain : dk_gain;
        if (g) {
            g += col < D ? col : col - D;
            *g = accumulate ? *g + s : s;
        }
    }
}

int qn_check(const char *name, int64_t b, int64_t S, int64_t H, int64_t D, const float *angles, int64_t n_pos, int64_t rot, int interleaved,
             float eps, int dtype, const int32_t *positions, const float *q_gain, const float *k_gain, QnArgs *a) {
    HAPMI_REQUIRE(hapmi_dtype_ok(dtype) && b >= 0 && S >= 1 && H >= 1 && D >= 1 && eps >= 0.f, HAPMI_EINVAL, "%s: bad argument", name);
    const int V = dtype == HAPMI_F32 ? 4 : 8;
    HAPMI_REQUIRE(D <= QN_MAX_DIM && H <= 65536 && S < (1ll << 31) && b < (1ll << 31), HAPMI_ELIMIT, "%s: head_dim at most %d, heads at most 65536", name,
                  QN_MAX_DIM);
    HAPMI_REQUIRE(D % V == 0, HAPMI_EALIGN, "%s: head_dim %lld must be a multiple of %d", name, (long long)D, V);
    HAPMI_REQUIRE((angles != nullptr) == (rot > 0), HAPMI_EINVAL, "%s: the angle table and rot > 0 come together", name);
    HAPMI_REQUIRE(rot >= 0 && rot <= D && rot % (interleaved ? V : 2 * V) == 0, HAPMI_EALIGN, "%s: rot = %lld must be a multiple of %d, at most head_dim", name,
                  (long long)rot, interleaved ? V : 2 * V);
    HAPMI_REQUIRE(!angles || n_pos >= 1, HAPMI_EINVAL, "%s: empty angle table", name);
    HAPMI_REQUIRE(!angles || positions || n_pos >= S, HAPMI_EINVAL, "%s: %lld positions in the table, sequences of %lld", name, (long long)n_pos, (long long)S);
    HAPMI_REQUIRE(b <= (1ll << 40) / (S * H), HAPMI_ELIMIT, "%s: b * S * H above 2^40", name);
    HAPMI_REQUIRE((uintptr_t)angles % 16 == 0 && (uintptr_t)positions % 4 == 0 && (uintptr_t)q_gain % 4 == 0 && (uintptr_t)k_gain % 4 == 0, HAPMI_EALIGN,
                  "%s: the angle table must be 16-byte aligned", name);
    a->q_gain = q_gain; a->k_gain = k_gain; a->angles = angles; a->positions = positions;
    a->rows = b * S * H; a->n_pos = n_pos;
    a->S = (int)S; a->H = (int)H; a->D = (int)D; a->rot = (int)rot; a->interleaved = interleaved ? 1 : 0;
    a->eps = eps;
    const int pairs = (int)((D / V + 1) / 2);
    a->group_log2 = 0;
    while ((1 << a->group_log2) < pairs) ++a->group_log2;
    return HAPMI_OK;
}

int64_t qn_blocks(const QnArgs &a, int64_t most) {
    const int64_t n = hapmi_cdiv(a.rows, QN_THREADS >> a.group_log2);
    return n < most ? n : most;
}

}  // namespace

extern "C" int hapmi_qk_norm_rotary_fwd(const void *qkv, void *out, const float *q_gain, const float *k_gain, const float *angles, int64_t n_pos,
                                        int64_t rot, int interleaved, const int32_t *positions, int64_t b, int64_t S, int64_t H, int64_t D, float eps,
                                        int dtype, hapmi_stream_t stream) {
    const char *name = "qk_norm_rotary_fwd";
    QnArgs a;
    const int rc = qn_check(name, b, S, H, D, angles, n_pos, rot, interleaved, eps, dtype, positions, q_gain, k_gain, &a);
    if (rc) return rc;
    if (b == 0) return HAPMI_OK;
    HAPMI_REQUIRE(qkv && out, HAPMI_EINVAL, "%s: null pointer", name);
    HAPMI_REQUIRE((uintptr_t)qkv % 16 == 0 && (uintptr_t)out % 16 == 0, HAPMI_EALIGN, "%s: qkv and out must be 16-byte aligned", name);
    const int64_t size = dtype == HAPMI_F32 ? 4 : 2, n = a.rows * 3 * D * size;
    const int rc2 = hapmi_apart(name, {{out, n}}, {{out == qkv ? nullptr : qkv, n}, {q_gain, D * 4}, {k_gain, D * 4}, {angles, n_pos * rot * 4},
                                                   {positions, b * S * 4}});
    if (rc2) return rc2;
    const dim3 grid((unsigned)qn_blocks(a, 1 << 20)), block(QN_THREADS);
    if (dtype == HAPMI_F32) hipLaunchKernelGGL((qk_norm_rotary_fwd_kernel<float>), grid, block, 0, (hipStream_t)stream, a, (const float *)qkv, (float *)out);
    else hipLaunchKernelGGL((qk_norm_rotary_fwd_kernel<bf16_t>), grid, block, 0, (hipStream_t)stream, a, (const bf16_t *)qkv, (bf16_t *)out);
    HAPMI_CHECK_LAUNCH(name);
    return HAPMI_OK;
}

extern "C" int hapmi_qk_norm_rotary_workspace_elems(int64_t D, int64_t *elems_host) {
    HAPMI_REQUIRE(elems_host && D >= 1 && D <= QN_MAX_DIM, HAPMI_EINVAL, "qk_norm_rotary_workspace_elems: bad argument");
    *elems_host = 2 * D * QN_MAX_BLOCKS;
    return HAPMI_OK;
}

extern "C" int hapmi_qk_norm_rotary_bwd(const void *dout, const void *qkv, void *dqkv, const float *q_gain, const float *k_gain, float *dq_gain,
                                        float *dk_gain, int accumulate, const float *angles, int64_t n_pos, int64_t rot, int interleaved,
                                        const int32_t *positions, int64_t b, int64_t S, int64_t H, int64_t D, float eps, int dtype, float *workspace,
                                        int64_t workspace_elems, hapmi_stream_t stream) {
    const char *name = "qk_norm_rotary_bwd";
    QnArgs a;
    const int rc = qn_check(name, b, S, H, D, angles, n_pos, rot, interleaved, eps, dtype, positions, q_gain, k_gain, &a);
    if (rc) return rc;
    HAPMI_REQUIRE(b >= 1, HAPMI_EINVAL, "%s: empty batch (the gains' gradients would stay unwritten)", name);
    HAPMI_REQUIRE(dout && qkv && dqkv, HAPMI_EINVAL, "%s: null pointer", name);
    HAPMI_REQUIRE((uintptr_t)dout % 16 == 0 && (uintptr_t)qkv % 16 == 0 && (uintptr_t)dqkv % 16 == 0 && (uintptr_t)dq_gain % 4 == 0 &&
                      (uintptr_t)dk_gain % 4 == 0 && (uintptr_t)workspace % 4 == 0,
                  HAPMI_EALIGN, "%s: dout, qkv and dqkv must be 16-byte aligned", name);
    const bool gains = dq_gain || dk_gain;
    HAPMI_REQUIRE(!gains || (workspace && workspace_elems >= 2 * D * QN_MAX_BLOCKS), HAPMI_ELIMIT, "%s: workspace of %lld floats, %lld needed", name,
                  (long long)(workspace ? workspace_elems : 0), (long long)(2 * D * QN_MAX_BLOCKS));
    const int64_t size = dtype == HAPMI_F32 ? 4 : 2, n = a.rows * 3 * D * size;
    int rc2 = hapmi_apart(name, {{dqkv, n}, {dq_gain, D * 4}, {dk_gain, D * 4}, {gains ? workspace : nullptr, 2 * D * QN_MAX_BLOCKS * 4}},
                          {{dout == dqkv ? nullptr : dout, n}, {qkv, n}, {q_gain, D * 4}, {k_gain, D * 4}, {angles, n_pos * rot * 4}, {positions, b * S * 4}});
    if (rc2) return rc2;
    const int64_t blocks = gains && qn_blocks(a, 1 << 20) <= QN_TURNS ? 1 : qn_blocks(a, gains ? QN_MAX_BLOCKS : 1 << 20);
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto kernel, auto zero) -> int {
        typedef decltype(zero) T;
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(QN_THREADS), 0, st, a, (const T *)dout, (const T *)qkv, (T *)dqkv, workspace, dq_gain, dk_gain, accumulate);
        HAPMI_CHECK_LAUNCH(name);
        return HAPMI_OK;
    };
    if (dtype == HAPMI_F32) rc2 = gains ? go(qk_norm_rotary_bwd_kernel<float, true>, 0.f) : go(qk_norm_rotary_bwd_kernel<float, false>, 0.f);
    else rc2 = gains ? go(qk_norm_rotary_bwd_kernel<bf16_t, true>, (bf16_t)0.f) : go(qk_norm_rotary_bwd_kernel<bf16_t, false>, (bf16_t)0.f);
    if (rc2 || !gains || blocks == 1) return rc2;
    hipLaunchKernelGGL(qk_gain_sum_kernel, dim3((unsigned)hapmi_cdiv(2 * D, 32)), dim3(1024), 0, st, (const float *)workspace, (int)blocks, (int)D, dq_gain,
                       dk_gain, accumulate);
    HAPMI_CHECK_LAUNCH(name);
    return HAPMI_OK;
}
