// Norms before and after a residual block, fused with the block's gate and residual scale, and the backward pass
// (include/sr_hip.h: sr_op_residual_norm, sr_op_residual_norm_bwd).  Row r holds the C channels of one position:
//
//   hat(v) = (v - m) / sqrt(mean((v - m)^2) + eps)      m = mean(v) for SR_NORM_LAYER, 0 for SR_NORM_RMS
//   p = post_gain hat(y) + post_bias                    (without SR_NORM_POST: p = y)
//   h = x + scale a p                                   a = gate, sigmoid(gate) or 1
//   n = pre_gain hat(h) + pre_bias                      (with SR_NORM_PRE; from the unrounded h)
//
//   T = dh + rs_h (g - mean(g) - hat(h) mean(g hat(h))),  g = dn pre_gain        (mean(g) for SR_NORM_LAYER only)
//   dx = T,  dgate = sum over the gate row's positions of scale a' p T,  dp = scale a T
//   dy = rs_y (q - mean(q) - hat(y) mean(q hat(y))),  q = dp post_gain
//   dpost_gain = sum dp hat(y), dpost_bias = sum dp, dpre_gain = sum dn hat(h), dpre_bias = sum dn
//
// Bound by HBM: the forward pass moves 4 tensors for ~16 operations an element, the backward pass 6 for ~40.  So a row is read
// once: a group of lanes (a "team") holds it in registers across all sums of the row, and the backward pass takes the row
// statistics again from what it holds instead of reading them.  Rows of up to 512 channels belong to 1..64 lanes of a wave, several
// rows to a wave, and their sums are lane exchanges; longer rows belong to a workgroup, which joins its waves' sums in LDS.  A lane
// holds 8 elements of a row (4 in the backward pass of 513 to 4096 channels where 8 need more registers than there are; above that it is
// 8 with what it spills, see bwd_plan) and has the same places of the team's next row on their way.  All sums and the values between them are fp32; tensors of 16 bits are rounded
// once, when they are stored.
#include "op_host.h"
#include "row_math.h"

#include <algorithm>

using namespace sr;
using namespace srh;

namespace {

constexpr int MAX_C = 8192;          // 1024 lanes x 8 channels
constexpr int WAVE_C = 512;          // up to here a row belongs to lanes of one wave

// no gate, a gate row for every position, for several, for a few (backward pass of rows within a wave)
enum Gate { G_NONE = 0, G_ROW = 1, G_SHARED = 2, G_GROUP = 3 };

// Work split of a backward pass: `per_group` workgroups share the `span` rows of a group (the rows that share a gate row, or all
// rows); that is a unit each.  Their teams take the group's rows in turn, so that what is read at one time lies together.  With
// G_GROUP a unit is a group, and the teams of all workgroups take the groups in turn.
struct Units {
    unsigned span, units, per_group;
};

// what a call does, a bit each
enum Flags { F_BRANCH = 1, F_POST = 2, F_PRE = 4, F_LAYER = 8, F_SIGMOID = 16, F_STREAM_GRAD = 32, F_READ_Y = 64 };

struct FwdArgs {
    const void *x, *y, *gate;
    const float *pw, *pb, *qw, *qb;  // post gain / bias, pre gain / bias
    void *h, *n;
    int ldx, ldy, ldg, ldh, ldn;
    unsigned rows, span;             // span: rows that share a gate row
    int C, tl, flags;                // tl: log2 of a team's lanes (rows within a wave)
    float scale, eps, inv_c;
};

struct BwdArgs {
    const void *h, *y, *gate, *dh, *dn;
    const float *pw, *pb, *qw;
    void *dx, *dy, *dgate;
    float *sums[4];                  // where the sums for post gain, post bias, pre gain, pre bias go (NULL: not wanted), `step` floats
    int64_t step;                    // from workgroup to workgroup: partial sums, or the gradients themselves where there is one workgroup
    float *gpart;                    // [units][pitch] partial sums of dgate where a gate row spans several units
    int pitch;                       // C rounded up to 4: the sums are read 16 bytes at a time
    int ldh, ldy, ldg, lddh, lddn, lddx, lddy, lddg;
    Units u;
    int C, tl, flags;
    float scale, eps, inv_c;
};

template <typename T>
__device__ __forceinline__ T* row_of(const void* p, unsigned r, int ld) {
    return (T*)p + (int64_t)((uint64_t)r * (unsigned)ld);
}

// What a thread knows about its place in a team.  A lane holds E elements as NV = E / VEC vectors, `lanes` vectors apart.
// TAIL: the row's last vector is not full (`part` elements of it are).
template <int E_, int VEC_, bool BLK_, bool TAIL_>
struct Team {
    static constexpr int E = E_, VEC = VEC_, NV = E / VEC;
    static constexpr bool BLK = BLK_, TAIL = TAIL_;
    int lanes, lane, row, rows;      // lanes of a team, this thread's lane, its team's number in the workgroup, teams in the workgroup
    int tl, C, part;
    float* red;                      // BLK: [2][16][8] floats: two buffers, up to 8 sums of up to 16 waves
    int phase = 0;

    __device__ Team(int tl_, int C_, float* red_) : tl(tl_), C(C_), part(C_ % VEC), red(red_) {
        if (BLK) {
            lanes = blockDim.x, lane = threadIdx.x, row = 0, rows = 1;
        } else {
            lanes = 1 << tl, lane = threadIdx.x & (lanes - 1), row = threadIdx.x >> tl, rows = blockDim.x >> tl;
        }
    }
    __device__ __forceinline__ int col(int j) const { return (j * lanes + lane) * VEC; }
    __device__ __forceinline__ bool full(int j) const { return col(j) + VEC <= C; }
    // does vector j hold the end of a row, and not all of it the row's?
    __device__ __forceinline__ bool ends(int j) const { return TAIL && !full(j) && col(j) < C; }
    // the place of column c in its vector
    __device__ __forceinline__ int place(int c) const {
        int d = c - (C - part);
        if (!TAIL || d < 0) return c % VEC;
        const int n4 = VEC == 8 ? part & 4 : 0;
        if (d < n4) return d;
        d -= n4;
        return d < (part & 2) ? VEC - 4 + d : VEC - 2;
    }

    // sums of K values over the team, in every lane
    template <int K>
    __device__ __forceinline__ void sum(float (&v)[K]) {
        static_assert(K <= 8, "places of a wave in red");
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = lanes_sum(v[k], BLK ? 6 : tl);
        if (BLK) {
            // two buffers in turn: a wave that writes the next sums cannot reach a buffer that others still read, because it
            // has to pass the barrier in between
            float* b = red + phase * 128;
            phase ^= 1;
            const int wave = threadIdx.x >> 6, nw = (blockDim.x + 63) >> 6, l = threadIdx.x & 15;
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int k = 0; k < K; ++k) b[wave * 8 + k] = v[k];
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = lanes_sum(l < nw ? b[l * 8 + k] : 0.f, 4);
        }
    }
};

// A lane's elements of a row as they are stored.  Lanes behind the row never load: what they hold stays 0 from here on, so the
// loads of a row are one branch and no selects.  A last vector of `part` < VEC elements is loaded and stored in pieces of 4, 2 and
// 1, which have fixed places in the vector: the order of a row's elements in registers does not matter.
template <typename T, typename TEAM>
struct Raw {
    Vec<T, TEAM::VEC> v[TEAM::NV];
    T one;                           // the piece of 1
    __device__ Raw() {
#pragma unroll
        for (int j = 0; j < TEAM::NV; ++j)
#pragma unroll
            for (int k = 0; k < TEAM::VEC; ++k) v[j].v[k] = (T)0.f;
        one = (T)0.f;
    }
};

template <typename T, typename TEAM>
__device__ __forceinline__ void load_raw(const T* p, int j, const TEAM& t, Raw<T, TEAM>& o) {
    o.v[j] = *reinterpret_cast<const Vec<T, TEAM::VEC>*>(p + t.col(j));
}

template <typename T, typename TEAM>
__device__ __forceinline__ void load_part(const T* p, int j, const TEAM& t, Raw<T, TEAM>& o) {
    constexpr int VEC = TEAM::VEC;
    const T* q = p + t.col(j);
    if (VEC == 8 && (t.part & 4)) {
        const Vec<T, 4> a = *reinterpret_cast<const Vec<T, 4>*>(q);
#pragma unroll
        for (int k = 0; k < 4; ++k) o.v[j].v[k] = a.v[k];
    }
    if (t.part & 2) {
        const Vec<T, 2> a = *reinterpret_cast<const Vec<T, 2>*>(q + (t.part & 4));
        o.v[j].v[VEC - 4] = a.v[0], o.v[j].v[VEC - 3] = a.v[1];
    }
    if (t.part & 1) o.one = q[t.part & 6];
}

template <typename T, typename TEAM>
__device__ __forceinline__ void unpack(const Raw<T, TEAM>& r, const TEAM& t, float (&v)[TEAM::E]) {
    constexpr int VEC = TEAM::VEC;
#pragma unroll
    for (int j = 0; j < TEAM::NV; ++j) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[j * VEC + k] = (float)r.v[j].v[k];
        if (TEAM::TAIL && t.ends(j)) v[j * VEC + VEC - 2] = (float)r.one;
    }
}

// zeros in the places of a last vector that are not the row's
template <typename TEAM>
__device__ __forceinline__ void trim(float (&v)[TEAM::E], const TEAM& t) {
    constexpr int VEC = TEAM::VEC;
    if (!TEAM::TAIL) return;
#pragma unroll
    for (int j = 0; j < TEAM::NV; ++j) {
        if (!t.ends(j)) continue;
        if (VEC == 8 && !(t.part & 4)) v[j * VEC] = v[j * VEC + 1] = v[j * VEC + 2] = v[j * VEC + 3] = 0.f;
        if (!(t.part & 2)) v[j * VEC + VEC - 4] = v[j * VEC + VEC - 3] = 0.f;
        if (!(t.part & 1)) v[j * VEC + VEC - 2] = 0.f;
        v[j * VEC + VEC - 1] = 0.f;
    }
}

template <typename T, typename TEAM>
__device__ __forceinline__ void store_row(T* p, const TEAM& t, const float (&v)[TEAM::E]) {
    constexpr int VEC = TEAM::VEC;
#pragma unroll
    for (int j = 0; j < TEAM::NV; ++j) {
        float o[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = v[j * VEC + k];
        T* q = p + t.col(j);
        if (t.full(j)) {
            store_vec<T, VEC>(q, o);
        } else if (TEAM::TAIL && t.col(j) < t.C) {
            if (VEC == 8 && (t.part & 4)) {
                const float w[4] = {o[0], o[1], o[2], o[3]};
                store_vec<T, 4>(q, w);
            }
            if (t.part & 2) {
                const float w[2] = {o[VEC - 4], o[VEC - 3]};
                store_vec<T, 2>(q + (t.part & 4), w);
            }
            if (t.part & 1) q[t.part & 6] = (T)o[VEC - 2];
        }
    }
}

// v -= mean over the row; v is 0 behind it and stays so
template <typename TEAM>
__device__ __forceinline__ void centre(float (&v)[TEAM::E], float mean, const TEAM& t) {
#pragma unroll
    for (int j = 0; j < TEAM::NV; ++j) {
        const float m = t.col(j) < t.C ? mean : 0.f;
#pragma unroll
        for (int k = 0; k < TEAM::VEC; ++k) v[j * TEAM::VEC + k] -= m;
    }
    trim(v, t);
}

template <int E>
__device__ __forceinline__ float sum_e(const float (&v)[E]) {
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int k = 0; k < E; k += 2) s += v[k], u += v[k + 1];
    return s + u;
}
template <int E>
__device__ __forceinline__ float dot_e(const float (&a)[E], const float (&b)[E]) {
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int k = 0; k < E; k += 2) s += a[k] * b[k], u += a[k + 1] * b[k + 1];
    return s + u;
}
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + expf(-g)); }   // rcp: 1 ulp
// its slope s (1 - s), where s = sigmoid(g).  1 - s is exp(-g) s as well, which keeps its precision where s is close to 1 (from g = 17
// on the difference is 0); far below 0 exp(-g) is infinite, but the difference exact to a rounding
__device__ __forceinline__ float sigmoid_slope(float g, float s) { return s * (g > 0.f ? expf(-g) * s : 1.f - s); }

// one row of anything, 0 behind it
template <typename T, typename TEAM>
__device__ __forceinline__ void load_row(const T* p, const TEAM& t, float (&v)[TEAM::E]) {
    Raw<T, TEAM> r;
#pragma unroll
    for (int j = 0; j < TEAM::NV; ++j) {
        if (t.full(j)) load_raw(p, j, t, r);
        else if (t.ends(j)) load_part(p, j, t, r);
    }
    unpack(r, t, v);
}

// a gain or bias, `none` where there is no vector; 0 behind the row, so that what is multiplied by it needs no mask
template <typename TEAM>
__device__ __forceinline__ void load_gain(const float* p, const TEAM& t, float (&v)[TEAM::E], float none) {
    if (p) {
        load_row(p, t, v);
    } else {
#pragma unroll
        for (int j = 0; j < TEAM::NV; ++j)
#pragma unroll
            for (int k = 0; k < TEAM::VEC; ++k) v[j * TEAM::VEC + k] = t.col(j) < t.C ? none : 0.f;
        trim(v, t);
    }
}

// ------------------------------------------------------------------------------------------------- forward
template <typename TEAM>
__device__ __forceinline__ void normalise(float (&v)[TEAM::E], const FwdArgs& a, TEAM& t) {
    if (a.flags & F_LAYER) {
        float m[1] = {sum_e(v)};
        t.sum(m);
        centre(v, m[0] * a.inv_c, t);
    }
    float s[1] = {dot_e(v, v)};
    t.sum(s);
    const float rs = rsqrtf(s[0] * a.inv_c + a.eps);
#pragma unroll
    for (int k = 0; k < TEAM::E; ++k) v[k] *= rs;
}

// The teams of all workgroups take the rows in turn, so that what is read at one time lies together: with a stretch of rows for each
// workgroup instead, the 942,080 x 64 call with an fp32 stream took 195 us instead of 138 (5.2 TB/s; 16384 x 4096 bf16: 98 us, 5.5 TB/s).
template <typename TS, typename TB, int E, int VEC, bool BLK, bool TAIL, int GATE>
__global__ void __launch_bounds__(BLK ? 1024 : 256) rn_fwd_kernel(const FwdArgs a) {
    using TEAM = Team<E, VEC, BLK, TAIL>;
    __shared__ float red[BLK ? 256 : 1];
    TEAM t(a.tl, a.C, red);
    float pw[E], pb[E], qw[E], qb[E];
    Raw<TS, TEAM> x;
    Raw<TB, TEAM> y, g;
    auto fetch = [&](unsigned r) {
        const TS* px = row_of<const TS>(a.x, r, a.ldx);
        const TB *py = row_of<const TB>(a.y, r, a.ldy), *pg = row_of<const TB>(a.gate, r, a.ldg);
#pragma unroll
        for (int j = 0; j < TEAM::NV; ++j) {
            if (t.full(j)) {
                load_raw(px, j, t, x);
                if (a.flags & F_BRANCH) load_raw(py, j, t, y);
                if (GATE == G_ROW) load_raw(pg, j, t, g);
            } else if (t.ends(j)) {
                load_part(px, j, t, x);
                if (a.flags & F_BRANCH) load_part(py, j, t, y);
                if (GATE == G_ROW) load_part(pg, j, t, g);
            }
        }
    };
    unsigned r = blockIdx.x * t.rows + t.row;
    const unsigned step = gridDim.x * t.rows;
    if (r < a.rows) fetch(r);
    load_gain(a.pw, t, pw, 1.f);
    load_gain(a.pb, t, pb, 0.f);
    load_gain(a.qw, t, qw, 1.f);
    load_gain(a.qb, t, qb, 0.f);
    float act[E];                    // scale times the gate that rows share, and the first row behind them
    unsigned end = 0;
    for (; r < a.rows; r += step) {
        float h[E], p[E], gt[E];
        unpack(x, t, h);
        unpack(y, t, p);
        if (GATE == G_ROW) unpack(g, t, gt);
        // the team's next row is on its way while this one is worked on
        if (r + step < a.rows) fetch(r + step);
        if (GATE == G_SHARED && r >= end) {
            const unsigned group = r / a.span;
            end = (group + 1) * a.span;
            load_row(row_of<const TB>(a.gate, group, a.ldg), t, act);
#pragma unroll
            for (int k = 0; k < E; ++k) act[k] = a.scale * (a.flags & F_SIGMOID ? sigmoid(act[k]) : act[k]);
        }
        if (a.flags & F_BRANCH) {
            if (a.flags & F_POST) {
                normalise(p, a, t);
#pragma unroll
                for (int k = 0; k < E; ++k) p[k] = p[k] * pw[k] + pb[k];
            }
            if (GATE == G_ROW) {
#pragma unroll
                for (int k = 0; k < E; ++k) p[k] *= a.flags & F_SIGMOID ? sigmoid(gt[k]) : gt[k];
            }
#pragma unroll
            for (int k = 0; k < E; ++k) h[k] += (GATE == G_SHARED ? act[k] : a.scale) * p[k];
            store_row(row_of<TS>(a.h, r, a.ldh), t, h);
        }
        if (a.flags & F_PRE) {
            normalise(h, a, t);
#pragma unroll
            for (int k = 0; k < E; ++k) h[k] = h[k] * qw[k] + qb[k];
            store_row(row_of<TB>(a.n, r, a.ldn), t, h);
        }
    }
}

// ------------------------------------------------------------------------------------------------- backward
// The sums over rows that a thread keeps for its columns, in LDS: in registers the four of them would cost a wave in four, and
// LDS has the time (two 16-byte reads and writes a sum and row, under a tenth of what the row takes to arrive).
// [wave][sum][half][lane] float4: no bank conflicts, and each thread's are its own until they are joined.  NS: how many sums
template <int E, int NS>
struct Sums {
    static constexpr int Q = E / 4, WAVE = NS * Q * 256;         // floats of a wave
    float4* at;
    __device__ Sums(float* lds) : at(reinterpret_cast<float4*>(lds + (threadIdx.x >> 6) * WAVE) + (threadIdx.x & 63)) {}
    // float k of quarter q of sum i of a lane of the first wave
    static __device__ __forceinline__ int place(int i, int lane, int q, int k) { return ((Q * i + q) * 64 + lane) * 4 + k; }
    __device__ __forceinline__ void zero(int i) const {
#pragma unroll
        for (int q = 0; q < Q; ++q) at[(Q * i + q) * 64] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __device__ __forceinline__ void add(int i, const float (&v)[E]) const {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            float4 a = at[(Q * i + q) * 64];
            a.x += v[4 * q], a.y += v[4 * q + 1], a.z += v[4 * q + 2], a.w += v[4 * q + 3];
            at[(Q * i + q) * 64] = a;
        }
    }
    __device__ __forceinline__ void get(int i, float (&v)[E]) const {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const float4 a = at[(Q * i + q) * 64];
            v[4 * q] = a.x, v[4 * q + 1] = a.y, v[4 * q + 2] = a.z, v[4 * q + 3] = a.w;
        }
    }
    __device__ __forceinline__ void set(int i, const float (&v)[E]) const {
#pragma unroll
        for (int q = 0; q < Q; ++q) at[(Q * i + q) * 64] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    }
};

// Few columns: 1 << splits() threads share one of `n`, each with a part of every wave's teams
template <typename TEAM>
__device__ __forceinline__ int splits(int n, const TEAM& t) {
    int s = 0;
    while (s < 6 - t.tl && n << (s + 1) <= (int)blockDim.x) ++s;
    return s;
}

// Column c of sum i over the teams of a workgroup, by 1 << s threads of which this is number k
template <int NS, typename TEAM>
__device__ __forceinline__ float joined(int i, int c, int k, int s, const TEAM& t, const float* lds) {
    // element e of thread l of every team
    const int j = c / TEAM::VEC, l = j & (t.lanes - 1), e = (j >> t.tl) * TEAM::VEC + t.place(c);
    const float* p = lds + Sums<TEAM::E, NS>::place(i, l + k * t.lanes, e / 4, e % 4);
    const int n = 64 >> (t.tl + s), step = t.lanes * 4 << s;
    float v = 0.f;
    for (int w = 0; w < (int)blockDim.x; w += 256, p += 4 * Sums<TEAM::E, NS>::WAVE) {     // four waves or eight
#pragma unroll 2
        for (int q = 0; q < n; ++q) {
            float o[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) o[h] = p[q * step + h * Sums<TEAM::E, NS>::WAVE];
            v += (o[0] + o[1]) + (o[2] + o[3]);
        }
    }
    return s ? lanes_sum(v, s) : v;
}

// Sum i over the teams of a workgroup to out[0 .. C), on top of what is there with `add`; the same thread has the same column
// every time
template <int NS, typename T, typename TEAM>
__device__ __forceinline__ void leave(int i, const Sums<TEAM::E, NS>& sums, const TEAM& t, const float* lds, T* out, bool add) {
    if constexpr (TEAM::BLK) {
        float v[TEAM::E], o[TEAM::E];
        sums.get(i, v);
        if (add) {
            load_row(out, t, o);
#pragma unroll
            for (int k = 0; k < TEAM::E; ++k) v[k] += o[k];
        }
        store_row(out, t, v);
    } else {
        const int s = splits(t.C, t), k = threadIdx.x & ((1 << s) - 1);
        for (int c = threadIdx.x >> s; c < t.C; c += blockDim.x >> s) {
            const float v = joined<NS>(i, c, k, s, t, lds);
            if (k == 0) out[c] = (T)(add ? (float)out[c] + v : v);
        }
    }
}

// The places in LDS that a backward pass has: its sums over rows; G_GROUP's sum for dgate; the slopes of a sigmoid gate that a unit's
// rows share.  Taken from the gate again at the end of the unit the slopes cost 0.4 us a unit (62,496 x 64 bf16, 16 rows each: 42 us and
// not 40); rows of a workgroup do that all the same, 1024 lanes leave no room for them.
template <int GATE, bool FULL, bool BLK>
constexpr int bwd_sums() { return (FULL ? 4 : GATE == G_SHARED ? 3 : 2) + (GATE == G_GROUP || (GATE == G_SHARED && !BLK)); }

// Rows in turn like the forward pass (8192 x 4096 bf16: 80.5 us, 5.0 TB/s; 163,840 x 64 fp32 with a gate an image: 50 us, 5.0 TB/s).
// FULL: layer norms or gradients of biases; without, only what rms norms with gains need is in registers.  The sums over rows are
// those of a unit; a workgroup with several units adds them up in its partial sums.  With a gate that a unit shares they are
//   A = sum T hat(y) (or T y), B = sum T   (T with the scale):  dpost_gain = a A, dpost_bias = a B, dgate = a' (post_gain A + post_bias B)
template <typename TS, typename TB, int E, int VEC, bool BLK, bool TAIL, int GATE, bool FULL>
__global__ void __launch_bounds__(BLK ? 1024 : 512, BLK ? 4 : 3) rn_bwd_kernel(const BwdArgs a) {
    extern __shared__ float lds[];   // the sums, then BLK's [2][16][8] floats
    constexpr bool ROW = GATE == G_ROW || GATE == G_GROUP;
    constexpr int NS = bwd_sums<GATE, FULL, BLK>();
    enum { S_PW, S_QW, S_PB, S_QB, S_GATE = NS - 1 };
    using TEAM = Team<E, VEC, BLK, TAIL>;
    TEAM t(a.tl, a.C, lds + NS * E * blockDim.x);
    const Sums<E, NS> sums(lds);
    constexpr bool SUM_T = FULL || GATE == G_SHARED;
    float pw[E], qw[E];
    Raw<TS, TEAM> hr, dr;
    Raw<TB, TEAM> yr, nr, gr;
    auto fetch = [&](unsigned r, unsigned gate) {
        const TS *ph = row_of<const TS>(a.h, r, a.ldh), *pd = row_of<const TS>(a.dh, r, a.lddh);
        const TB *py = row_of<const TB>(a.y, r, a.ldy), *pn = row_of<const TB>(a.dn, r, a.lddn), *pg = row_of<const TB>(a.gate, gate, a.ldg);
#pragma unroll
        for (int j = 0; j < TEAM::NV; ++j) {
            if (t.full(j)) {
                if (a.flags & F_PRE) load_raw(ph, j, t, hr), load_raw(pn, j, t, nr);
                if (a.flags & F_READ_Y) load_raw(py, j, t, yr);
                if (a.flags & F_STREAM_GRAD) load_raw(pd, j, t, dr);
                if (ROW) load_raw(pg, j, t, gr);
            } else if (t.ends(j)) {
                if (a.flags & F_PRE) load_part(ph, j, t, hr), load_part(pn, j, t, nr);
                if (a.flags & F_READ_Y) load_part(py, j, t, yr);
                if (a.flags & F_STREAM_GRAD) load_part(pd, j, t, dr);
                if (ROW) load_part(pg, j, t, gr);
            }
        }
    };
    const unsigned last = GATE == G_GROUP ? gridDim.x : a.u.units;
    for (unsigned u = blockIdx.x; u < last; u += gridDim.x) {
        const unsigned group = u / a.u.per_group, step = GATE == G_GROUP ? gridDim.x * t.rows : a.u.per_group * t.rows;
        const unsigned r1 = GATE == G_GROUP ? a.u.units * a.u.span : (group + 1) * a.u.span;
        unsigned gate = u * t.rows + t.row, left = a.u.span;         // G_GROUP: the row's gate row, rows that it has from here on
        const unsigned r0 = GATE == G_GROUP ? gate * a.u.span : group * a.u.span + (u - group * a.u.per_group) * t.rows + t.row;
        if (r0 < r1) fetch(r0, GATE == G_GROUP ? gate : r0);
        if (u == blockIdx.x) {
            load_gain(a.pw, t, pw, 1.f);
            load_gain(a.qw, t, qw, 1.f);
        }
        sums.zero(S_PW), sums.zero(S_QW);
        if (SUM_T) sums.zero(S_PB);
        if (FULL) sums.zero(S_QB);
        if (GATE == G_GROUP) sums.zero(S_GATE);
        float act[E];
        if (GATE == G_SHARED) {
            load_row(row_of<const TB>(a.gate, group, a.ldg), t, act);
            if (!BLK && a.flags & F_SIGMOID) {
                float slope[E];
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const float ac = sigmoid(act[k]);
                    slope[k] = sigmoid_slope(act[k], ac), act[k] = ac;
                }
                sums.set(S_GATE, slope);
            } else {
#pragma unroll
                for (int k = 0; k < E; ++k) act[k] = a.flags & F_SIGMOID ? sigmoid(act[k]) : act[k];
            }
        }
        unsigned next = 0;
        for (unsigned r = r0; r < r1; r = next) {
            float hv[E], yv[E], T[E], g[E], gt[E];
            unpack(hr, t, hv);
            unpack(nr, t, g);
            unpack(yr, t, yv);
            unpack(dr, t, T);
            if (ROW) unpack(gr, t, gt);
            next = GATE != G_GROUP ? r + step : left > 1 ? r + 1 : r + 1 + (step - 1) * a.u.span;
            if (next < r1) fetch(next, GATE == G_GROUP ? gate + (left > 1 ? 0 : step) : next);
            float s[FULL ? 4 : 3];
            if (FULL && (a.flags & F_LAYER)) {
                float m[2] = {sum_e(hv), sum_e(yv)};
                t.sum(m);
                if (a.flags & F_PRE) centre(hv, m[0] * a.inv_c, t);
                if (a.flags & F_POST) centre(yv, m[1] * a.inv_c, t);
            }
            {
                float w[E];
#pragma unroll
                for (int k = 0; k < E; ++k) w[k] = g[k] * qw[k];
                s[0] = dot_e(hv, hv), s[1] = dot_e(w, hv), s[2] = dot_e(yv, yv);
                if (FULL) s[FULL ? 3 : 0] = sum_e(w);
            }
            t.sum(s);
            const float rs_y = a.flags & F_POST ? rsqrtf(s[2] * a.inv_c + a.eps) : 1.f;
            if (a.flags & F_PRE) {
                const float rs = rsqrtf(s[0] * a.inv_c + a.eps);
                const float m2 = s[1] * rs * a.inv_c, m1 = FULL && (a.flags & F_LAYER) ? s[FULL ? 3 : 0] * a.inv_c : 0.f;
                if (FULL) sums.add(S_QB, g);
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    const float hat = hv[k] * rs;
                    T[k] += rs * (g[k] * qw[k] - m1 - hat * m2);
                    g[k] *= hat;
                }
                sums.add(S_QW, g);
            }
            store_row(row_of<TS>(a.dx, r, a.lddx), t, T);
            if (a.flags & F_BRANCH) {
#pragma unroll
                for (int k = 0; k < E; ++k) T[k] *= a.scale, yv[k] *= rs_y;
                if (ROW) {
                    float dg[E], pb[E];
                    if (a.flags & F_POST) {
                        load_gain(a.pb, t, pb, 0.f);
#pragma unroll
                        for (int k = 0; k < E; ++k) dg[k] = T[k] * (yv[k] * pw[k] + pb[k]);
                    } else {
#pragma unroll
                        for (int k = 0; k < E; ++k) dg[k] = T[k] * yv[k];
                    }
#pragma unroll
                    for (int k = 0; k < E; ++k) {
                        const float ac = a.flags & F_SIGMOID ? sigmoid(gt[k]) : gt[k];
                        dg[k] *= a.flags & F_SIGMOID ? sigmoid_slope(gt[k], ac) : 1.f;
                        T[k] *= ac;
                    }
                    if (GATE == G_ROW && a.dgate) store_row(row_of<TB>(a.dgate, r, a.lddg), t, dg);
                    if (GATE == G_GROUP) {
                        sums.add(S_GATE, dg);
                        if (--left == 0) {
                            sums.get(S_GATE, dg);
                            if (a.dgate) store_row(row_of<TB>(a.dgate, gate, a.lddg), t, dg);
                            sums.zero(S_GATE);
                            left = a.u.span, gate += step;
                        }
                    }
                }
                if (SUM_T) sums.add(S_PB, T);
#pragma unroll
                for (int k = 0; k < E; ++k) {
                    g[k] = T[k] * yv[k];
                    if (GATE == G_SHARED) T[k] *= act[k];
                }
                sums.add(S_PW, g);
                if (a.flags & F_POST) {
#pragma unroll
                    for (int k = 0; k < E; ++k) T[k] *= pw[k];       // behind the row T is what the pre norm left there, pw is 0
                    float q[FULL ? 2 : 1] = {dot_e(T, yv)};
                    if (FULL) q[FULL ? 1 : 0] = sum_e(T);
                    t.sum(q);
                    const float m2 = q[0] * a.inv_c, m1 = FULL && (a.flags & F_LAYER) ? q[FULL ? 1 : 0] * a.inv_c : 0.f;
#pragma unroll
                    for (int k = 0; k < E; ++k) T[k] = rs_y * (T[k] - m1 - yv[k] * m2);
                }
                store_row(row_of<TB>(a.dy, r, a.lddy), t, T);
            }
        }
        if (GATE == G_SHARED) {
            float v[E], w[E], pb[E];
            sums.get(S_PW, v);
            sums.get(S_PB, w);
            load_gain(a.pb, t, pb, 0.f);
            // S_PB's place takes dgate until it is out
#pragma unroll
            for (int k = 0; k < E; ++k) pb[k] = a.flags & F_POST ? pw[k] * v[k] + pb[k] * w[k] : v[k];
            if (a.flags & F_SIGMOID && a.dgate) {
                float slope[E];
                if constexpr (BLK) {
                    load_row(row_of<const TB>(a.gate, group, a.ldg), t, slope);
#pragma unroll
                    for (int k = 0; k < E; ++k) slope[k] = sigmoid_slope(slope[k], act[k]);
                } else {
                    sums.get(S_GATE, slope);
                }
#pragma unroll
                for (int k = 0; k < E; ++k) pb[k] *= slope[k];
            }
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] *= act[k], w[k] *= act[k];
            sums.set(S_PW, v);
            sums.set(S_PB, pb);
            if (!BLK) __syncthreads();
            if (a.dgate) {
                if (a.u.per_group == 1) leave(S_PB, sums, t, lds, row_of<TB>(a.dgate, group, a.lddg), false);
                else leave(S_PB, sums, t, lds, a.gpart + (int64_t)u * a.pitch, false);
            }
            if (FULL) {
                if (!BLK) __syncthreads();
                sums.set(S_PB, w);
            }
        }
        if (!BLK) __syncthreads();
        const int64_t off = (int64_t)blockIdx.x * a.step;
        const bool add = u != blockIdx.x;
        if constexpr (BLK) {
            if (a.sums[0]) leave(S_PW, sums, t, lds, a.sums[0] + off, add);
            if (a.sums[2]) leave(S_QW, sums, t, lds, a.sums[2] + off, add);
            if (FULL && a.sums[1]) leave(S_PB, sums, t, lds, a.sums[1] + off, add);
            if (FULL && a.sums[3]) leave(S_QB, sums, t, lds, a.sums[3] + off, add);
        } else {                     // all columns of all sums at once: few columns would leave most threads idle
            const int n = (FULL ? 4 : 2) * a.C, s = splits(n, t), k = threadIdx.x & ((1 << s) - 1);
            for (int i = threadIdx.x >> s; i < n; i += blockDim.x >> s) {
                const int sum = i / a.C, c = i - sum * a.C;
                float* out = sum == S_PW ? a.sums[0] : sum == S_QW ? a.sums[2] : sum == S_PB ? a.sums[1] : a.sums[3];
                if (!out) continue;
                const float v = joined<NS>(sum, c, k, s, t, lds);
                out += off + c;
                if (k == 0) *out = add ? *out + v : v;
            }
            if (u + gridDim.x < a.u.units) __syncthreads();      // before the next unit's sums
        }
    }
}

// The partial sums of a backward pass joined in a fixed order: 4 columns a thread, LC threads side by side, 1024 / LC slices of the
// partial sums.  16 threads side by side read 256 bytes at a time (24 MB of sums for 6000 channels: 7.0 us, with 4 threads 12.9), 4
// give four times the workgroups where the columns are few (2 x 771: 5.4 us instead of 12.4).  blockIdx.y < 4: the gradient of that
// gain or bias over the workgroups; beyond: gate row blockIdx.y - 4 over its units, or, where these are few, a thread for 4 columns of
// any gate row (4000 x 1000 bf16 with 500 gate rows of 2 units: 26 us and not 45 for the call; 8192 x 4096 with 16 rows of 32 units:
// 114 and not 109).
constexpr int FEW_UNITS = 16;
struct JoinArgs {
    const float* part;
    float* out[4];
    int blocks, nslot, slot[4], C, pitch;
    const float* gpart;
    void* dgate;
    int64_t lddg;
    int per_group, branch_type, gates;
};

// 4 columns from c on of a row of dgate
__device__ __forceinline__ void store_gate(const JoinArgs& a, int64_t row, int c, const float (&s)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (c + k >= a.C) break;
        const int64_t i = row * a.lddg + c + k;
        if (a.branch_type == SR_T_F32) ((float*)a.dgate)[i] = s[k];
        else if (a.branch_type == SR_T_BF16) ((bf16_t*)a.dgate)[i] = (bf16_t)s[k];
        else ((f16_t*)a.dgate)[i] = (f16_t)s[k];
    }
}

template <int LC>
__global__ void __launch_bounds__(1024) rn_join_kernel(const JoinArgs a) {
    constexpr int SL = 1024 / LC;
    __shared__ float4 sm[SL * LC];
    const int cl = threadIdx.x % LC, sl = threadIdx.x / LC, c = (blockIdx.x * LC + cl) * 4, job = blockIdx.y;
    const bool gate = job >= 4;
    if (gate && a.per_group <= FEW_UNITS) {
        const int64_t q = a.pitch / 4, i = ((int64_t)(job - 4) * gridDim.x + blockIdx.x) * 1024 + threadIdx.x, row = i / q;
        if (row >= a.gates) return;
        const int at = (int)(i - row * q) * 4;
        const float* p = a.gpart + row * a.per_group * a.pitch + at;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int u = 0; u < a.per_group; ++u) {
            const float4 v = *reinterpret_cast<const float4*>(p + (int64_t)u * a.pitch);
            s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
        }
        store_gate(a, row, at, s);
        return;
    }
    if (!gate && !a.out[job]) return;
    const float* p = gate ? a.gpart + (int64_t)(job - 4) * a.per_group * a.pitch : a.part + (int64_t)a.slot[job] * a.pitch;
    const int64_t step = gate ? a.pitch : (int64_t)a.nslot * a.pitch;
    const int n = gate ? a.per_group : a.blocks;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < a.C) {                   // behind the last column is room, and what stands there stays unused
#pragma unroll 8
        for (int i = sl; i < n; i += SL) {
            const float4 v = *reinterpret_cast<const float4*>(p + i * step + c);
            s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
        }
    }
    // the slices, eight to one each time
#pragma unroll
    for (int h = SL; h > 1; h = (h + 7) / 8) {
        const int next = (h + 7) / 8;
        if (sl >= next && sl < h) sm[sl * LC + cl] = make_float4(s[0], s[1], s[2], s[3]);
        __syncthreads();
        if (sl < next) {
#pragma unroll
            for (int i = 1; i < 8; ++i) {
                if (sl + i * next >= h) break;
                const float4 o = sm[(sl + i * next) * LC + cl];
                s[0] += o.x, s[1] += o.y, s[2] += o.z, s[3] += o.w;
            }
        }
        __syncthreads();
    }
    if (sl) return;
    if (gate) {
        store_gate(a, job - 4, c, s);
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (c + k < a.C) a.out[job][c + k] = s[k];
}

// ------------------------------------------------------------------------------------------------- host
struct Shape {
    bool blk;
    int e;                           // elements of a lane
    int threads, tl, teams;          // threads of a workgroup, log2 of a team's lanes (rows within a wave), teams of a workgroup
};

Shape shape_of(const sr_residual_norm_desc* d, int e) {
    Shape s;
    const int lanes = (d->channels + e - 1) / e;
    s.e = e;
    s.blk = d->channels > WAVE_C;
    s.tl = 0;
    while (!s.blk && (1 << s.tl) < lanes) ++s.tl;
    s.threads = s.blk ? (lanes + 63) / 64 * 64 : 256;
    s.teams = s.blk ? 1 : 256 >> s.tl;
    return s;
}

struct Split {
    Units u = {1, 0, 1};
    int blocks = 0, resident = 0;    // workgroups; how many the GPU holds at once
    bool shared_gate = false;
};

// `waves`: how many waves of the kernel a CU holds at once; `tight`: a quarter of them on each of its four SIMDs and no more, so that a workgroup of 5 waves,
// which is two waves to one of them, fits twice and not three times (11648 x 1030 bf16 gated backward: 87 -> 70 us).  The workgroups are
// as many as that gives: a few more would cost a second round of them, and with many more a team has too few rows to have the next
// one on its way (16384 x 4096 bf16 forward: 100 us with 16 waves a CU, 105 with 48, 112 with one row a workgroup)
Split split_of(const sr_residual_norm_desc* d, const Shape& s, bool gate, unsigned rpg, int waves, bool tight) {
    Split p;
    if (d->rows == 0) return p;
    p.shared_gate = gate && rpg > 1;
    p.u.span = p.shared_gate ? rpg : (unsigned)d->rows;
    const int wg = s.threads / 64, fit = tight && wg > 4 ? waves / 4 / ((wg + 3) / 4) : waves / wg;
    const int64_t groups = d->rows / p.u.span, resident = p.resident = 256 * std::max(1, fit);
    const int64_t most = (p.u.span + s.teams - 1) / s.teams;
    p.u.per_group = (unsigned)std::min(most, std::max<int64_t>(1, resident / groups));
    p.u.units = (unsigned)(groups * p.u.per_group);
    p.blocks = (int)std::min<int64_t>(p.u.units, resident);
    return p;
}

// 16-bit tensors on both sides: a lane's 8 elements are one 16-byte vector; with fp32 on one side two vectors of 4, a team apart,
// so that a wave's access is contiguous there too
#define RN_TYPES(LAUNCH)                                                                              \
    do {                                                                                              \
        if (d->stream_type == SR_T_BF16) LAUNCH(bf16_t, bf16_t, 8);                                   \
        else if (d->stream_type == SR_T_F16) LAUNCH(f16_t, f16_t, 8);                                 \
        else if (d->branch_type == SR_T_F32) LAUNCH(float, float, 4);                                 \
        else if (d->branch_type == SR_T_BF16) LAUNCH(float, bf16_t, 4);                               \
        else LAUNCH(float, f16_t, 4);                                                                 \
    } while (0)

template <typename TS, typename TB, int VEC, bool BLK, bool TAIL>
void launch_fwd(const FwdArgs& a, int gate, int blocks, int threads, hipStream_t st) {
    if (gate == G_NONE) rn_fwd_kernel<TS, TB, 8, VEC, BLK, TAIL, G_NONE><<<blocks, threads, 0, st>>>(a);
    else if (gate == G_ROW) rn_fwd_kernel<TS, TB, 8, VEC, BLK, TAIL, G_ROW><<<blocks, threads, 0, st>>>(a);
    else rn_fwd_kernel<TS, TB, 8, VEC, BLK, TAIL, G_SHARED><<<blocks, threads, 0, st>>>(a);
}

template <typename TS, typename TB, int VEC>
void launch(const FwdArgs& a, bool blk, int gate, int blocks, int threads, hipStream_t st) {
    if (blk && a.C % VEC) launch_fwd<TS, TB, VEC, true, true>(a, gate, blocks, threads, st);
    else if (blk) launch_fwd<TS, TB, VEC, true, false>(a, gate, blocks, threads, st);
    else if (a.C % VEC) launch_fwd<TS, TB, VEC, false, true>(a, gate, blocks, threads, st);
    else launch_fwd<TS, TB, VEC, false, false>(a, gate, blocks, threads, st);
}

template <typename TS, typename TB, int E, int VEC, bool BLK, bool TAIL, int GATE, bool FULL>
void launch_bwd(const BwdArgs& a, int blocks, int threads, hipStream_t st) {
    const int lds = 4 * bwd_sums<GATE, FULL, BLK>() * E * threads + (BLK ? 1024 : 0);
    if (lds > 64 * 1024)             // a launch may have 64 KiB unless the function says more
        (void)hipFuncSetAttribute((const void*)rn_bwd_kernel<TS, TB, E, VEC, BLK, TAIL, GATE, FULL>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    rn_bwd_kernel<TS, TB, E, VEC, BLK, TAIL, GATE, FULL><<<blocks, threads, lds, st>>>(a);
}

template <typename TS, typename TB, int E, int VEC, bool BLK, bool TAIL>
void launch_bwd(const BwdArgs& a, int gate, bool full, int blocks, int threads, hipStream_t st) {
    if (gate == G_NONE) {
        if constexpr (E == 8 || sizeof(TS) == 4)      // see bwd_plan
            full ? launch_bwd<TS, TB, E, VEC, BLK, TAIL, G_NONE, true>(a, blocks, threads, st) : launch_bwd<TS, TB, E, VEC, BLK, TAIL, G_NONE, false>(a, blocks, threads, st);
    } else if (gate == G_GROUP) {
        if constexpr (!BLK)
            full ? launch_bwd<TS, TB, E, VEC, BLK, TAIL, G_GROUP, true>(a, blocks, threads, st) : launch_bwd<TS, TB, E, VEC, BLK, TAIL, G_GROUP, false>(a, blocks, threads, st);
    } else if (gate == G_ROW) full ? launch_bwd<TS, TB, E, VEC, BLK, TAIL, G_ROW, true>(a, blocks, threads, st) : launch_bwd<TS, TB, E, VEC, BLK, TAIL, G_ROW, false>(a, blocks, threads, st);
    else full ? launch_bwd<TS, TB, E, VEC, BLK, TAIL, G_SHARED, true>(a, blocks, threads, st) : launch_bwd<TS, TB, E, VEC, BLK, TAIL, G_SHARED, false>(a, blocks, threads, st);
}

template <typename TS, typename TB, int VEC>
void launch(const BwdArgs& a, const Shape& s, int gate, bool full, int blocks, hipStream_t st) {
    if (s.blk && s.e == 4) a.C % 4 ? launch_bwd<TS, TB, 4, 4, true, true>(a, gate, full, blocks, s.threads, st) : launch_bwd<TS, TB, 4, 4, true, false>(a, gate, full, blocks, s.threads, st);
    else if (s.blk) a.C % VEC ? launch_bwd<TS, TB, 8, VEC, true, true>(a, gate, full, blocks, s.threads, st) : launch_bwd<TS, TB, 8, VEC, true, false>(a, gate, full, blocks, s.threads, st);
    else a.C % VEC ? launch_bwd<TS, TB, 8, VEC, false, true>(a, gate, full, blocks, s.threads, st) : launch_bwd<TS, TB, 8, VEC, false, false>(a, gate, full, blocks, s.threads, st);
}

// A backward pass: the plan its workspace and its launch go by.  `full` (kernel template) is not known to the workspace query, which
// therefore takes the larger of both.
struct BwdPlan {
    Shape s;
    Split p;
    size_t part, bytes;              // bytes of the partial sums, of everything
    bool single;                     // one workgroup, which leaves the gradients themselves and needs no workspace
    bool group;                      // G_GROUP
};

BwdPlan bwd_plan(const sr_residual_norm_desc* d, bool gate, unsigned rpg, bool full) {
    BwdPlan q;
    const int C = d->channels;
    const bool whole8 = C % 8 == 0, whole4 = C % 4 == 0;
    // 8 elements a lane are fewer waves to a row and so more rows at a time, but with a gate or fp32 tensors more than the registers
    // hold.  us at 12 M elements, 8 elements a lane / 4:
    //   16 bits, no gate:      776 channels rms 35.5 / 37.5, layer 43 / 49; 1541: 37 / 46, 49 / 60; 4095: 39 / 45, 54 / 58
    //   16 bits, gated, % 8:   640: 54.6 / 51.0; 1304: 51 / 59; 2312: 50 / 61; 3400: 49 / 53;   other channels: 1541: 64 / 59; 4095: 68 / 57
    //   fp32, no gate, % 4, where 4 elements make rows of 9 to 12 waves, of which a CU holds one: 2056: 53 / 68, layer 63 / 75; 2600:
    //   55 / 62, 66 / 69;   else: 776: 59.9 / 56.3, 76 / 60; 1544: 57.6 / 53.7; 3400: 57 / 59, 69 / 67;   other channels: 2050: 66 / 54
    // Above 4096 channels 1024 lanes of 4 do not hold a row: 8 in any case, and most of these kernels spill.  Bytes of scratch a lane, gains
    // only / all sums: fp32 streams 0 / 0..20 and gated 0..68 / 44..108 where C % 4 == 0, else 108..148 / 236..268 and gated 200..280 /
    // 316..380; 16 bits gated 0 / 20..28 where C % 8 == 0, else 0 / 52 and gated 60..116 / 124..188.  us at 12 M elements, 5120 and 6145
    // channels: bf16 36 / 44 and 37 / 52, gated 49 / 59 and 56 / 79; fp32 58 / 67 and 73 / 93, gated 95 / 104 and 109 / 127 (the traffic alone: 27,
    // gated 36; 53, gated 71).  Of the shorter rows these do: 16 bits, odd, no gate, all sums (52); fp32 streams of odd channels with a gate
    // (12..44 above 512 channels, 28..60 for fp32 branches below).
    const int wide = (C + 255) / 256;
    const bool e8 = d->stream_type == SR_T_F32 ? !gate && whole4 && wide > 8 && wide <= 12 : !gate || (whole8 && C > 1024);
    q.s = shape_of(d, C <= WAVE_C || C > 4096 || e8 ? 8 : 4);
    // Few rows: one workgroup of up to 8 waves, and no launch that joins partial sums.  A call from Python takes 2.7 us less (of 17 to
    // 22).  On the GPU a team's only row takes 3 us less, two one after the other -2.5 .. 1, a third 0 .. 2 us more, with a gate 2 .. 5.
    const unsigned span = gate && rpg > 1 ? rpg : (unsigned)std::max<int64_t>(d->rows, 1);
    const int threads = q.s.blk ? q.s.threads : q.s.tl ? 512 : 256, teams = q.s.blk ? 1 : threads >> q.s.tl;
    const int64_t in_turn = d->rows / span * ((span + teams - 1) / teams);      // rows that a team then takes one after the other
    q.group = false;
    q.single = d->rows && in_turn <= (gate ? 2 : 3);
    if (q.single) {
        q.s.threads = threads, q.s.teams = teams;
        q.p.u = {span, (unsigned)(d->rows / span), 1};
        q.p.blocks = 1, q.p.shared_gate = gate && rpg > 1;
        q.part = q.bytes = 0;
        return q;
    }
    q.p = split_of(d, q.s, gate, rpg, q.s.blk || (!full && !gate && whole8) ? 16 : 12, q.s.e == 8 || !whole4);
    // Many gate rows, few rows each: a team takes a group by itself where that is a third of the rows one after the other, with 4 for
    // the joining of a group's sums by a workgroup (62,499 x 64 bf16, 3 rows each: 25 us and not 172; 1,333,332 x 3: 41 and not 10,568;
    // but 16 rows each, 62,496 x 64: 41 and not 55, 3 rows each, 1200 x 250: 14 and not 20)
    if (q.p.shared_gate && !q.s.blk && q.p.u.per_group == 1) {
        const int64_t groups = q.p.u.units, wgs = q.p.resident, teams = q.s.teams;
        const int64_t by_team = (groups + wgs * teams - 1) / (wgs * teams) * span, shared = (groups + wgs - 1) / wgs * ((span + teams - 1) / teams + 4);
        q.group = 3 * by_team <= shared;
        if (q.group) q.p.blocks = (int)std::min(wgs, (groups + teams - 1) / teams);
    }
    const size_t row = (size_t)round_up(d->channels, 4) * 4;
    q.part = round_up_sz((size_t)q.p.blocks * 4 * row);
    q.bytes = q.part + (q.p.shared_gate && q.p.u.per_group > 1 ? (size_t)q.p.u.units * row : 0);
    return q;
}

int check_desc(const sr_residual_norm_desc* d, const char* who) {
    if (!d) return fail(nullptr, SR_ERR_ARG, "%s: descriptor is NULL", who);
    if (d->rows < 0 || d->rows > 2000000000) return fail(nullptr, SR_ERR_ARG, "%s: rows must be 0 .. 2e9", who);
    if (d->channels < 1 || d->channels > MAX_C) return fail(nullptr, SR_ERR_ARG, "%s: channels must be 1 .. %d", who, MAX_C);
    if (!type_bytes(d->stream_type) || !type_bytes(d->branch_type)) return fail(nullptr, SR_ERR_ARG, "%s: unknown type", who);
    if (d->stream_type != d->branch_type && d->stream_type != SR_T_F32)
        return fail(nullptr, SR_ERR_ARG, "%s: the branch's type must be the stream's, or a 16-bit type beside an fp32 stream", who);
    if (d->kind != SR_NORM_RMS && d->kind != SR_NORM_LAYER) return fail(nullptr, SR_ERR_ARG, "%s: unknown kind", who);
    if (d->norms < 1 || d->norms > 3) return fail(nullptr, SR_ERR_ARG, "%s: norms must be SR_NORM_POST, SR_NORM_PRE or both", who);
    if (d->gate_act != SR_GATE_LINEAR && d->gate_act != SR_GATE_SIGMOID) return fail(nullptr, SR_ERR_ARG, "%s: unknown gate_act", who);
    if (!(d->eps > 0.f) || !(d->eps < 3e38f)) return fail(nullptr, SR_ERR_ARG, "%s: eps must be positive and finite", who);
    if (!(d->scale > -3e38f && d->scale < 3e38f)) return fail(nullptr, SR_ERR_ARG, "%s: scale must be finite", who);
    return SR_OK;
}

// rows that share a gate row
int check_gate(const sr_residual_norm_desc* d, bool gate, const char* who, unsigned* rpg) {
    *rpg = (unsigned)std::max<int64_t>(d->rows, 1);
    if (!gate) return SR_OK;
    if (d->rows_per_gate < 1 || (d->rows && (d->rows_per_gate > d->rows || d->rows % d->rows_per_gate)))
        return fail(nullptr, SR_ERR_ARG, "%s: rows_per_gate must divide the rows", who);
    if (d->rows) *rpg = (unsigned)d->rows_per_gate;
    return SR_OK;
}

int region(Region* out, const void* p, int64_t rows, int64_t ld, int C, int bytes, const char* who, const char* what) {
    *out = Region{(const char*)p, p ? rows : 0, ld * bytes, (int64_t)C * bytes};
    if (p && rows > 1 && (ld < C || ld > INT32_MAX)) return fail(nullptr, SR_ERR_ARG, "%s: the row pitch of %s is below the channels or over 2^31 - 1", who, what);
    if (p && (uintptr_t)p % bytes) return fail(nullptr, SR_ERR_ARG, "%s: %s is not aligned to its elements", who, what);
    return SR_OK;
}

// out may be `in` itself where a lane reads and writes the same elements, else they share nothing
int apart(const Region& out, const Region& in, bool may_be_same, const char* who) {
    if (disjoint(out, in) || (may_be_same && same(out, in))) return SR_OK;
    return fail(nullptr, SR_ERR_ARG, "%s: an output overlaps another tensor", who);
}

#define RN_TRY(call)          \
    do {                      \
        const int rc_ = call; \
        if (rc_) return rc_;  \
    } while (0)

}  // namespace

extern "C" int sr_op_residual_norm(int device, const sr_residual_norm_desc* d, const void* x, const void* y, const void* gate,
                                   const float* post_gain, const float* post_bias, const float* pre_gain, const float* pre_bias,
                                   void* h, void* n, void* hip_stream) {
    const char* who = "sr_op_residual_norm";
    RN_TRY(check_desc(d, who));
    const bool post = d->norms & SR_NORM_POST, pre = d->norms & SR_NORM_PRE;
    unsigned rpg;
    RN_TRY(check_gate(d, gate != nullptr, who, &rpg));
    const int sb = type_bytes(d->stream_type), bb = type_bytes(d->branch_type), C = d->channels;
    if (d->rows) {
        if (!x || (pre && !n) || (y && !h)) return fail(nullptr, SR_ERR_ARG, "%s: NULL tensor pointer", who);
        if (!y && (post || gate)) return fail(nullptr, SR_ERR_ARG, "%s: without a branch y there is only SR_NORM_PRE and no gate", who);
    }
    if (!y) h = nullptr;             // h would be x
    if (!pre) n = nullptr;
    Region in[3], rh, rn;
    RN_TRY(region(&in[0], x, d->rows, d->ldx, C, sb, who, "x"));
    RN_TRY(region(&in[1], y, d->rows, d->ldy, C, bb, who, "y"));
    RN_TRY(region(&in[2], gate, d->rows / rpg, d->ldg, C, bb, who, "gate"));
    RN_TRY(region(&rh, h, d->rows, d->ldh, C, sb, who, "h"));
    RN_TRY(region(&rn, n, d->rows, d->ldn, C, bb, who, "n"));
    for (const Region& o : {rh, rn}) {
        for (int i = 0; i < 3; ++i) RN_TRY(apart(o, in[i], i < 2 || rpg == 1, who));
        for (const float* p : {post_gain, post_bias, pre_gain, pre_bias}) {
            Region g;
            RN_TRY(region(&g, p, 1, C, C, 4, who, "a gain or bias"));
            RN_TRY(apart(o, g, false, who));
        }
    }
    RN_TRY(apart(rh, rn, false, who));
    OnDevice on;
    RN_TRY(on.enter(device));
    if (d->rows == 0) return SR_OK;
    const Shape s = shape_of(d, 8);
    const Split p = split_of(d, s, false, 1, 16, false);
    const int flags = (y ? F_BRANCH : 0) | (post ? F_POST : 0) | (pre ? F_PRE : 0) | (d->kind == SR_NORM_LAYER ? F_LAYER : 0) |
                      (d->gate_act == SR_GATE_SIGMOID ? F_SIGMOID : 0);
    const FwdArgs a = {x, y, gate, post ? post_gain : nullptr, post ? post_bias : nullptr, pre ? pre_gain : nullptr, pre ? pre_bias : nullptr,
                       h, n, (int)d->ldx, (int)d->ldy, (int)d->ldg, (int)d->ldh, (int)d->ldn, (unsigned)d->rows, rpg, C, s.tl, flags, d->scale, d->eps,
                       1.f / (float)C};
    hipStream_t st = (hipStream_t)hip_stream;
    const int gt = !gate ? G_NONE : rpg > 1 ? G_SHARED : G_ROW;
#define LAUNCH(TS, TB, VEC) launch<TS, TB, VEC>(a, s.blk, gt, p.blocks, s.threads, st)
    RN_TYPES(LAUNCH);
#undef LAUNCH
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(nullptr, SR_ERR_HIP, "launch residual_norm: %s", hipGetErrorString(e));
    return SR_OK;
}

extern "C" int sr_op_residual_norm_bwd_workspace(const sr_residual_norm_desc* d, int gate, size_t* bytes) {
    const char* who = "sr_op_residual_norm_bwd_workspace";
    RN_TRY(check_desc(d, who));
    if (!bytes) return fail(nullptr, SR_ERR_ARG, "%s: bytes is NULL", who);
    unsigned rpg;
    RN_TRY(check_gate(d, gate != 0, who, &rpg));
    *bytes = std::max(bwd_plan(d, gate != 0, rpg, false).bytes, bwd_plan(d, gate != 0, rpg, true).bytes);
    return SR_OK;
}

extern "C" int sr_op_residual_norm_bwd(int device, const sr_residual_norm_desc* d, const void* h, const void* y, const void* gate,
                                       const float* post_gain, const float* post_bias, const float* pre_gain, const void* dh,
                                       const void* dn, void* dx, void* dy, void* dgate, float* dpost_gain, float* dpost_bias,
                                       float* dpre_gain, float* dpre_bias, void* workspace, size_t workspace_bytes,
                                       void* hip_stream) {
    const char* who = "sr_op_residual_norm_bwd";
    RN_TRY(check_desc(d, who));
    const bool post = d->norms & SR_NORM_POST, pre = d->norms & SR_NORM_PRE;
    unsigned rpg;
    RN_TRY(check_gate(d, gate != nullptr, who, &rpg));
    const int sb = type_bytes(d->stream_type), bb = type_bytes(d->branch_type), C = d->channels;
    if (d->rows && !dy && (post || gate)) return fail(nullptr, SR_ERR_ARG, "%s: without a branch (dy) there is only SR_NORM_PRE and no gate", who);
    if (dgate && !gate) return fail(nullptr, SR_ERR_ARG, "%s: dgate without gate", who);
    if ((!post && (dpost_gain || dpost_bias)) || (!pre && (dpre_gain || dpre_bias)))
        return fail(nullptr, SR_ERR_ARG, "%s: a gradient of a norm that is not there", who);
    if (d->rows) {
        if (!dx || (pre && (!h || !dn)) || (!pre && !dh) || ((post || gate) && !y))
            return fail(nullptr, SR_ERR_ARG, "%s: NULL tensor pointer", who);
    }
    if (!post && !gate) y = nullptr;     // not needed
    Region in[5], out[3], wr[5];
    RN_TRY(region(&in[0], pre ? h : nullptr, d->rows, d->ldh, C, sb, who, "h"));
    RN_TRY(region(&in[1], y, d->rows, d->ldy, C, bb, who, "y"));
    RN_TRY(region(&in[2], dh, d->rows, d->lddh, C, sb, who, "dh"));
    RN_TRY(region(&in[3], pre ? dn : nullptr, d->rows, d->lddn, C, bb, who, "dn"));
    RN_TRY(region(&in[4], gate, d->rows / rpg, d->ldg, C, bb, who, "gate"));
    RN_TRY(region(&out[0], dx, d->rows, d->lddx, C, sb, who, "dx"));
    RN_TRY(region(&out[1], dy, d->rows, d->lddy, C, bb, who, "dy"));
    RN_TRY(region(&out[2], dgate, d->rows / rpg, d->lddg, C, bb, who, "dgate"));
    float* vec[4] = {dpost_gain, dpost_bias, dpre_gain, dpre_bias};
    for (int i = 0; i < 4; ++i) RN_TRY(region(&wr[i], vec[i], 1, C, C, 4, who, "a gradient of a gain or bias"));
    size_t need;
    RN_TRY(sr_op_residual_norm_bwd_workspace(d, gate != nullptr, &need));
    if (need && (!workspace || (uintptr_t)workspace % 16)) return fail(nullptr, SR_ERR_ARG, "%s: the workspace is NULL or not aligned to 16 bytes", who);
    if (workspace_bytes < need) return fail(nullptr, SR_ERR_ARG, "%s: the workspace holds %zu bytes, this call needs %zu", who, workspace_bytes, need);
    wr[4] = Region{(const char*)workspace, need ? 1 : 0, (int64_t)need, (int64_t)need};
    for (int o = 0; o < 3; ++o) {
        for (int i = 0; i < 5; ++i) RN_TRY(apart(out[o], in[i], rpg == 1 || (o < 2 && i < 4), who));
        for (int i = o + 1; i < 3; ++i) RN_TRY(apart(out[o], out[i], false, who));
        for (const Region& w : wr) RN_TRY(apart(out[o], w, false, who));
    }
    for (int o = 0; o < 5; ++o) {
        for (const Region& i : in) RN_TRY(apart(wr[o], i, false, who));
        for (int i = o + 1; i < 5; ++i) RN_TRY(apart(wr[o], wr[i], false, who));
    }
    for (const float* p : {post_gain, post_bias, pre_gain}) {
        Region g;
        RN_TRY(region(&g, p, 1, C, C, 4, who, "a gain or bias"));
        for (const Region& o : out) RN_TRY(apart(o, g, false, who));
        for (const Region& o : wr) RN_TRY(apart(o, g, false, who));
    }
    OnDevice on;
    RN_TRY(on.enter(device));
    hipStream_t st = (hipStream_t)hip_stream;
    const bool full = d->kind == SR_NORM_LAYER || dpost_bias || dpre_bias;
    const BwdPlan q = bwd_plan(d, gate != nullptr, rpg, full);
    const Split& p = q.p;
    float* part = (float*)workspace;
    float* gpart = (float*)((char*)workspace + q.part);
    JoinArgs j = {part, {}, p.blocks, 0, {-1, -1, -1, -1}, C, round_up(C, 4), gpart, dgate, d->lddg, (int)p.u.per_group, d->branch_type};
    float* sums[4];
    for (int i = 0; i < 4; ++i) {
        j.out[i] = sums[i] = vec[i];
        if (!vec[i] || q.single) continue;
        j.slot[i] = j.nslot++;
        sums[i] = part + (int64_t)j.slot[i] * j.pitch;
    }
    if (d->rows) {
        const int flags = (dy ? F_BRANCH : 0) | (post ? F_POST : 0) | (pre ? F_PRE : 0) | (d->kind == SR_NORM_LAYER ? F_LAYER : 0) |
                          (d->gate_act == SR_GATE_SIGMOID ? F_SIGMOID : 0) | (dh ? F_STREAM_GRAD : 0) | (y ? F_READ_Y : 0);
        const BwdArgs a = {h, y, gate, dh, dn, post ? post_gain : nullptr, post ? post_bias : nullptr, pre ? pre_gain : nullptr, dx, dy, dgate,
                           {sums[0], sums[1], sums[2], sums[3]}, (int64_t)j.nslot * j.pitch, gpart, j.pitch, (int)d->ldh, (int)d->ldy, (int)d->ldg, (int)d->lddh, (int)d->lddn, (int)d->lddx, (int)d->lddy,
                           (int)d->lddg, p.u, C, q.s.tl, flags, d->scale, d->eps,
                           1.f / (float)C};
        const int gt = !gate ? G_NONE : q.group ? G_GROUP : p.shared_gate ? G_SHARED : G_ROW;
#define LAUNCH(TS, TB, VEC) launch<TS, TB, VEC>(a, q.s, gt, full, p.blocks, st)
        RN_TYPES(LAUNCH);
#undef LAUNCH
    }
    hipError_t e = hipGetLastError();
    const unsigned gates = dgate && p.shared_gate && p.u.per_group > 1 ? (unsigned)(d->rows / rpg) : 0;
    if (e == hipSuccess && (j.nslot || gates)) {
        const bool wide = (int64_t)(j.nslot + gates) * C >= 2048;
        const unsigned across = (C + (wide ? 63 : 15)) / (wide ? 64 : 16);
        const int64_t quads = (int64_t)gates * (j.pitch / 4);
        j.gates = (int)gates;
        const dim3 grid(across, 4 + (p.u.per_group <= FEW_UNITS ? (unsigned)((quads + across * 1024 - 1) / (across * 1024)) : gates));
        if (wide) rn_join_kernel<16><<<grid, 1024, 0, st>>>(j);
        else rn_join_kernel<4><<<grid, 1024, 0, st>>>(j);
        e = hipGetLastError();
    }
    if (e != hipSuccess) return fail(nullptr, SR_ERR_HIP, "launch residual_norm_bwd: %s", hipGetErrorString(e));
    return SR_OK;
}
