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
// once: a group of lanes (a "team") holds it in registers, 8 elements a lane, across all sums of the row, and the backward pass
// takes the row statistics again from what it holds instead of reading them.  Rows of up to 512 channels belong to 1..64 lanes of a
// wave, several rows to a wave, and their sums are lane exchanges; longer rows belong to a workgroup, which joins its waves' sums
// in LDS.  All sums and the values between them are fp32; tensors of 16 bits are rounded once, when they are stored.
#include "op_host.h"
#include "row_math.h"

#include <algorithm>

using namespace sr;
using namespace srh;

namespace {

constexpr int MAX_C = 8192;          // 1024 lanes x 8 channels
constexpr int WAVE_C = 512;          // up to here a row belongs to lanes of one wave

struct FwdArgs {
    const void *x, *y, *gate;
    const float *pw, *pb, *qw, *qb;  // post gain / bias, pre gain / bias
    void *h, *n;
    int64_t ldx, ldy, ldg, ldh, ldn;
    unsigned rows, rpg;              // rpg: rows that share a gate row
    int C, tl;                       // tl: log2 of a team's lanes (rows within a wave)
    int layer, post, pre, sigmoid;
    float scale, eps, inv_c;
};

struct BwdArgs {
    const void *h, *y, *gate, *dh, *dn;
    const float *pw, *pb, *qw;
    void *dx, *dy, *dgate;
    float *part;                     // [blocks][nslot][C] partial sums of the gains' and biases' gradients
    float *gpart;                    // [units][C] partial sums of dgate where a gate row spans several units
    int64_t ldh, ldy, ldg, lddh, lddn, lddx, lddy, lddg;
    unsigned span;                   // rows of a group: those that share a gate row, or all
    unsigned units, chunk, per_group;   // a unit is `chunk` rows of one group; per_group units make up a group
    int by_row;                      // the gate has a row for every position
    int C, tl;
    int layer, post, pre, sigmoid;
    int nslot, slot[4];              // where post gain, post bias, pre gain, pre bias are in `part`; -1: not wanted
    float scale, eps, inv_c;
};

// What a thread knows about its place in a team.  A lane holds 8 elements as 8 / VEC vectors, `team` vectors apart.
template <int VEC, bool BLK>
struct Team {
    int lanes, lane, row, rows;      // lanes of a team, this thread's lane, its team's number in the workgroup, teams in the workgroup
    int tl, C;
    float* red;                      // BLK: [2][16][8] floats
    int phase = 0;

    __device__ Team(int tl_, int C_, float* red_) : tl(tl_), C(C_), red(red_) {
        if (BLK) {
            lanes = blockDim.x, lane = threadIdx.x, row = 0, rows = 1;
        } else {
            lanes = 1 << tl, lane = threadIdx.x & (lanes - 1), row = threadIdx.x >> tl, rows = blockDim.x >> tl;
        }
    }
    __device__ __forceinline__ int col(int j) const { return (j * lanes + lane) * VEC; }

    // sums of K values over the team, in every lane
    template <int K>
    __device__ __forceinline__ void sum(float (&v)[K]) {
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

template <typename T, int VEC, bool TAIL, bool BLK>
__device__ __forceinline__ void load_row(const T* p, const Team<VEC, BLK>& t, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8 / VEC; ++j) {
        const int c = t.col(j);
        float o[VEC];
        if (c + VEC <= t.C) {
            load_vec<T, VEC>(p + c, o);
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) o[k] = TAIL && c + k < t.C ? (float)p[c + k] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[j * VEC + k] = o[k];
    }
}

template <typename T, int VEC, bool TAIL, bool BLK>
__device__ __forceinline__ void store_row(T* p, const Team<VEC, BLK>& t, const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8 / VEC; ++j) {
        const int c = t.col(j);
        float o[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = v[j * VEC + k];
        if (c + VEC <= t.C) {
            store_vec<T, VEC>(p + c, o);
        } else if (TAIL) {
#pragma unroll
            for (int k = 0; k < VEC; ++k)
                if (c + k < t.C) p[c + k] = (T)o[k];
        }
    }
}

// v -= mean over the row (0 beyond it)
template <int VEC, bool TAIL, bool BLK>
__device__ __forceinline__ void centre(float (&v)[8], float mean, const Team<VEC, BLK>& t) {
#pragma unroll
    for (int j = 0; j < 8 / VEC; ++j)
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[j * VEC + k] = t.col(j) + k < t.C ? v[j * VEC + k] - mean : 0.f;
}

__device__ __forceinline__ float sum8(const float (&v)[8]) {
    return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
}
__device__ __forceinline__ float dot8(const float (&a)[8], const float (&b)[8]) {
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k += 2) s += a[k] * b[k], u += a[k + 1] * b[k + 1];
    return s + u;
}
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + expf(-g)); }   // rcp: 1 ulp

template <int VEC, bool TAIL, bool BLK>
__device__ __forceinline__ void load_gain(const float* p, const Team<VEC, BLK>& t, float (&v)[8], float none) {
    if (p) {
        load_row<float, VEC, TAIL, BLK>(p, t, v);
    } else {                         // 0 beyond the row: what is multiplied by a gain needs no further mask
#pragma unroll
        for (int j = 0; j < 8 / VEC; ++j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[j * VEC + k] = t.col(j) + k < t.C ? none : 0.f;
    }
}

// ------------------------------------------------------------------------------------------------- forward
// v becomes hat(v); returns nothing else, the statistics live only here
template <int VEC, bool TAIL, bool BLK>
__device__ __forceinline__ void normalise(float (&v)[8], const FwdArgs& a, Team<VEC, BLK>& t) {
    if (a.layer) {
        float m[1] = {sum8(v)};
        t.sum(m);
        centre<VEC, TAIL, BLK>(v, m[0] * a.inv_c, t);
    }
    float s[1] = {dot8(v, v)};
    t.sum(s);
    const float rs = rsqrtf(s[0] * a.inv_c + a.eps);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= rs;
}

template <typename TS, typename TB, int VEC, bool TAIL, bool BLK>
__global__ void __launch_bounds__(BLK ? 1024 : 256) rn_fwd_kernel(const FwdArgs a) {
    __shared__ float red[BLK ? 256 : 1];
    Team<VEC, BLK> t(a.tl, a.C, red);
    float pw[8], pb[8], qw[8], qb[8];
    load_gain<VEC, TAIL, BLK>(a.pw, t, pw, 1.f);
    load_gain<VEC, TAIL, BLK>(a.pb, t, pb, 0.f);
    load_gain<VEC, TAIL, BLK>(a.qw, t, qw, 1.f);
    load_gain<VEC, TAIL, BLK>(a.qb, t, qb, 0.f);
    for (unsigned r = blockIdx.x * t.rows + t.row; r < a.rows; r += gridDim.x * t.rows) {
        float h[8], p[8], g[8];
        load_row<TS, VEC, TAIL, BLK>((const TS*)a.x + r * a.ldx, t, h);
        if (a.y) {
            load_row<TB, VEC, TAIL, BLK>((const TB*)a.y + r * a.ldy, t, p);
            if (a.gate) load_row<TB, VEC, TAIL, BLK>((const TB*)a.gate + (a.rpg == 1 ? r : r / a.rpg) * a.ldg, t, g);
            if (a.post) {
                normalise<VEC, TAIL, BLK>(p, a, t);
#pragma unroll
                for (int k = 0; k < 8; ++k) p[k] = p[k] * pw[k] + pb[k];
            }
            if (a.gate) {
#pragma unroll
                for (int k = 0; k < 8; ++k) p[k] *= a.sigmoid ? sigmoid(g[k]) : g[k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) h[k] += a.scale * p[k];
            store_row<TS, VEC, TAIL, BLK>((TS*)a.h + r * a.ldh, t, h);
        }
        if (a.pre) {
            normalise<VEC, TAIL, BLK>(h, a, t);
#pragma unroll
            for (int k = 0; k < 8; ++k) h[k] = h[k] * qw[k] + qb[k];
            store_row<TB, VEC, TAIL, BLK>((TB*)a.n + r * a.ldn, t, h);
        }
    }
}

// ------------------------------------------------------------------------------------------------- backward
// Sums of an accumulator over the teams of a workgroup; the threads of team 0 end with them.  `buf`: 4 waves x 512 floats.
template <int VEC>
__device__ __forceinline__ void join_teams(float (&v)[8], const Team<VEC, false>& t, float* buf) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
        for (int d = t.lanes; d < 64; d <<= 1) v[k] += __shfl_xor(v[k], d);
    const int wave = threadIdx.x >> 6;
    __syncthreads();                 // the buffer's last readers are done
    if ((threadIdx.x & 63) < t.lanes) {
#pragma unroll
        for (int k = 0; k < 8; ++k) buf[wave * 512 + k * 64 + t.lane] = v[k];
    }
    __syncthreads();
    if ((int)threadIdx.x < t.lanes) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (buf[k * 64 + t.lane] + buf[512 + k * 64 + t.lane]) + (buf[1024 + k * 64 + t.lane] + buf[1536 + k * 64 + t.lane]);
    }
}

template <typename TS, typename TB, int VEC, bool TAIL, bool BLK>
__global__ void __launch_bounds__(BLK ? 1024 : 256) rn_bwd_kernel(const BwdArgs a) {
    __shared__ float buf[BLK ? 256 : 2048];
    Team<VEC, BLK> t(a.tl, a.C, buf);
    float pw[8], pb[8], qw[8];
    load_gain<VEC, TAIL, BLK>(a.pw, t, pw, 1.f);
    load_gain<VEC, TAIL, BLK>(a.pb, t, pb, 0.f);
    load_gain<VEC, TAIL, BLK>(a.qw, t, qw, 1.f);
    float s_pw[8] = {}, s_pb[8] = {}, s_qw[8] = {}, s_qb[8] = {};
    const bool shared_gate = a.dgate && !a.by_row;
    for (unsigned u = blockIdx.x; u < a.units; u += gridDim.x) {
        const unsigned group = u / a.per_group, first = (u - group * a.per_group) * a.chunk;
        const unsigned r0 = group * a.span + first, r1 = r0 + min(a.chunk, a.span - first);
        float s_g[8] = {};
        for (unsigned r = r0 + t.row; r < r1; r += t.rows) {
            float hv[8], yv[8], T[8], g[8], gt[8];
            if (a.pre) load_row<TS, VEC, TAIL, BLK>((const TS*)a.h + r * a.ldh, t, hv);
            if (a.y) load_row<TB, VEC, TAIL, BLK>((const TB*)a.y + r * a.ldy, t, yv);
            if (a.pre) load_row<TB, VEC, TAIL, BLK>((const TB*)a.dn + r * a.lddn, t, g);
            if (a.dh) {
                load_row<TS, VEC, TAIL, BLK>((const TS*)a.dh + r * a.lddh, t, T);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) T[k] = 0.f;
            }
            if (a.gate) load_row<TB, VEC, TAIL, BLK>((const TB*)a.gate + (a.by_row ? r : group) * a.ldg, t, gt);
            if (a.layer) {
                float m[2] = {a.pre ? sum8(hv) : 0.f, a.post ? sum8(yv) : 0.f};
                t.sum(m);
                if (a.pre) centre<VEC, TAIL, BLK>(hv, m[0] * a.inv_c, t);
                if (a.post) centre<VEC, TAIL, BLK>(yv, m[1] * a.inv_c, t);
            }
            float rs_y = 0.f;
            {
                float s[4] = {0.f, 0.f, 0.f, 0.f};
                float w[8];
                if (a.pre) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) w[k] = g[k] * qw[k];
                    s[0] = dot8(hv, hv), s[1] = dot8(w, hv), s[2] = sum8(w);
                }
                if (a.post) s[3] = dot8(yv, yv);
                t.sum(s);
                rs_y = rsqrtf(s[3] * a.inv_c + a.eps);
                if (a.pre) {
                    const float rs = rsqrtf(s[0] * a.inv_c + a.eps);
                    const float m2 = s[1] * rs * a.inv_c, m1 = a.layer ? s[2] * a.inv_c : 0.f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float hat = hv[k] * rs;
                        s_qw[k] += g[k] * hat;
                        s_qb[k] += g[k];
                        T[k] += rs * (w[k] - m1 - hat * m2);
                    }
                }
            }
            store_row<TS, VEC, TAIL, BLK>((TS*)a.dx + r * a.lddx, t, T);
            if (!a.dy) continue;
#pragma unroll
            for (int k = 0; k < 8; ++k) T[k] *= a.scale;
            if (a.post) {
#pragma unroll
                for (int k = 0; k < 8; ++k) yv[k] *= rs_y;
            }
            if (a.gate) {
                float dg[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float act = a.sigmoid ? sigmoid(gt[k]) : gt[k], slope = a.sigmoid ? act * (1.f - act) : 1.f;
                    const float p = a.post ? yv[k] * pw[k] + pb[k] : yv[k];
                    dg[k] = T[k] * p * slope;
                    T[k] *= act;
                }
                if (shared_gate) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) s_g[k] += dg[k];
                } else if (a.dgate) {
                    store_row<TB, VEC, TAIL, BLK>((TB*)a.dgate + r * a.lddg, t, dg);
                }
            }
            if (a.post) {
                float q[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    s_pw[k] += T[k] * yv[k];
                    s_pb[k] += T[k];
                    q[k] = T[k] * pw[k];     // beyond the row T is what the pre norm left there, pw is 0
                }
                float s[2] = {sum8(q), dot8(q, yv)};
                t.sum(s);
                const float m1 = a.layer ? s[0] * a.inv_c : 0.f, m2 = s[1] * a.inv_c;
#pragma unroll
                for (int k = 0; k < 8; ++k) T[k] = rs_y * (q[k] - m1 - yv[k] * m2);
            }
            store_row<TB, VEC, TAIL, BLK>((TB*)a.dy + r * a.lddy, t, T);
        }
        if (shared_gate) {
            if constexpr (!BLK) join_teams<VEC>(s_g, t, buf);
            if (t.row == 0) {
                if (a.per_group == 1)
                    store_row<TB, VEC, TAIL, BLK>((TB*)a.dgate + group * a.lddg, t, s_g);
                else
                    store_row<float, VEC, TAIL, BLK>(a.gpart + (int64_t)u * a.C, t, s_g);
            }
        }
    }
    float* part = a.part + (int64_t)blockIdx.x * a.nslot * a.C;
    const float(*all[4])[8] = {&s_pw, &s_pb, &s_qw, &s_qb};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (a.slot[i] < 0) continue;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (*all[i])[k];
        if constexpr (!BLK) join_teams<VEC>(v, t, buf);
        if (t.row == 0) store_row<float, VEC, TAIL, BLK>(part + (int64_t)a.slot[i] * a.C, t, v);
    }
}

// The partial sums of a backward pass joined in a fixed order: 16 columns x 64 slices a workgroup.  blockIdx.y < 4: the gradient
// of that gain or bias over the workgroups; beyond: gate row blockIdx.y - 4 over its units.
struct JoinArgs {
    const float* part;
    float* out[4];
    int blocks, nslot, slot[4], C;
    const float* gpart;
    void* dgate;
    int64_t lddg;
    int per_group, branch_type;
};

__global__ void __launch_bounds__(1024) rn_join_kernel(const JoinArgs a) {
    __shared__ float sm[64][17];
    const int cl = threadIdx.x & 15, sl = threadIdx.x >> 4, c = blockIdx.x * 16 + cl, job = blockIdx.y;
    const bool gate = job >= 4;
    if (!gate && !a.out[job]) return;
    const float* p = gate ? a.gpart + (int64_t)(job - 4) * a.per_group * a.C : a.part + (int64_t)a.slot[job] * a.C;
    const int64_t step = gate ? a.C : (int64_t)a.nslot * a.C;
    const int n = gate ? a.per_group : a.blocks;
    float s = 0.f;
    if (c < a.C) {
#pragma unroll 8
        for (int i = sl; i < n; i += 64) s += p[i * step + c];
    }
    sm[sl][cl] = s;
    __syncthreads();
    if (sl < 8) {
#pragma unroll
        for (int i = 1; i < 8; ++i) s += sm[sl + 8 * i][cl];
    }
    __syncthreads();
    if (sl < 8) sm[sl][cl] = s;
    __syncthreads();
    if (sl || c >= a.C) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += sm[i][cl];
    if (!gate)
        a.out[job][c] = s;
    else if (a.branch_type == SR_T_F32)
        ((float*)a.dgate)[(job - 4) * a.lddg + c] = s;
    else if (a.branch_type == SR_T_BF16)
        ((bf16_t*)a.dgate)[(job - 4) * a.lddg + c] = (bf16_t)s;
    else
        ((f16_t*)a.dgate)[(job - 4) * a.lddg + c] = (f16_t)s;
}

// ------------------------------------------------------------------------------------------------- host
struct Shape {
    bool blk, tail;
    int threads, tl, teams;          // threads of a workgroup, log2 of a team's lanes (rows within a wave), teams of a workgroup
};

// 16-bit tensors on both sides: a lane's 8 elements are one 16-byte vector; with fp32 on one side two vectors of 4, a team apart,
// so that a wave's access is contiguous there too
int vec_of(int stream_type) { return stream_type == SR_T_F32 ? 4 : 8; }

Shape shape_of(int C, int vec) {
    Shape s;
    const int lanes = (C + 7) / 8;
    s.blk = C > WAVE_C;
    s.tail = C % vec != 0;
    s.tl = 0;
    while (!s.blk && (1 << s.tl) < lanes) ++s.tl;
    s.threads = s.blk ? (lanes + 63) / 64 * 64 : 256;
    s.teams = s.blk ? 1 : 256 >> s.tl;
    return s;
}

// Work split of a backward pass: units of `chunk` rows inside one group of rows that share a gate row (without such a gate all
// rows are one group), `blocks` workgroups over them
struct Split {
    unsigned span = 1, chunk = 1, per_group = 1, units = 0;
    int blocks = 0;
    bool shared_gate = false;
};

Split split_of(const sr_residual_norm_desc* d, const Shape& s, bool gate, unsigned rpg) {
    Split p;
    if (d->rows == 0) return p;
    p.shared_gate = gate && rpg > 1;
    p.span = p.shared_gate ? rpg : (unsigned)d->rows;
    const int64_t target = s.blk ? (s.threads > 512 ? 256 : 512) : 1024;
    int64_t chunk = (d->rows + target - 1) / target;
    chunk = std::min<int64_t>((chunk + s.teams - 1) / s.teams * s.teams, p.span);
    p.chunk = (unsigned)chunk;
    p.per_group = (unsigned)((p.span + chunk - 1) / chunk);
    p.units = (unsigned)(d->rows / p.span * p.per_group);
    p.blocks = (int)std::min<int64_t>(p.units, 2 * target);
    return p;
}

#define RN_TYPES(LAUNCH)                                                                              \
    do {                                                                                              \
        if (d->stream_type == SR_T_BF16) LAUNCH(bf16_t, bf16_t, 8);                                   \
        else if (d->stream_type == SR_T_F16) LAUNCH(f16_t, f16_t, 8);                                 \
        else if (d->branch_type == SR_T_F32) LAUNCH(float, float, 4);                                 \
        else if (d->branch_type == SR_T_BF16) LAUNCH(float, bf16_t, 4);                               \
        else LAUNCH(float, f16_t, 4);                                                                 \
    } while (0)

#define RN_SHAPES(KERNEL, TS, TB, VEC, GRID)                                                                          \
    do {                                                                                                              \
        if (s.blk && s.tail) KERNEL<TS, TB, VEC, true, true><<<GRID, s.threads, 0, st>>>(a);                          \
        else if (s.blk) KERNEL<TS, TB, VEC, false, true><<<GRID, s.threads, 0, st>>>(a);                              \
        else if (s.tail) KERNEL<TS, TB, VEC, true, false><<<GRID, s.threads, 0, st>>>(a);                             \
        else KERNEL<TS, TB, VEC, false, false><<<GRID, s.threads, 0, st>>>(a);                                        \
    } while (0)

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
    if (p && rows > 1 && (ld < C || ld > ((int64_t)1 << 40))) return fail(nullptr, SR_ERR_ARG, "%s: the row pitch of %s is below the channels or over 2^40", who, what);
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
    const Shape s = shape_of(C, vec_of(d->stream_type));
    const FwdArgs a = {x, y, gate, post ? post_gain : nullptr, post ? post_bias : nullptr, pre ? pre_gain : nullptr,
                       pre ? pre_bias : nullptr, h, n, d->ldx, d->ldy, d->ldg, d->ldh, d->ldn, (unsigned)d->rows, rpg, C, s.tl,
                       d->kind == SR_NORM_LAYER, post, pre, d->gate_act == SR_GATE_SIGMOID, d->scale, d->eps, 1.f / (float)C};
    const int grid = (int)std::min<int64_t>((d->rows + s.teams - 1) / s.teams, 1 << 20);
    hipStream_t st = (hipStream_t)hip_stream;
#define LAUNCH(TS, TB, VEC) RN_SHAPES(rn_fwd_kernel, TS, TB, VEC, grid)
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
    const Split p = split_of(d, shape_of(d->channels, vec_of(d->stream_type)), gate != 0, rpg);
    const size_t row = (size_t)d->channels * 4;
    *bytes = round_up_sz((size_t)p.blocks * 4 * row) + (p.shared_gate && p.per_group > 1 ? (size_t)p.units * row : 0);
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
    const Shape s = shape_of(C, vec_of(d->stream_type));
    const Split p = split_of(d, s, gate != nullptr, rpg);
    float* part = (float*)workspace;
    float* gpart = (float*)((char*)workspace + round_up_sz((size_t)p.blocks * 4 * C * 4));
    JoinArgs j = {part, {}, p.blocks, 0, {-1, -1, -1, -1}, C, gpart, dgate, d->lddg, (int)p.per_group, d->branch_type};
    for (int i = 0; i < 4; ++i) {
        j.out[i] = vec[i];
        if (vec[i]) j.slot[i] = j.nslot++;
    }
    if (d->rows) {
        const BwdArgs a = {h, y, gate, dh, dn, post ? post_gain : nullptr, post ? post_bias : nullptr, pre ? pre_gain : nullptr, dx, dy, dgate,
                           part, gpart, d->ldh, d->ldy, d->ldg, d->lddh, d->lddn, d->lddx, d->lddy, d->lddg, p.span,
                           p.units, p.chunk, p.per_group, gate && rpg == 1, C, s.tl, d->kind == SR_NORM_LAYER, post, pre, d->gate_act == SR_GATE_SIGMOID,
                           j.nslot, {j.slot[0], j.slot[1], j.slot[2], j.slot[3]}, d->scale, d->eps, 1.f / (float)C};
#define LAUNCH(TS, TB, VEC) RN_SHAPES(rn_bwd_kernel, TS, TB, VEC, p.blocks)
        RN_TYPES(LAUNCH);
#undef LAUNCH
    }
    hipError_t e = hipGetLastError();
    const unsigned gates = dgate && p.shared_gate && p.per_group > 1 ? (unsigned)(d->rows / rpg) : 0;
    if (e == hipSuccess && (j.nslot || gates)) {
        rn_join_kernel<<<dim3((C + 15) / 16, 4 + gates), 1024, 0, st>>>(j);
        e = hipGetLastError();
    }
    if (e != hipSuccess) return fail(nullptr, SR_ERR_HIP, "launch residual_norm_bwd: %s", hipGetErrorString(e));
    return SR_OK;
}
