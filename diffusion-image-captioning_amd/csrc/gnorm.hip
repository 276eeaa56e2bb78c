// The norms around a block with its gate and the residual scale: n = post(y), x_new = r x + gate n, a = pre(x_new), and the gradients.
//   u = (v - mean) rstd;  layer: mean = sum v / D, rstd = (sum (v - mean)^2 / D + eps)^-1/2;  rms: mean = 0;  norm(v) = u w + b
//   norm'(g) = rstd (g w - [layer] sum(g w) / D - u sum(g w u) / D);  dw = sum over rows of g u, db = sum over rows of g
// One pass over the rows in each direction, bound by memory: forward reads x, y and writes x_new, a; backward reads dx_new, da, x_new, y and writes dx, dy.
// A team of TPR threads holds a row in registers, NV groups of 4 consecutive elements per thread, and forms its sums by shuffles (and LDS where a
// team is several waves).  Loads are of 4 elements at any alignment of whole elements, the last group of a row that is no multiple of 4 by element.
#include <cmath>
#include <type_traits>
#include "common.h"
#include "../../include/dic_hip.h"

namespace {

struct Norm { const float *w, *b; int kind; float eps; };
struct NormArgs {
    const void *x, *y, *dx_new, *da;
    void *x_new, *a, *dx, *dy;
    const float* gate;
    float* saved;
    float *dgate;                       // final rows of dgate, or (gate_parts > 1) its partial sums [segment][part][D]
    float *cols;                        // backward: column sums of a block, [block][4][D]: dpost_w, dpost_b, dpre_w, dpre_b
    Norm post, pre;
    long long rows, seg_rows;           // rows that share a gate row
    long long pieces, piece_rows;       // backward: a piece is a run of rows of one segment, gate_parts pieces to a segment
    int gate_parts, pieces_per_block;
    int D;
    float r, inv_d;
};

// 4 elements as they lie in memory, at any whole-element address; `cnt` of them exist
template <typename T> struct Raw;
template <> struct Raw<bf16_t> {
    uint2 v;
    __device__ __forceinline__ void load(const bf16_t* p, int cnt) {
        v = make_uint2(0u, 0u);
        if (cnt == 4) __builtin_memcpy(&v, p, 8);
        else if (cnt > 0) {
            v.x = p[0] | (cnt > 1 ? (unsigned)p[1] << 16 : 0u);
            v.y = cnt > 2 ? p[2] : 0u;
        }
    }
    __device__ __forceinline__ f32x4 f() const {
        return f32x4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
    }
};
template <> struct Raw<float> {
    f32x4 v;
    __device__ __forceinline__ void load(const float* p, int cnt) {
        v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (cnt == 4) __builtin_memcpy(&v, p, 16);
        else {
#pragma unroll
            for (int e = 0; e < 3; ++e) if (e < cnt) v[e] = p[e];
        }
    }
    __device__ __forceinline__ f32x4 f() const { return v; }
};
template <typename T> __device__ __forceinline__ void stv(T* p, f32x4 v, int cnt) {
    if (cnt == 4) {
        if constexpr (sizeof(T) == 2) { const uint2 u = make_uint2(pack2bf(v[0], v[1]), pack2bf(v[2], v[3])); __builtin_memcpy(p, &u, 8); }
        else __builtin_memcpy(p, &v, 16);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e) if (e < cnt) Elem<T>::st(p + e, v[e]);
    }
}

// Sums over 16 lanes by lane permutations inside the adds (two neighbours, two pairs, two quads, two eights), over a wave by reading the four sums:
// a row's statistics are two dependent sums, and through LDS (ds_bpermute) each took six round trips.
template <int CTRL> __device__ __forceinline__ float dpp(float v) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)); }
__device__ __forceinline__ float sum16(float v) {
    v += dpp<0xB1>(v);          // quad_perm 1 0 3 2
    v += dpp<0x4E>(v);          // quad_perm 2 3 0 1
    v += dpp<0x141>(v);         // row_half_mirror
    v += dpp<0x140>(v);         // row_mirror
    return v;
}
__device__ __forceinline__ float sum64(float v) {
    const int s = __float_as_int(sum16(v));
    return (__int_as_float(__builtin_amdgcn_readlane(s, 0)) + __int_as_float(__builtin_amdgcn_readlane(s, 16)))
           + (__int_as_float(__builtin_amdgcn_readlane(s, 32)) + __int_as_float(__builtin_amdgcn_readlane(s, 48)));
}

template <int TPR, int NV> struct Team {
    static constexpr int THREADS = TPR > 256 ? TPR : 256, TEAMS = THREADS / TPR, WAVES = TPR / 64, WIDTH = TPR * NV * 4;
    int lane, col[NV], cnt[NV];
    __device__ __forceinline__ Team(int D) {
        lane = threadIdx.x % TPR;
#pragma unroll
        for (int c = 0; c < NV; ++c) { col[c] = (c * TPR + lane) * 4; cnt[c] = D - col[c] < 0 ? 0 : D - col[c] > 4 ? 4 : D - col[c]; }
    }
    template <typename T> __device__ __forceinline__ void load(const void* p, long long at, Raw<T> (&v)[NV]) const {
#pragma unroll
        for (int c = 0; c < NV; ++c) v[c].load((const T*)p + at + col[c], cnt[c]);
    }
    __device__ __forceinline__ void load_or(const float* p, float other, f32x4 (&v)[NV]) const {
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            Raw<float> r;
            r.v = f32x4{other, other, other, other};
            if (p) r.load(p + col[c], cnt[c]);
            v[c] = r.v;
        }
    }
    template <typename T> __device__ __forceinline__ void store(void* p, long long at, const f32x4 (&v)[NV]) const {
#pragma unroll
        for (int c = 0; c < NV; ++c) stv<T>((T*)p + at + col[c], v[c], cnt[c]);
    }
    // both sums over the team, in every lane.  Teams of several waves: `red` has 2 slots per wave; calls alternate between two halves of it, so that one
    // barrier per call is enough.
    __device__ __forceinline__ void sum2(float& a, float& b, float* red, int& turn) const {
        if constexpr (TPR == 16) { a = sum16(a); b = sum16(b); }
        else { a = sum64(a); b = sum64(b); }
        if constexpr (TPR > 64) {
            float* at = red + (turn & 1) * 2 * WAVES;
            turn ^= 1;
            if ((threadIdx.x & 63) == 0) { at[2 * (threadIdx.x >> 6)] = a; at[2 * (threadIdx.x >> 6) + 1] = b; }
            __syncthreads();
            a = 0.f; b = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) { a += at[2 * w]; b += at[2 * w + 1]; }
        }
    }
};
// N vectors of D floats that every row uses.  Several teams in a workgroup: in LDS, since registers are what limits the rows in flight; one team: in its
// registers, where each thread needs its own columns only.
template <int TPR, int NV, int N> struct Vectors {
    using TM = Team<TPR, NV>;
    static constexpr bool SHARED = TM::TEAMS > 1;
    f32x4 own[SHARED ? 1 : N][SHARED ? 1 : NV];
    __device__ __forceinline__ f32x4 get(const float* lds, const TM& tm, int k, int c) const {
        if constexpr (SHARED) return *(const f32x4*)(lds + k * TM::WIDTH + tm.col[c]);
        else return own[k][c];
    }
    // (shared: every thread of the workgroup calls, with barriers around the calls)
    __device__ __forceinline__ void set(float* lds, const TM& tm, int k, const float* p, float other, int D, const float* times = nullptr) {
        if constexpr (SHARED) {
            for (int i = threadIdx.x; i < TM::WIDTH; i += TM::THREADS) lds[k * TM::WIDTH + i] = i < D ? (p ? p[i] : other) * (times ? times[i] : 1.f) : 0.f;
        } else {
            tm.load_or(p, other, own[k]);
            if (times) {
                f32x4 t[NV];
                tm.load_or(times, 1.f, t);
#pragma unroll
                for (int c = 0; c < NV; ++c) own[k][c] = own[k][c] * t[c];
            }
        }
    }
};
__device__ __forceinline__ float hsum(f32x4 v) { return (v[0] + v[1]) + (v[2] + v[3]); }

// mean and rstd of a row; two passes over the registers
template <int TPR, int NV>
__device__ __forceinline__ void moments(const Team<TPR, NV>& tm, const f32x4 (&v)[NV], const Norm& n, float inv_d, float* red, int& turn, float& mean, float& rstd) {
    float s = 0.f, q = 0.f;
    mean = 0.f;
    if (n.kind == DIC_NORM_LAYER) {
#pragma unroll
        for (int c = 0; c < NV; ++c) s += hsum(v[c]);
        tm.sum2(s, q, red, turn);
        mean = s * inv_d;
        q = 0.f;
    }
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) { const float d = e < tm.cnt[c] ? v[c][e] - mean : 0.f; q += d * d; }
    s = 0.f;
    tm.sum2(q, s, red, turn);
    rstd = 1.0f / sqrtf(q * inv_d + n.eps);
}

// A team walks rows and has the next one on its way while it works on one.  135168 rows of 768, bf16: 839 MB in 183 us, 4.6 TB/s, what a copy reaches.
template <typename T, typename TX, int TPR, int NV>
__global__ __launch_bounds__((Team<TPR, NV>::THREADS)) void gated_norm_fwd_kernel(const NormArgs p) {
    using TM = Team<TPR, NV>;
    using VS = Vectors<TPR, NV, 4>;
    __shared__ float red[TPR > 64 ? 4 * TM::WAVES : 1];
    __shared__ __attribute__((aligned(16))) float vec[VS::SHARED ? 4 * TM::WIDTH : 1];
    enum { W2, B2, W1, B1 };
    const TM tm(p.D);
    int turn = 0;
    VS vs;
    vs.set(vec, tm, W2, p.post.w, 1.f, p.D); vs.set(vec, tm, B2, p.post.b, 0.f, p.D);
    vs.set(vec, tm, W1, p.pre.w, 1.f, p.D); vs.set(vec, tm, B1, p.pre.b, 0.f, p.D);
    if constexpr (VS::SHARED) __syncthreads();
    f32x4 g[NV];
    long long seg_end = 0;
    tm.load_or(nullptr, 1.f, g);
    // consecutive rows stay in a workgroup: the gate row changes rarely
    const long long per = ((p.rows + gridDim.x - 1) / gridDim.x + TM::TEAMS - 1) / TM::TEAMS * TM::TEAMS;
    const long long first = per * blockIdx.x + threadIdx.x / TPR, end = min(per * (blockIdx.x + 1ll), p.rows);
    Raw<TX> rx[NV];                                          // the next row, on its way while this one is worked on
    Raw<T> ry[NV];
    if (first < end) { tm.template load<TX>(p.x, first * p.D, rx); if (p.y) tm.template load<T>(p.y, first * p.D, ry); }
    for (long long row = first; row < end; row += TM::TEAMS) {
        f32x4 v[NV], n[NV];
#pragma unroll
        for (int c = 0; c < NV; ++c) { v[c] = rx[c].f(); n[c] = ry[c].f(); }
        if (p.gate && row >= seg_end) {
            const long long seg = row / p.seg_rows;
            seg_end = (seg + 1) * p.seg_rows;
            tm.load_or(p.gate + seg * p.D, 1.f, g);
        }
        if (row + TM::TEAMS < end) { tm.template load<TX>(p.x, (row + TM::TEAMS) * p.D, rx); if (p.y) tm.template load<T>(p.y, (row + TM::TEAMS) * p.D, ry); }
        float m2 = 0.f, r2 = 0.f, m1 = 0.f, r1 = 0.f;
        if (p.y) {
            if (p.post.kind != DIC_NORM_NONE) {
                moments(tm, n, p.post, p.inv_d, red, turn, m2, r2);
#pragma unroll
                for (int c = 0; c < NV; ++c) {
                    const f32x4 w = vs.get(vec, tm, W2, c), b = vs.get(vec, tm, B2, c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) n[c][e] = (n[c][e] - m2) * r2 * w[e] + b[e];
                }
            }
#pragma unroll
            for (int c = 0; c < NV; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[c][e] = e < tm.cnt[c] ? fmaf(g[c][e], n[c][e], p.r * v[c][e]) : 0.f;
        } else {
#pragma unroll
            for (int c = 0; c < NV; ++c) v[c] = v[c] * p.r;
        }
        if (p.x_new) tm.template store<TX>(p.x_new, row * p.D, v);
        if (p.pre.kind != DIC_NORM_NONE) {
            moments(tm, v, p.pre, p.inv_d, red, turn, m1, r1);
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                const f32x4 w = vs.get(vec, tm, W1, c), b = vs.get(vec, tm, B1, c);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[c][e] = (v[c][e] - m1) * r1 * w[e] + b[e];
            }
            tm.template store<T>(p.a, row * p.D, v);
        }
        if (tm.lane == 0 && p.saved) { p.saved[row] = m2; p.saved[p.rows + row] = r2; p.saved[2 * p.rows + row] = m1; p.saved[3 * p.rows + row] = r1; }
    }
}

// A workgroup walks consecutive pieces (ONE: it has one); its teams take the rows of a piece in turn.  Column sums: d and d u over a piece give that
// piece's share of the gate's gradient (w sum(d u) + b sum(d), folded over the teams through LDS), and, times the gate, of the post norm's weight and bias.
// 17408 rows of 768, fp32 stream, bf16 blocks: 247 MB in 60 us, 4.1 TB/s, and 5 us for the fold; 8200 rows of 2048 in fp32: 403 MB in 93 us, 4.3 TB/s.
// Above 4096 columns a row's operands, column sums and vectors are more than the 128 registers that 16 waves leave each: 17 to 29 are spilled in fp32, 70 to 99
// with bf16 blocks (2052 rows of 8192: 119 us in fp32, 147 in bf16, 150 beside an fp32 stream; a copy's rate would be 84, 42 and 63).
template <typename T, typename TX, int TPR, int NV, bool ONE>
__global__ __launch_bounds__((Team<TPR, NV>::THREADS)) void gated_norm_bwd_kernel(const NormArgs p) {
    using TM = Team<TPR, NV>;
    using VS = Vectors<TPR, NV, 2>;
    __shared__ float red[TPR > 64 ? 4 * TM::WAVES : 1];
    __shared__ __attribute__((aligned(16))) float vec[VS::SHARED ? 2 * TM::WIDTH : 1];
    __shared__ __attribute__((aligned(16))) float fold[TM::TEAMS > 1 ? TM::TEAMS * TM::WIDTH : 1];
    enum { W1, GW2 };                                        // pre's weight; the gate times post's
    const TM tm(p.D);
    const int team = threadIdx.x / TPR;
    int turn = 0;
    VS vs;
    f32x4 sdu[NV], sd[NV], sw2[ONE ? 1 : NV], sb2[ONE ? 1 : NV], sw1[NV], sb1[NV], g[NV];
    const f32x4 zero{0.f, 0.f, 0.f, 0.f};
    vs.set(vec, tm, W1, p.pre.w, 1.f, p.D);
#pragma unroll
    for (int c = 0; c < NV; ++c) { sw1[c] = sb1[c] = zero; if constexpr (!ONE) sw2[c] = sb2[c] = zero; }
    const bool layer1 = p.pre.kind == DIC_NORM_LAYER, layer2 = p.post.kind == DIC_NORM_LAYER, pre = p.pre.kind != DIC_NORM_NONE, post = p.post.kind != DIC_NORM_NONE;
    // sums over the teams, in a fixed order, to out[0 .. D)
    auto fold_teams = [&](float* out, const f32x4 (&v)[NV]) {
        if constexpr (TM::TEAMS == 1) tm.template store<float>(out, 0, v);
        else {
            tm.template store<float>(fold + team * TM::WIDTH, 0, v);
            __syncthreads();
            for (int i = threadIdx.x; i < p.D; i += TM::THREADS) {
                float s = 0.f;
#pragma unroll
                for (int t = 0; t < TM::TEAMS; ++t) s += fold[t * TM::WIDTH + i];
                out[i] = s;
            }
            __syncthreads();
        }
    };
    const long long q0 = ONE ? blockIdx.x : (long long)blockIdx.x * p.pieces_per_block, q1 = ONE ? q0 + 1 : min(q0 + p.pieces_per_block, p.pieces);
    for (long long q = q0; q < q1; ++q) {
        const long long seg = q / p.gate_parts, part = q - seg * p.gate_parts;
        const long long first = seg * p.seg_rows + part * p.piece_rows, end = min(first + p.piece_rows, min((seg + 1) * p.seg_rows, p.rows));
        const float* gate = p.gate ? p.gate + seg * p.D : nullptr;
        if (VS::SHARED && !ONE && q > q0 && p.gate) __syncthreads();                 // the last piece's rows are done with
        if (q == q0 || p.gate) vs.set(vec, tm, GW2, p.post.w, 1.f, p.D, gate);
        Raw<TX> rd[NV], rx[NV];                              // the next row, on its way while this one is worked on
        Raw<T> re[NV], ry[NV];
        auto fetch = [&](long long row) {
            if (p.dx_new) tm.template load<TX>(p.dx_new, row * p.D, rd);
            if (pre) { tm.template load<T>(p.da, row * p.D, re); tm.template load<TX>(p.x_new, row * p.D, rx); }
            if (p.y) tm.template load<T>(p.y, row * p.D, ry);
        };
        constexpr bool AHEAD = TPR < 1024;                   // (16 waves to a row have 128 registers each: no room for the next one)
        if (AHEAD && first + team < end) fetch(first + team);
        if constexpr (VS::SHARED) { if (q == q0 || p.gate) __syncthreads(); }
#pragma unroll
        for (int c = 0; c < NV; ++c) sdu[c] = sd[c] = zero;
        for (long long row = first + team; row < end; row += TM::TEAMS) {
            f32x4 d[NV], e[NV], x[NV], y[NV];
            if (!AHEAD) fetch(row);
#pragma unroll
            for (int c = 0; c < NV; ++c) {
                d[c] = p.dx_new ? rd[c].f() : zero;
                if (pre) { e[c] = re[c].f(); x[c] = rx[c].f(); }
                if (p.y) y[c] = ry[c].f();
            }
            if (AHEAD && row + TM::TEAMS < end) fetch(row + TM::TEAMS);
            if (pre) {
                const float m = p.saved[2 * p.rows + row], rs = p.saved[3 * p.rows + row];
                float c1 = 0.f, c2 = 0.f;
#pragma unroll
                for (int c = 0; c < NV; ++c) {
                    const f32x4 w = vs.get(vec, tm, W1, c);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float u = k < tm.cnt[c] ? (x[c][k] - m) * rs : 0.f;
                        sw1[c][k] += e[c][k] * u;
                        sb1[c][k] += e[c][k];
                        const float f = e[c][k] * w[k];
                        c1 += f; c2 += f * u;
                        x[c][k] = u; e[c][k] = f;
                    }
                }
                tm.sum2(c1, c2, red, turn);
                c1 = layer1 ? c1 * p.inv_d : 0.f;
                c2 *= p.inv_d;
#pragma unroll
                for (int c = 0; c < NV; ++c)
#pragma unroll
                    for (int k = 0; k < 4; ++k) d[c][k] += rs * (e[c][k] - c1 - x[c][k] * c2);
            }
            if (p.dx) {
#pragma unroll
                for (int c = 0; c < NV; ++c) x[c] = d[c] * p.r;
                tm.template store<TX>(p.dx, row * p.D, x);
            }
            if (p.y) {
                const float m = post ? p.saved[row] : 0.f, rs = post ? p.saved[p.rows + row] : 1.f;
                float c1 = 0.f, c2 = 0.f;
#pragma unroll
                for (int c = 0; c < NV; ++c) {
                    const f32x4 w = vs.get(vec, tm, GW2, c);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const bool in = k < tm.cnt[c];
                        const float u = in ? (y[c][k] - m) * rs : 0.f, dd = in ? d[c][k] : 0.f;
                        sdu[c][k] += dd * u;
                        sd[c][k] += dd;
                        const float f = dd * w[k];
                        c1 += f; c2 += f * u;
                        y[c][k] = u; d[c][k] = f;
                    }
                }
                if (post) {
                    tm.sum2(c1, c2, red, turn);
                    c1 = layer2 ? c1 * p.inv_d : 0.f;
                    c2 *= p.inv_d;
#pragma unroll
                    for (int c = 0; c < NV; ++c)
#pragma unroll
                        for (int k = 0; k < 4; ++k) d[c][k] = rs * (d[c][k] - c1 - y[c][k] * c2);
                }
                if (p.dy) tm.template store<T>(p.dy, row * p.D, d);
            }
        }
        tm.load_or(gate, 1.f, g);
        if constexpr (!ONE) {
#pragma unroll
            for (int c = 0; c < NV; ++c) { sw2[c] += sdu[c] * g[c]; sb2[c] += sd[c] * g[c]; }
        }
        if (p.dgate) {
            f32x4 w2[NV], b2[NV], share[NV];
            tm.load_or(p.post.w, 1.f, w2); tm.load_or(p.post.b, 0.f, b2);
#pragma unroll
            for (int c = 0; c < NV; ++c) share[c] = sdu[c] * w2[c] + sd[c] * b2[c];
            fold_teams(p.dgate + q * p.D, share);
        }
    }
    if (!p.cols) return;
    float* out = p.cols + (long long)blockIdx.x * 4 * p.D;
    if constexpr (ONE) {
#pragma unroll
        for (int c = 0; c < NV; ++c) { sdu[c] = sdu[c] * g[c]; sd[c] = sd[c] * g[c]; }
        fold_teams(out, sdu); fold_teams(out + p.D, sd);
    } else { fold_teams(out, sw2); fold_teams(out + p.D, sb2); }
    fold_teams(out + 2 * p.D, sw1); fold_teams(out + 3 * p.D, sb1);
}

// out[c] = sum over k < n of in[k * ld + c]: 32 columns by 32 interleaved groups of rows per workgroup, the groups added in a fixed order
struct Fold { const float* in; float* out; long long n, ld; };
struct Folds { Fold f[4]; Fold gate; long long gate_in, gate_rows; int D; };
__global__ __launch_bounds__(1024) void fold_kernel(const Folds p) {
    __shared__ float part[32][33];
    Fold f;
    if (blockIdx.y < 4) { f = p.f[blockIdx.y]; if (!f.out) return; }
    else { f = p.gate; const long long s = blockIdx.y - 4; f.in += s * p.gate_in; f.out += s * p.D; }
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), grp = threadIdx.x >> 5;
    float s = 0.f;
    if (c < p.D)
#pragma unroll 4
        for (long long k = grp; k < f.n; k += 32) s += f.in[k * f.ld + c];
    part[grp][threadIdx.x & 31] = s;
    __syncthreads();
    if (threadIdx.x < 32 && c < p.D) {
        s = 0.f;
#pragma unroll
        for (int k = 0; k < 32; ++k) s += part[k][threadIdx.x];
        f.out[c] = s;
    }
}

// ------------------------------------------------------------------------------------------------ host side
// Teams are as small as keeps a row in at most 16 registers per operand and thread: a row inside one wave needs no barrier (135168 bf16 rows of 768, forward:
// 64 threads 183 us, 256 threads 290; the 66 rows of one caption 6.2 and 4.7), and beyond 16 the registers leave too few rows in flight (8200 rows of 2048 in
// fp32, backward: 64 threads 157 us, 256 threads 92).
template <typename F> int by_width(int D, F&& f) {
    if (D <= 64) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    if (D <= 128) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 2>());
    if (D <= 256) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    if (D <= 512) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    if (D <= 768) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 3>());
    if (D <= 1024) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
    if (D <= 2048) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
    if (D <= 4096) return f(std::integral_constant<int, 512>(), std::integral_constant<int, 2>());
    return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
}
int teams_of(int D) { return D <= 128 ? 16 : D <= 1024 ? 4 : 1; }

// How the backward pass cuts the rows: pieces inside one gate segment, and few workgroups where rows are wide, as each leaves 4 D partial sums behind that the
// fold reads again (1024 / 512 / 256 of them: 3000 x 17 rows of 64 25 / 33 / 49 us; 8200 of 1024 57 / 48 / 56; 8200 of 2048 in fp32 102 / 100 / 102; 4000 of
// 4096 70 / 57 / 52; 2052 of 8192 in fp32 150 / 135 / 119).
struct Plan { long long segs, seg_rows, parts, piece_rows, pieces, per_block, blocks; };
Plan plan_of(const DicGatedNormParams* p) {
    Plan l;
    const long long BLOCKS = p->D <= 512 ? 1024 : p->D <= 2048 ? 512 : 256;
    l.seg_rows = p->gate ? p->rows_per_gate : p->rows;
    l.segs = p->rows / l.seg_rows;
    const long long want = (p->rows + BLOCKS - 1) / BLOCKS, least = teams_of(p->D);           // rows of a piece: at least one for each team
    const long long rows = want > least ? want : least;
    l.parts = (l.seg_rows + rows - 1) / rows;
    l.piece_rows = (l.seg_rows + l.parts - 1) / l.parts;
    l.parts = (l.seg_rows + l.piece_rows - 1) / l.piece_rows;
    l.pieces = l.segs * l.parts;
    l.per_block = (l.pieces + BLOCKS - 1) / BLOCKS;
    l.blocks = (l.pieces + l.per_block - 1) / l.per_block;
    return l;
}
size_t ws_floats(const DicGatedNormParams* p, const Plan& l) {
    return (size_t)l.blocks * 4 * p->D + (p->gate && l.parts > 1 ? (size_t)l.pieces * p->D : 0);
}

bool norm_ok(const DicNorm& n) {
    return (n.kind == DIC_NORM_NONE && !n.weight && !n.bias) || ((n.kind == DIC_NORM_LAYER || n.kind == DIC_NORM_RMS) && n.eps >= 0.f && std::isfinite(n.eps));
}
int check(int dtype, const DicGatedNormParams* p) {
    DIC_REQUIRE(p != nullptr, "dic_gated_norm: no parameters");
    DIC_REQUIRE(dtype == DIC_F32 || dtype == DIC_BF16 || dtype == (DIC_BF16 | DIC_RES_F32), "dic_gated_norm: dtype must be DIC_F32, DIC_BF16 or DIC_BF16 | DIC_RES_F32");
    DIC_REQUIRE(p->D >= 1 && p->D <= 8192, "dic_gated_norm: rows of 1 to 8192 elements");
    DIC_REQUIRE(p->rows >= 0 && p->rows < (1ll << 40), "dic_gated_norm: rows out of range");
    DIC_REQUIRE(norm_ok(p->post) && norm_ok(p->pre), "dic_gated_norm: a norm is DIC_NORM_NONE (without weight and bias), DIC_NORM_LAYER or DIC_NORM_RMS, with a finite eps >= 0");
    DIC_REQUIRE(!p->gate || (p->rows_per_gate >= 1 && p->rows % p->rows_per_gate == 0), "dic_gated_norm: rows must be a multiple of rows_per_gate");
    DIC_REQUIRE(std::isfinite(p->residual_scale), "dic_gated_norm: the residual scale must be finite");
    return 0;
}
NormArgs args_of(const DicGatedNormParams* p) {
    NormArgs a{};
    a.x = p->x; a.y = p->y; a.dx_new = p->dx_new; a.da = p->da; a.x_new = p->x_new; a.a = p->a; a.dx = p->dx; a.dy = p->dy;
    a.gate = p->gate; a.saved = p->saved;
    a.post = Norm{p->post.weight, p->post.bias, p->post.kind, p->post.eps};
    a.pre = Norm{p->pre.weight, p->pre.bias, p->pre.kind, p->pre.eps};
    a.rows = p->rows; a.seg_rows = p->gate ? p->rows_per_gate : p->rows;
    a.D = p->D; a.r = p->residual_scale; a.inv_d = 1.0f / (float)p->D;
    return a;
}
template <typename T, typename TX> int fwd(const NormArgs& a, hipStream_t st) {
    return by_width(a.D, [&](auto tpr, auto nv) -> int {
        using TM = Team<decltype(tpr)::value, decltype(nv)::value>;
        const long long teams = (a.rows + TM::TEAMS - 1) / TM::TEAMS, most = 256 * 2048 / TM::THREADS;
        hipLaunchKernelGGL((gated_norm_fwd_kernel<T, TX, decltype(tpr)::value, decltype(nv)::value>), dim3((unsigned)(teams < most ? teams : most)), dim3(TM::THREADS), 0, st, a);
        DIC_CHECK_LAUNCH();
        return 0;
    });
}
template <typename T, typename TX> int bwd(const NormArgs& a, long long blocks, hipStream_t st) {
    return by_width(a.D, [&](auto tpr, auto nv) -> int {
        using TM = Team<decltype(tpr)::value, decltype(nv)::value>;
        if (a.pieces_per_block == 1) hipLaunchKernelGGL((gated_norm_bwd_kernel<T, TX, decltype(tpr)::value, decltype(nv)::value, true>), dim3((unsigned)blocks), dim3(TM::THREADS), 0, st, a);
        else hipLaunchKernelGGL((gated_norm_bwd_kernel<T, TX, decltype(tpr)::value, decltype(nv)::value, false>), dim3((unsigned)blocks), dim3(TM::THREADS), 0, st, a);
        DIC_CHECK_LAUNCH();
        return 0;
    });
}
}  // namespace

extern "C" size_t dic_gated_norm_ws_bytes(int dtype, const DicGatedNormParams* p) {
    if (check(dtype, p) || p->rows == 0) return 0;
    return ws_floats(p, plan_of(p)) * sizeof(float);
}

extern "C" int dic_gated_norm_fwd(int dtype, const DicGatedNormParams* p, void* stream) {
    if (int rc = check(dtype, p)) return rc;
    const bool pre = p->pre.kind != DIC_NORM_NONE;
    if (p->rows == 0) return 0;
    DIC_REQUIRE(p->y || (!p->gate && p->post.kind == DIC_NORM_NONE && pre), "dic_gated_norm_fwd: without y there is a pre norm and nothing else");
    DIC_REQUIRE(p->x && (p->x_new || !p->y) && (p->a || !pre), "dic_gated_norm_fwd: null pointer");
    const NormArgs a = args_of(p);
    hipStream_t st = (hipStream_t)stream;
    return dtype == DIC_F32 ? fwd<float, float>(a, st) : dtype == DIC_BF16 ? fwd<bf16_t, bf16_t>(a, st) : fwd<bf16_t, float>(a, st);
}

extern "C" int dic_gated_norm_bwd(int dtype, const DicGatedNormParams* p, void* stream) {
    if (int rc = check(dtype, p)) return rc;
    const bool pre = p->pre.kind != DIC_NORM_NONE, post = p->post.kind != DIC_NORM_NONE;
    DIC_REQUIRE(p->y || p->rows == 0 || (!p->gate && !post && pre && !p->dy), "dic_gated_norm_bwd: without y there is a pre norm and nothing else");
    DIC_REQUIRE((!p->dgate || p->gate) && (post || (!p->dpost_w && !p->dpost_b)) && (pre || (!p->dpre_w && !p->dpre_b)), "dic_gated_norm_bwd: a gradient of something that is not there");
    DIC_REQUIRE(p->D >= 1 && (p->rows == 0 || ((pre ? p->da && p->x_new : p->dx_new != nullptr) && p->dx && (p->dy || !p->y) && (p->saved || (!pre && !post)))), "dic_gated_norm_bwd: null pointer");
    hipStream_t st = (hipStream_t)stream;
    NormArgs a = args_of(p);
    Folds f{};
    f.D = p->D;
    float* outs[4] = {p->dpost_w, p->dpost_b, p->dpre_w, p->dpre_b};
    const bool cols = outs[0] || outs[1] || outs[2] || outs[3];
    Plan l{};
    if (p->rows > 0) {
        l = plan_of(p);
        const size_t need = ws_floats(p, l) * sizeof(float);
        DIC_REQUIRE(p->ws && ((uintptr_t)p->ws & 15) == 0 && p->ws_bytes >= need, "dic_gated_norm_bwd: workspace missing or too small (dic_gated_norm_ws_bytes)");
        float* ws = (float*)p->ws;
        a.seg_rows = l.seg_rows; a.pieces = l.pieces; a.piece_rows = l.piece_rows; a.gate_parts = (int)l.parts; a.pieces_per_block = (int)l.per_block;
        a.cols = cols ? ws : nullptr;
        a.dgate = p->dgate && l.parts > 1 ? ws + (size_t)l.blocks * 4 * p->D : p->dgate;
        const int rc = dtype == DIC_F32 ? bwd<float, float>(a, l.blocks, st) : dtype == DIC_BF16 ? bwd<bf16_t, bf16_t>(a, l.blocks, st) : bwd<bf16_t, float>(a, l.blocks, st);
        if (rc) return rc;
        for (int k = 0; k < 4; ++k) f.f[k] = Fold{ws + (size_t)k * p->D, outs[k], l.blocks, 4ll * p->D};
        if (p->dgate && l.parts > 1) { f.gate = Fold{a.dgate, p->dgate, l.parts, p->D}; f.gate_in = l.parts * p->D; f.gate_rows = l.segs; }
    } else {
        for (int k = 0; k < 4; ++k) f.f[k] = Fold{nullptr, outs[k], 0, 0};       // no rows: the sums are zero
    }
    if (cols || f.gate_rows) {
        hipLaunchKernelGGL(fold_kernel, dim3((p->D + 31) / 32, (unsigned)(4 + f.gate_rows)), dim3(1024), 0, st, f);
        DIC_CHECK_LAUNCH();
    }
    return 0;
}
