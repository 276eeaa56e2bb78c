// Attention over long token rows: a sliding window per query, the first `sinks` keys visible behind it, any number of query heads per key head.
//   s_ij = scale q_i . k_j over the visible j,  lse_i = log sum_j exp s_ij,  p_ij = exp(s_ij - lse_i),  out_i = sum_j p_ij v_j
//   delta_i = dout_i . out_i,  ds_ij = p_ij (dout_i . v_j - delta_i) scale,  dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
// Every product runs on 32x32 MFMA tiles with the score tile TRANSPOSED or not so that the dimension that is reduced next lies in a lane's registers:
// the forward and the dq kernel hold S^T (lane = query, registers = keys), the dk / dv kernel holds S (lane = key, registers = queries).  A lane's 16
// values are then the B operand of the next product as they are -- no LDS round trip for P or dS -- if that product's A operand is read token-major
// from LDS in the same token order, which ds_read_b64_tr_b16 (bf16) or plain 4-byte reads (fp32) give.
// Tiles come in by LDS-DMA, double-buffered; rows of keys that nobody may see (key_mask, kv_len) are zero-filled by the descriptor's bounds check, so
// that an infinity or NaN in them cannot reach 0 * v.
#include <cmath>
#include "common.h"
#include "../../include/dic_hip.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int FAR = (1 << 30) - 2;              // positions and bounds are clamped to +-FAR: sums of two stay inside 32 bits

struct Strides { long long n, t, h; };
struct WinArgs {
    const void *q, *k, *v, *o, *dout;
    void *out, *dq, *dk, *dv;
    float* lse;                                 // forward: written [N][H][Tq]; backward: read
    float* stats;                               // backward workspace: for every 32 queries of (n, h) 32 x lse * log2(e), then 32 x dout . out
    Strides sq, sk, sv, so, sdo, sdq, sdk, sdv; // elements
    const uint8_t* key_mask;
    const int* kv_len;
    const int* q_pos;
    int N, Tq, Tk, H, Hkv, G, left, right, sinks;
    float scale, c;                             // c = scale * log2(e)
};

__device__ __forceinline__ int tok(int r, int hi) { return (r & 3) + 8 * (r >> 2) + 4 * hi; }     // row of register r of a 32x32 accumulator
__device__ __forceinline__ f32x16 zero16() { f32x16 z; for (int i = 0; i < 16; ++i) z[i] = 0.f; return z; }

// An LDS tile holds token rows of DH elements as 16-byte chunks, chunk c of row r at slot c ^ swz(r).  The order makes both readings free of bank
// conflicts: 16 consecutive rows at one chunk index (row operands, ds_read_b128), and 64 bytes of each of 4 consecutive rows (transposing reads).
template <typename T, int DH> struct Lay {
    static constexpr int ROWB = DH * (int)sizeof(T), CH = ROWB / 16, NF = ROWB / 32, ND = DH / 32, PIECE_ROWS = 1024 / ROWB;
    __device__ static __forceinline__ int swz(int row) { return CH == 8 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 3) : ((row & 3) << 2) | ((row >> 2) & 3); }
};

// Row operand of a 32-token block: lane holds row (lane & 31), bytes 32 s + 16 (lane >> 5).
template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
    typedef bf16x8 Frag;
    __device__ static __forceinline__ f32x16 mac(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    // acc[d][col] += sum over 32 tokens of tile[token][32 db + d] * p[token][col], p in accumulator order
    template <int DH> __device__ static __forceinline__ f32x16 mac_t(const char* tile, int row0, int db, const f32x16& p, f32x16 acc, int lane) {
        using L = Lay<bf16_t, DH>;
        const int hi = lane >> 5, half = (lane >> 4) & 1, t = lane & 15;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int r0 = row0 + 16 * s + 4 * hi + (t >> 2), c = db * 4 + half * 2 + ((t & 3) >> 1), sub = (t & 1) * 8;
            s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(tile + r0 * L::ROWB + ((c ^ L::swz(r0)) << 4) + sub));
            s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(tile + (r0 + 8) * L::ROWB + ((c ^ L::swz(r0 + 8)) << 4) + sub));
            s16x8 a = __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7);
            i32x4 b;
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = (int)pack2bf(p[8 * s + 2 * e], p[8 * s + 2 * e + 1]);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
        }
        return acc;
    }
    __device__ static __forceinline__ float dot(Frag a, Frag b) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf((float)a[e], (float)b[e], s);
        return s;
    }
    __device__ static __forceinline__ void st4(bf16_t* p, float a, float b, float c, float d) { *(uint2*)p = make_uint2(pack2bf(a, b), pack2bf(c, d)); }
};
template <> struct Mma<float> {
    typedef f32x4 Frag;
    __device__ static __forceinline__ f32x16 mac(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    template <int DH> __device__ static __forceinline__ f32x16 mac_t(const char* tile, int row0, int db, const f32x16& p, f32x16 acc, int lane) {
        using L = Lay<float, DH>;
        const int hi = lane >> 5, d = lane & 31;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int row = row0 + tok(r, hi);
            const float a = *(const float*)(tile + row * L::ROWB + (((db * 8 + (d >> 2)) ^ L::swz(row)) << 4) + (d & 3) * 4);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc, 0, 0, 0);
        }
        return acc;
    }
    __device__ static __forceinline__ float dot(Frag a, Frag b) { return (a[0] * b[0] + a[1] * b[1]) + (a[2] * b[2] + a[3] * b[3]); }
    __device__ static __forceinline__ void st4(float* p, float a, float b, float c, float d) { *(f32x4*)p = f32x4{a, b, c, d}; }
};

// ---- LDS-DMA.  The base of a descriptor is the tile's first row (64-bit arithmetic per tile, 32-bit offsets inside it); a lane whose row is not
// to be read passes an offset beyond num_records and gets zeros.
__device__ __forceinline__ i32x4 tile_rsrc(const void* base) {
    const unsigned long long b = (unsigned long long)base;
    i32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)b);
    r[1] = __builtin_amdgcn_readfirstlane((int)((b >> 32) & 0xffffu));
    r[2] = 0x7fffffff;
    r[3] = 0x00020000;
    return r;
}
__device__ __forceinline__ void dma16(unsigned voff, const i32x4& rsrc, unsigned lds_addr) {           // 64 lanes x 16 B -> 1 KiB at lds_addr
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(lds_addr)) : "memory");
}
__device__ __forceinline__ void dma4(unsigned voff, const i32x4& rsrc, unsigned lds_addr) {            // 64 lanes x 4 B
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(lds_addr)) : "memory");
}
// this wave's DMA has landed and, behind the barrier, everybody's has; everybody is done with the buffer that is refilled next
__device__ __forceinline__ void dma_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ROWS token rows from `base` (row stride st bytes) into a tile; bit r of `valid`: row r is read, else zero.  NW waves share the pieces.
template <typename T, int DH, int ROWS, int NW>
__device__ __forceinline__ void load_tile(const char* base, unsigned st, unsigned long long valid, unsigned lds, int wave, int lane) {
    using L = Lay<T, DH>;
    const i32x4 rs = tile_rsrc(base);
    constexpr int P = ROWS / L::PIECE_ROWS;
    static_assert(ROWS % L::PIECE_ROWS == 0 && P % NW == 0, "pieces divide over the waves");
#pragma unroll
    for (int j = 0; j < P / NW; ++j) {
        const int piece = j * NW + wave, row = piece * L::PIECE_ROWS + lane / L::CH, c = (lane % L::CH) ^ L::swz(row);
        const unsigned off = ((valid >> row) & 1ull) ? (unsigned)row * st + (unsigned)c * 16u : 0xfffffff0u;
        dma16(off, rs, lds + (unsigned)piece * 1024u);
    }
}
template <typename T, int DH>
__device__ __forceinline__ typename Mma<T>::Frag row_frag(const char* tile, int row, int s, int hi) {
    using L = Lay<T, DH>;
    return *(const typename Mma<T>::Frag*)(tile + row * L::ROWB + (((2 * s + hi) ^ L::swz(row)) << 4));
}

__device__ __forceinline__ unsigned long long below(int x) { return x <= 0 ? 0ull : x >= 64 ? ~0ull : (1ull << x) - 1ull; }
__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// The keys of one sequence that exist, and the position of its first query.
struct Seq { int kvl, pos; };
__device__ __forceinline__ Seq sequence(const WinArgs& a, int n) {
    Seq s;
    s.kvl = a.kv_len ? clampi(a.kv_len[n], 0, a.Tk) : a.Tk;
    s.pos = a.q_pos ? clampi(a.q_pos[n], -FAR / 2, FAR / 2) : 0;
    return s;
}
// Query at position t sees the keys [lo, hi) and [0, sk).
struct Span { int lo, hi, sk; };
__device__ __forceinline__ Span span_of(const WinArgs& a, int t, int kvl) {
    Span s;
    s.lo = a.left < 0 ? 0 : max(0, t - a.left);
    s.hi = a.right < 0 ? kvl : clampi(t + a.right + 1, 0, kvl);
    s.sk = a.left < 0 ? 0 : min(a.sinks, s.hi);
    return s;
}
__device__ __forceinline__ unsigned long long visible(const Span& s, int j0) { return (below(s.hi - j0) & ~below(s.lo - j0)) | below(s.sk - j0); }

// The key tiles that the queries at positions t0..t1 need: those of the sinks, then those of the windows.
struct Walk {
    int ns, w0, nt, kvl;
    __device__ __forceinline__ int j0(int t, int bn) const { return (t < ns ? t : w0 + t - ns) * bn; }
};
__device__ __forceinline__ Walk walk_of(const WinArgs& a, int t0, int t1, int kvl, int bn) {
    Walk w;
    const int lo = span_of(a, t0, kvl).lo;
    const Span e = span_of(a, t1, kvl);
    w.kvl = kvl;
    w.ns = (e.sk + bn - 1) / bn;
    w.w0 = max(lo / bn, w.ns);
    w.nt = w.ns + max(0, (e.hi + bn - 1) / bn - w.w0);
    return w;
}
// consecutive work items on one XCD (workgroups are dealt to the 8 XCDs in turn), so that neighbours share their keys in its L2
__device__ __forceinline__ int xcd_item() {
    const int g = gridDim.x, b = blockIdx.x, q = g >> 3, r = g & 7, x = b & 7;
    return x * q + min(x, r) + (b >> 3);
}
// key_mask bits of a tile: lane reads its key's byte (called one tile ahead), the ballot is the tile's mask
__device__ __forceinline__ int mask_byte(const WinArgs& a, int n, int j) { return a.key_mask && j >= 0 && j < a.Tk ? a.key_mask[(size_t)n * a.Tk + j] : 1; }

constexpr int BM = 128, NWAVE = 4;              // queries (or keys) per workgroup: 32 per wave
constexpr int BQ = 32;                          // queries per tile of the dk / dv kernel
__host__ __device__ __forceinline__ long long stats_floats(long long N, long long H, long long Tq) { return N * H * ((Tq + BQ - 1) / BQ) * 2 * BQ; }
__device__ __forceinline__ long long stats_at(const WinArgs& a, int n, int h, int i0) { return stats_floats(1, (long long)n * a.H + h, a.Tq) + 2 * i0; }

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int DH, int BN>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void win_fwd_kernel(const WinArgs a) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    constexpr int NB = BN / 32, TILE = BN * L::ROWB;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hi = lane >> 5;
    const int nqt = (a.Tq + BM - 1) / BM;
    int item = xcd_item();
    const int g = item % a.G; item /= a.G;
    const int qt = nqt - 1 - item % nqt; item /= nqt;         // long rows first
    const int hk = item % a.Hkv, n = item / a.Hkv, h = hk * a.G + g;
    const Seq sq = sequence(a, n);
    const int i0 = qt * BM + wave * 32, i = i0 + (lane & 31), ic = min(i, a.Tq - 1);
    const Walk wk = walk_of(a, sq.pos + qt * BM, sq.pos + min(qt * BM + BM, a.Tq) - 1, sq.kvl, BN);
    const Span sp = span_of(a, sq.pos + ic, sq.kvl);
    const bool wave_rows = i0 < a.Tq;
    // what every row of this wave sees: [in_lo, in_hi)
    const int in_lo = span_of(a, sq.pos + min(i0 + 31, a.Tq - 1), sq.kvl).lo, in_hi = span_of(a, sq.pos + min(i0, a.Tq - 1), sq.kvl).hi;

    typename M::Frag qf[L::NF];
    {
        const char* p = (const char*)((const T*)a.q + n * a.sq.n + ic * a.sq.t + h * a.sq.h);
#pragma unroll
        for (int s = 0; s < L::NF; ++s) qf[s] = *(const typename M::Frag*)(p + 32 * s + 16 * hi);
    }
    const char* kb = (const char*)((const T*)a.k + n * a.sk.n + hk * a.sk.h);
    const char* vb = (const char*)((const T*)a.v + n * a.sv.n + hk * a.sv.h);
    const long long kst = a.sk.t * (long long)sizeof(T), vst = a.sv.t * (long long)sizeof(T);
    const unsigned lds = (unsigned)(uintptr_t)(LDS_PTR(char))smem;
    auto issue = [&](int j0, unsigned long long valid, int buf) {
        load_tile<T, DH, BN, NWAVE>(kb + j0 * kst, (unsigned)kst, valid, lds + buf * 2 * TILE, wave, lane);
        load_tile<T, DH, BN, NWAVE>(vb + j0 * vst, (unsigned)vst, valid, lds + buf * 2 * TILE + TILE, wave, lane);
    };
    auto valid_of = [&](int byte, int j0) { return __ballot(byte != 0) & below(min(BN, wk.kvl - j0)); };

    f32x16 acc[L::ND];
#pragma unroll
    for (int d = 0; d < L::ND; ++d) acc[d] = zero16();
    float m = -INFINITY, l = 0.f;
    unsigned long long valid = 0, valid_next = 0;
    int byte = 1;                                             // key_mask of this lane's key in the tile after the next
    if (wk.nt > 0) {
        valid = valid_of(mask_byte(a, n, wk.j0(0, BN) + lane), wk.j0(0, BN));
        issue(wk.j0(0, BN), valid, 0);
        if (wk.nt > 1) byte = mask_byte(a, n, wk.j0(1, BN) + lane);
    }
    for (int t = 0; t < wk.nt; ++t) {
        const int j0 = wk.j0(t, BN);
        if (t + 1 < wk.nt) {
            valid_next = valid_of(byte, wk.j0(t + 1, BN));
            if (t + 2 < wk.nt) byte = mask_byte(a, n, wk.j0(t + 2, BN) + lane);
        }
        dma_barrier();
        if (t + 1 < wk.nt) issue(wk.j0(t + 1, BN), valid_next, (t + 1) & 1);
        const char* kt = smem + (t & 1) * 2 * TILE;
        const char* vt = kt + TILE;
        unsigned long long bits = ~0ull;
        const bool full = j0 >= in_lo && j0 + BN <= in_hi && valid == below(BN);
        if (!full) bits = visible(sp, j0) & valid;
        if (wave_rows && (full || __any(bits != 0))) {
            f32x16 st[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                st[b] = zero16();
#pragma unroll
                for (int s = 0; s < L::NF; ++s) st[b] = M::mac(row_frag<T, DH>(kt, 32 * b + (lane & 31), s, hi), qf[s], st[b]);
            }
            if (!full) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const unsigned w = (unsigned)(bits >> (32 * b)) >> (4 * hi);
#pragma unroll
                    for (int r = 0; r < 16; ++r) st[b][r] = (w >> tok(r, 0)) & 1u ? st[b][r] : -INFINITY;
                }
            }
            float mt = st[0][0];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) mt = fmaxf(mt, st[b][r]);
            mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * a.c;
            // The reference point m of the exponentials follows the running maximum only when that is more than 2^8 above it: the sums are in
            // 32 bits and P's relative rounding does not depend on its size, and most tiles then leave the accumulators as they are.
            if (__any(mt > m + 8.f)) {
                const float mn = fmaxf(m, mt), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
                m = mn;
                l *= f;
#pragma unroll
                for (int d = 0; d < L::ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[d][r] *= f;
            }
            const float mm = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) { st[b][r] = __builtin_amdgcn_exp2f(fmaf(st[b][r], a.c, -mm)); l += st[b][r]; }
#pragma unroll
                for (int d = 0; d < L::ND; ++d) acc[d] = M::template mac_t<DH>(vt, 32 * b, d, st[b], acc[d], lane);
            }
        }
        valid = valid_next;
    }
    l += __shfl_xor(l, 32, 64);
    if (i < a.Tq) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* o = (T*)a.out + n * a.so.n + i * a.so.t + h * a.so.h;
#pragma unroll
        for (int d = 0; d < L::ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) M::st4(o + 32 * d + tok(r, hi), acc[d][r] * inv, acc[d][r + 1] * inv, acc[d][r + 2] * inv, acc[d][r + 3] * inv);
        if (a.lse && hi == 0) a.lse[((long long)n * a.H + h) * a.Tq + i] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * LN2;
    }
}

// ------------------------------------------------------------------------------------------------ backward: dq (and delta)
template <typename T, int DH, int BN>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void win_bwd_dq_kernel(const WinArgs a) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    constexpr int NB = BN / 32, TILE = BN * L::ROWB;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hi = lane >> 5;
    const int nqt = (a.Tq + BM - 1) / BM;
    int item = xcd_item();
    const int g = item % a.G; item /= a.G;
    const int qt = nqt - 1 - item % nqt; item /= nqt;
    const int hk = item % a.Hkv, n = item / a.Hkv, h = hk * a.G + g;
    const Seq sq = sequence(a, n);
    const int i0 = qt * BM + wave * 32, i = i0 + (lane & 31), ic = min(i, a.Tq - 1);
    const Walk wk = walk_of(a, sq.pos + qt * BM, sq.pos + min(qt * BM + BM, a.Tq) - 1, sq.kvl, BN);
    const Span sp = span_of(a, sq.pos + ic, sq.kvl);
    const bool wave_rows = i0 < a.Tq;
    const int in_lo = span_of(a, sq.pos + min(i0 + 31, a.Tq - 1), sq.kvl).lo, in_hi = span_of(a, sq.pos + min(i0, a.Tq - 1), sq.kvl).hi;

    typename M::Frag qf[L::NF], df[L::NF];
    float delta = 0.f;
    {
        const char* p = (const char*)((const T*)a.q + n * a.sq.n + ic * a.sq.t + h * a.sq.h);
        const char* pd = (const char*)((const T*)a.dout + n * a.sdo.n + ic * a.sdo.t + h * a.sdo.h);
        const char* po = (const char*)((const T*)a.o + n * a.so.n + ic * a.so.t + h * a.so.h);
#pragma unroll
        for (int s = 0; s < L::NF; ++s) {
            qf[s] = *(const typename M::Frag*)(p + 32 * s + 16 * hi);
            df[s] = *(const typename M::Frag*)(pd + 32 * s + 16 * hi);
            delta += M::dot(df[s], *(const typename M::Frag*)(po + 32 * s + 16 * hi));
        }
        delta += __shfl_xor(delta, 32, 64);
    }
    const float l2 = a.lse[((long long)n * a.H + h) * a.Tq + ic] * LOG2E;
    if (i < a.Tq) a.stats[stats_at(a, n, h, i0) + lane] = hi ? delta : l2;

    const char* kb = (const char*)((const T*)a.k + n * a.sk.n + hk * a.sk.h);
    const char* vb = (const char*)((const T*)a.v + n * a.sv.n + hk * a.sv.h);
    const long long kst = a.sk.t * (long long)sizeof(T), vst = a.sv.t * (long long)sizeof(T);
    const unsigned lds = (unsigned)(uintptr_t)(LDS_PTR(char))smem;
    auto issue = [&](int j0, unsigned long long valid, int buf) {
        load_tile<T, DH, BN, NWAVE>(kb + j0 * kst, (unsigned)kst, valid, lds + buf * 2 * TILE, wave, lane);
        load_tile<T, DH, BN, NWAVE>(vb + j0 * vst, (unsigned)vst, valid, lds + buf * 2 * TILE + TILE, wave, lane);
    };
    auto valid_of = [&](int byte, int j0) { return __ballot(byte != 0) & below(min(BN, wk.kvl - j0)); };
    f32x16 acc[L::ND];
#pragma unroll
    for (int d = 0; d < L::ND; ++d) acc[d] = zero16();
    unsigned long long valid = 0, valid_next = 0;
    int byte = 1;
    if (wk.nt > 0) {
        valid = valid_of(mask_byte(a, n, wk.j0(0, BN) + lane), wk.j0(0, BN));
        issue(wk.j0(0, BN), valid, 0);
        if (wk.nt > 1) byte = mask_byte(a, n, wk.j0(1, BN) + lane);
    }
    for (int t = 0; t < wk.nt; ++t) {
        const int j0 = wk.j0(t, BN);
        if (t + 1 < wk.nt) {
            valid_next = valid_of(byte, wk.j0(t + 1, BN));
            if (t + 2 < wk.nt) byte = mask_byte(a, n, wk.j0(t + 2, BN) + lane);
        }
        dma_barrier();
        if (t + 1 < wk.nt) issue(wk.j0(t + 1, BN), valid_next, (t + 1) & 1);
        const char* kt = smem + (t & 1) * 2 * TILE;
        const char* vt = kt + TILE;
        unsigned long long bits = ~0ull;
        const bool full = j0 >= in_lo && j0 + BN <= in_hi && valid == below(BN);
        if (!full) bits = visible(sp, j0) & valid;
        if (wave_rows && (full || __any(bits != 0))) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                f32x16 st = zero16(), dp = zero16();
#pragma unroll
                for (int s = 0; s < L::NF; ++s) {
                    st = M::mac(row_frag<T, DH>(kt, 32 * b + (lane & 31), s, hi), qf[s], st);
                    dp = M::mac(row_frag<T, DH>(vt, 32 * b + (lane & 31), s, hi), df[s], dp);
                }
                const unsigned w = (unsigned)(bits >> (32 * b)) >> (4 * hi);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(st[r], a.c, -l2)) * (dp[r] - delta);
                    st[r] = full || ((w >> tok(r, 0)) & 1u) ? p : 0.f;
                }
#pragma unroll
                for (int d = 0; d < L::ND; ++d) acc[d] = M::template mac_t<DH>(kt, 32 * b, d, st, acc[d], lane);
            }
        }
        valid = valid_next;
    }
    if (i < a.Tq) {
        T* o = (T*)a.dq + n * a.sdq.n + i * a.sdq.t + h * a.sdq.h;
#pragma unroll
        for (int d = 0; d < L::ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                M::st4(o + 32 * d + tok(r, hi), acc[d][r] * a.scale, acc[d][r + 1] * a.scale, acc[d][r + 2] * a.scale, acc[d][r + 3] * a.scale);
    }
}

// ------------------------------------------------------------------------------------------------ backward: dk, dv
template <typename T, int DH>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void win_bwd_dkv_kernel(const WinArgs a) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    constexpr int TILE = BQ * L::ROWB, STAGE = 2 * TILE + 256;        // Q, dout, {lse2, delta} of 32 queries
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hi = lane >> 5;
    const int nkt = (a.Tk + BM - 1) / BM;
    int item = xcd_item();
    const int kt = item % nkt; item /= nkt;                           // the tile with the sinks first: every query sees it
    const int hk = item % a.Hkv, n = item / a.Hkv;
    const Seq sq = sequence(a, n);
    const int jb = kt * BM, j = jb + wave * 32 + (lane & 31), jc = min(j, a.Tk - 1);
    const bool seen = j < sq.kvl && (!a.key_mask || a.key_mask[(size_t)n * a.Tk + jc]);
    // rows of queries that see key jj: [lo, hi)
    auto first_row = [&](int jj) { return a.right < 0 ? 0 : clampi(jj - a.right - sq.pos, 0, a.Tq); };
    auto end_row = [&](int jj) { return a.left < 0 || jj < a.sinks ? a.Tq : clampi(jj + a.left - sq.pos + 1, 0, a.Tq); };
    const int lo = seen ? first_row(j) : 0, end = seen ? end_row(j) : 0;
    const int last = min(jb + BM, sq.kvl) - 1;                        // last key of the tile that exists
    int r0 = 0, r1 = 0;
    if (last >= jb) { r0 = first_row(jb) & ~(BQ - 1); r1 = jb < a.sinks ? a.Tq : end_row(last); }
    const int nq = r1 > r0 ? (r1 - r0 + BQ - 1) / BQ : 0, nt = nq * a.G;

    typename M::Frag kf[L::NF], vf[L::NF];
    {
        const char* pk = (const char*)((const T*)a.k + n * a.sk.n + jc * a.sk.t + hk * a.sk.h);
        const char* pv = (const char*)((const T*)a.v + n * a.sv.n + jc * a.sv.t + hk * a.sv.h);
        const typename M::Frag zero = {};
#pragma unroll
        for (int s = 0; s < L::NF; ++s) {
            kf[s] = seen ? *(const typename M::Frag*)(pk + 32 * s + 16 * hi) : zero;
            vf[s] = seen ? *(const typename M::Frag*)(pv + 32 * s + 16 * hi) : zero;
        }
    }
    const long long qst = a.sq.t * (long long)sizeof(T), dst = a.sdo.t * (long long)sizeof(T);
    const unsigned lds = (unsigned)(uintptr_t)(LDS_PTR(char))smem;
    auto issue = [&](int t, int buf) {
        const int h = hk * a.G + t / nq, i0 = r0 + (t % nq) * BQ;
        const unsigned long long valid = below(a.Tq - i0);
        const unsigned at = lds + buf * STAGE;
        load_tile<T, DH, BQ, NWAVE>((const char*)((const T*)a.q + n * a.sq.n + h * a.sq.h) + i0 * qst, (unsigned)qst, valid, at, wave, lane);
        load_tile<T, DH, BQ, NWAVE>((const char*)((const T*)a.dout + n * a.sdo.n + h * a.sdo.h) + i0 * dst, (unsigned)dst, valid, at + TILE, wave, lane);
        if (wave == 0) dma4((unsigned)lane * 4u, tile_rsrc(a.stats + stats_at(a, n, h, i0)), at + 2 * TILE);
    };
    f32x16 dk[L::ND], dv[L::ND];
#pragma unroll
    for (int d = 0; d < L::ND; ++d) { dk[d] = zero16(); dv[d] = zero16(); }
    if (nt > 0) issue(0, 0);
    for (int t = 0; t < nt; ++t) {
        dma_barrier();
        if (t + 1 < nt) issue(t + 1, (t + 1) & 1);
        const char* qt = smem + (t & 1) * STAGE;
        const char* dt = qt + TILE;
        const float* st2 = (const float*)(qt + 2 * TILE);
        const int i0 = r0 + (t % nq) * BQ;
        const unsigned bits = (unsigned)(below(min(end - i0, 32)) & ~below(lo - i0));
        if (__any(bits != 0)) {
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int f = 0; f < L::NF; ++f) {
                s = M::mac(row_frag<T, DH>(qt, lane & 31, f, hi), kf[f], s);
                dp = M::mac(row_frag<T, DH>(dt, lane & 31, f, hi), vf[f], dp);
            }
            const unsigned w = bits >> (4 * hi);
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x4 l2 = *(const f32x4*)(st2 + tok(r, hi)), de = *(const f32x4*)(st2 + 32 + tok(r, hi));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool on = (w >> tok(r + e, 0)) & 1u;
                    const float p = on ? __builtin_amdgcn_exp2f(fmaf(s[r + e], a.c, -l2[e])) : 0.f;
                    s[r + e] = p;
                    dp[r + e] = on ? p * (dp[r + e] - de[e]) : 0.f;
                }
            }
#pragma unroll
            for (int d = 0; d < L::ND; ++d) {
                dv[d] = M::template mac_t<DH>(dt, 0, d, s, dv[d], lane);
                dk[d] = M::template mac_t<DH>(qt, 0, d, dp, dk[d], lane);
            }
        }
    }
    if (j < a.Tk) {
        T* ok = (T*)a.dk + n * a.sdk.n + j * a.sdk.t + hk * a.sdk.h;
        T* ov = (T*)a.dv + n * a.sdv.n + j * a.sdv.t + hk * a.sdv.h;
#pragma unroll
        for (int d = 0; d < L::ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                M::st4(ok + 32 * d + tok(r, hi), dk[d][r] * a.scale, dk[d][r + 1] * a.scale, dk[d][r + 2] * a.scale, dk[d][r + 3] * a.scale);
                M::st4(ov + 32 * d + tok(r, hi), dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]);
            }
    }
}

// ------------------------------------------------------------------------------------------------ host side
bool fits(const DicStrides& s, long long tokens, int size) {
    // 16-byte rows, and 64 rows of a tile inside a descriptor's 31-bit range
    return s.n % (16 / size) == 0 && s.t % (16 / size) == 0 && s.h % (16 / size) == 0 && s.n >= 0 && s.t >= 0 && s.h >= 0 && (tokens <= 1 || s.t <= (1ll << 24) / size);
}
bool apart(const DicStrides& s, int N, int T, int H, int dh) { return (N <= 1 || s.n >= dh) && (T <= 1 || s.t >= dh) && (H <= 1 || s.h >= dh); }
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }
Strides st(const DicStrides& s) { return Strides{s.n, s.t, s.h}; }

int check(int dtype, const DicWinAttnParams* p, bool bwd, bool pointers = true) {
    DIC_REQUIRE(p != nullptr, "dic_win_attn: no parameters");
    DIC_REQUIRE(dtype == DIC_F32 || dtype == DIC_BF16, "dic_win_attn: dtype must be DIC_F32 or DIC_BF16");
    const int size = dtype == DIC_BF16 ? 2 : 4;
    DIC_REQUIRE(p->dh == 64 || p->dh == 128, "dic_win_attn: head dim must be 64 or 128");
    DIC_REQUIRE(p->N >= 0 && p->Tq >= 0 && p->Tk >= 0 && p->Tq <= (1 << 28) && p->Tk <= (1 << 28), "dic_win_attn: sizes out of range");
    DIC_REQUIRE(p->H > 0 && p->Hkv > 0 && p->H % p->Hkv == 0, "dic_win_attn: the number of heads must be a multiple of the number of key heads");
    DIC_REQUIRE(p->sinks >= 0 && std::isfinite(p->scale) && p->scale > 0.f, "dic_win_attn: sinks >= 0 and a positive finite scale are needed");
    const long long tiles_q = ((long long)p->Tq + BM - 1) / BM, tiles_k = ((long long)p->Tk + BM - 1) / BM;
    DIC_REQUIRE((long long)p->N * p->H * tiles_q < (1ll << 31) && (long long)p->N * p->Hkv * tiles_k < (1ll << 31), "dic_win_attn: too many tiles for one launch");
    if (!pointers) return 0;
    const bool nq = p->N && p->Tq, nk = p->N && p->Tk;
    DIC_REQUIRE(!nq || (p->q && (bwd ? p->out && p->lse && p->dout && p->dq : p->out != nullptr)), "dic_win_attn: null query-side pointer");
    DIC_REQUIRE(!nk || (p->k && p->v && (!bwd || (p->dk && p->dv))), "dic_win_attn: null key-side pointer");
    DIC_REQUIRE(aligned(p->q) && aligned(p->k) && aligned(p->v) && aligned(p->out) && (!bwd || (aligned(p->dout) && aligned(p->dq) && aligned(p->dk) && aligned(p->dv))),
                "dic_win_attn: pointers must be 16-byte aligned");
    DIC_REQUIRE(fits(p->q_stride, p->Tq, size) && fits(p->out_stride, p->Tq, size) && fits(p->k_stride, p->Tk, size) && fits(p->v_stride, p->Tk, size)
                && (!bwd || (fits(p->dout_stride, p->Tq, size) && fits(p->dq_stride, p->Tq, size) && fits(p->dk_stride, p->Tk, size) && fits(p->dv_stride, p->Tk, size))),
                "dic_win_attn: strides must be non-negative multiples of 16 bytes, and a token stride at most 16 MiB");
    DIC_REQUIRE(bwd ? apart(p->dq_stride, p->N, p->Tq, p->H, p->dh) && apart(p->dk_stride, p->N, p->Tk, p->Hkv, p->dh) && apart(p->dv_stride, p->N, p->Tk, p->Hkv, p->dh)
                    : apart(p->out_stride, p->N, p->Tq, p->H, p->dh), "dic_win_attn: rows of an output overlap");
    return 0;
}
WinArgs args_of(const DicWinAttnParams* p) {
    WinArgs a{};
    a.q = p->q; a.k = p->k; a.v = p->v; a.o = p->out; a.out = p->out; a.dout = p->dout;
    a.dq = p->dq; a.dk = p->dk; a.dv = p->dv; a.lse = p->lse;
    a.sq = st(p->q_stride); a.sk = st(p->k_stride); a.sv = st(p->v_stride); a.so = st(p->out_stride);
    a.sdo = st(p->dout_stride); a.sdq = st(p->dq_stride); a.sdk = st(p->dk_stride); a.sdv = st(p->dv_stride);
    a.key_mask = p->key_mask; a.kv_len = p->kv_len; a.q_pos = p->q_pos;
    a.N = p->N; a.Tq = p->Tq; a.Tk = p->Tk; a.H = p->H; a.Hkv = p->Hkv; a.G = p->H / p->Hkv;
    a.left = p->left < 0 ? -1 : (p->left < FAR / 2 ? p->left : FAR / 2);
    a.right = p->right < 0 ? -1 : (p->right < FAR / 2 ? p->right : FAR / 2);
    a.sinks = p->sinks; a.scale = p->scale; a.c = p->scale * LOG2E;
    return a;
}
template <typename K> int launch(K kernel, long long blocks, size_t lds, const WinArgs& a, hipStream_t st) {
    // (set on every launch: the attribute belongs to the current device's copy of the kernel)
    hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) { dic_set_error(hipGetErrorString(e)); return (int)e; }
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), lds, st, a);
    DIC_CHECK_LAUNCH();
    return 0;
}
template <typename T, int DH> int fwd(const WinArgs& a, hipStream_t st) {
    constexpr int BN = sizeof(T) == 2 ? 64 : 32;
    return launch(win_fwd_kernel<T, DH, BN>, (long long)a.N * a.H * ((a.Tq + BM - 1) / BM), (size_t)4 * BN * Lay<T, DH>::ROWB, a, st);
}
template <typename T, int DH> int bwd(const WinArgs& a, hipStream_t st) {
    constexpr int BN = sizeof(T) == 2 ? 64 : 32;
    if (a.Tq > 0)
        if (int rc = launch(win_bwd_dq_kernel<T, DH, BN>, (long long)a.N * a.H * ((a.Tq + BM - 1) / BM), (size_t)4 * BN * Lay<T, DH>::ROWB, a, st)) return rc;
    if (a.Tk > 0) return launch(win_bwd_dkv_kernel<T, DH>, (long long)a.N * a.Hkv * ((a.Tk + BM - 1) / BM), (size_t)2 * (2 * BQ * Lay<T, DH>::ROWB + 256), a, st);
    return 0;
}
}  // namespace

extern "C" size_t dic_win_attn_ws_bytes(int dtype, int backward, const DicWinAttnParams* p) {
    if (check(dtype, p, false, false)) return 0;
    return backward ? (size_t)stats_floats(p->N, p->H, p->Tq) * sizeof(float) : 0;
}

extern "C" int dic_win_attn_fwd(int dtype, const DicWinAttnParams* p, void* stream) {
    if (int rc = check(dtype, p, false)) return rc;
    if (p->N == 0 || p->Tq == 0) return 0;
    const WinArgs a = args_of(p);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DIC_BF16) return p->dh == 64 ? fwd<bf16_t, 64>(a, st) : fwd<bf16_t, 128>(a, st);
    return p->dh == 64 ? fwd<float, 64>(a, st) : fwd<float, 128>(a, st);
}

extern "C" int dic_win_attn_bwd(int dtype, const DicWinAttnParams* p, void* stream) {
    if (int rc = check(dtype, p, true)) return rc;
    if (p->N == 0) return 0;
    const size_t need = (size_t)stats_floats(p->N, p->H, p->Tq) * sizeof(float);
    DIC_REQUIRE(need == 0 || (p->ws && aligned(p->ws) && p->ws_bytes >= need), "dic_win_attn_bwd: workspace missing or too small (dic_win_attn_ws_bytes)");
    WinArgs a = args_of(p);
    a.stats = (float*)p->ws;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == DIC_BF16) return p->dh == 64 ? bwd<bf16_t, 64>(a, st) : bwd<bf16_t, 128>(a, st);
    return p->dh == 64 ? bwd<float, 64>(a, st) : bwd<float, 128>(a, st);
}
