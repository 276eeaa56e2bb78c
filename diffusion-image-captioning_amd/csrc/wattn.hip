// Attention over long token rows: a sliding window per query, the first `sinks` keys visible behind it, any number of query heads per key head.
//   s_ij = scale q_i . k_j over the visible j,  lse_i = log sum_j exp s_ij,  p_ij = exp(s_ij - lse_i),  out_i = sum_j p_ij v_j
//   delta_i = dout_i . out_i,  ds_ij = p_ij (dout_i . v_j - delta_i) scale,  dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
// Every product runs on 32x32 MFMA tiles with the score tile TRANSPOSED or not so that the dimension that is reduced next lies in a lane's registers:
// the forward and the dq kernel hold S^T (lane = query, registers = keys), the dk / dv kernel holds S (lane = key, registers = queries).  A lane's 16
// values are then the B operand of the next product as they are -- no LDS round trip for P or dS -- if that product's A operand is read token-major
// from LDS in the same token order, which ds_read_b64_tr_b16 (bf16) or plain 4-byte reads (fp32) give.
// Tiles come in by LDS-DMA, double-buffered; rows of keys that nobody may see (key_mask, kv_len) are zero-filled by the descriptor's bounds check, so
// that an infinity or NaN in them cannot reach 0 * v.
#include <atomic>
#include <cmath>
#include <type_traits>
#include "common.h"
#include "../../include/dic_hip.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// Positions are clamped to +-FAR_POS and bounds to FAR, which is behind every key from every position (there are at most 2^28 rows), so that a finite bound
// never cuts where the unclamped one would not; position + rows + bound stays inside 32 bits.
constexpr int FAR_POS = 1 << 29, FAR = (1 << 30) - 2;

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
    float* sinks_ws;                            // backward workspace [N Hkv][chunks][sink_rows][dk, dv]
    float* parts;                               // few-rows workspace: [N Hkv][splits][rows][DH], then {m, l} of each
    int N, Tq, Tk, H, Hkv, G, left, right, sinks;
    int near_sinks;                             // backward: sinks that the window pass takes along
    int sink_keys, sink_rows, chunks;           // or those that have a pass of their own, that rounded up to 32, and pieces of that pass
    float scale, c;                             // c = scale * log2(e)
};

__device__ __forceinline__ int tok(int r, int hi) { return (r & 3) + 8 * (r >> 2) + 4 * hi; }     // row of register r of a 32x32 accumulator
__device__ __forceinline__ f32x16 zero16() { f32x16 z; for (int i = 0; i < 16; ++i) z[i] = 0.f; return z; }

// An LDS tile holds token rows of DH elements, cut into segments of 64 bytes (4 chunks of 16).  One DMA instruction fills a piece of 1 KiB, in which the same
// segment of 4 rows (512-byte rows: 2) lies side by side; pieces are PS bytes apart.  Both readings are then free of bank conflicts -- 64 bytes of each of 4
// rows are 256 consecutive bytes (transposing reads), and the padding between pieces turns 16 consecutive rows at one chunk over all banks (row operands,
// ds_read_b128; 128-byte rows, two quads to a piece, also swap neighbouring chunks in every odd quad) -- and every address is a lane's base plus a constant.
template <typename T, int DH> struct Lay {
    static constexpr int ROWB = DH * (int)sizeof(T), CH = ROWB / 16, NF = ROWB / 32, ND = DH / 32, PIECE_ROWS = 1024 / ROWB;
    static constexpr int PS = CH == 8 ? 1056 : 1040, SEG = CH == 32 ? 128 : 256;            // bytes between pieces; between a row's segments
    static constexpr int bytes(int rows) { return rows / PIECE_ROWS * PS; }
    // what a lane of the DMA instruction carries: row and chunk inside the piece
    __device__ static __forceinline__ int dma_row(int lane) { return CH == 8 ? (lane >> 5) * 4 + ((lane >> 2) & 3) : CH == 16 ? (lane >> 2) & 3 : (lane >> 2) & 1; }
    __device__ static __forceinline__ int dma_chunk(int lane) {
        return CH == 8 ? ((lane >> 4) & 1) * 4 + ((lane & 3) ^ (lane >> 5)) : CH == 16 ? (lane >> 4) * 4 + (lane & 3) : (lane >> 3) * 4 + (lane & 3);
    }
    // row operand of a 32-row block: lane's row lane & 31, chunk 2 s + (lane >> 5) at base + step(s)
    __device__ static __forceinline__ int row_base(int lane) {
        const int r = lane & 31, hi = lane >> 5, q = (r >> 2) & 1;
        return CH == 8 ? (r >> 3) * PS + q * 512 + (r & 3) * 64 + ((hi ^ q) << 4) : CH == 16 ? (r >> 2) * PS + (r & 3) * 64 + (hi << 4) : (r >> 1) * PS + (r & 1) * 64 + (hi << 4);
    }
    static constexpr int step(int s) { return (s >> 1) * SEG + (s & 1) * 32; }
    // bf16, transposing reads: 4 elements of rows 4 hi + (t >> 2), t = lane & 15, of a 16-row block; + up for the rows 8 further on
    __device__ static __forceinline__ int tr_base(int lane) {
        const int hi = lane >> 5, c = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1), r = (lane & 15) >> 2, sub = (lane & 1) * 8;
        return CH == 8 ? hi * 512 + r * 64 + ((c ^ hi) << 4) + sub : hi * PS + r * 64 + (c << 4) + sub;
    }
    static constexpr int up = 8 / PIECE_ROWS * PS;
    // fp32, by element: lane's element lane & 31 of row tok(r, hi), at base + at(r)
    __device__ static __forceinline__ int el_base(int lane) { return (lane >> 5) * (4 / PIECE_ROWS) * PS + ((lane >> 4) & 1) * SEG + (lane & 15) * 4; }
    static constexpr int at(int r) { return (8 / PIECE_ROWS) * (r >> 2) * PS + (PIECE_ROWS == 4 ? (r & 3) * 64 : ((r & 3) >> 1) * PS + (r & 1) * 64); }
};

// Row operand of a 32-token block: lane holds row (lane & 31), bytes 32 s + 16 (lane >> 5).
template <typename T> struct Mma;
template <> struct Mma<bf16_t> {
    typedef bf16x8 Frag;
    __device__ static __forceinline__ f32x16 mac(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    // acc[d][col] += sum over 32 tokens of tile[token][32 db + d] * p[token][col], p in accumulator order: the tile's part, p's part, the product
    struct Turned { bf16x8 f[2]; };
    struct Right { bf16x8 f[2]; };
    template <int DH> __device__ static __forceinline__ Turned turned(const char* tile, int db, int lane) {
        using L = Lay<bf16_t, DH>;
        const char* base = tile + L::tr_base(lane) + db * L::SEG;
        Turned a;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(base + 2 * s * L::up));
            s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_PTR(s16x4))(base + (2 * s + 1) * L::up));
            a.f[s] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7));
        }
        return a;
    }
    __device__ static __forceinline__ Right right(const f32x16& p) {
        Right r;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            i32x4 b;
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = (int)pack2bf(p[8 * s + 2 * e], p[8 * s + 2 * e + 1]);
            r.f[s] = __builtin_bit_cast(bf16x8, b);
        }
        return r;
    }
    __device__ static __forceinline__ f32x16 mac_t(const Turned& a, const Right& b, f32x16 acc) {
#pragma unroll
        for (int s = 0; s < 2; ++s) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.f[s], b.f[s], acc, 0, 0, 0);
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
    struct Turned { float f[16]; };
    typedef f32x16 Right;
    template <int DH> __device__ static __forceinline__ Turned turned(const char* tile, int db, int lane) {
        using L = Lay<float, DH>;
        const char* base = tile + L::el_base(lane) + 2 * db * L::SEG;
        Turned a;
#pragma unroll
        for (int r = 0; r < 16; ++r) a.f[r] = *(const float*)(base + L::at(r));
        return a;
    }
    __device__ static __forceinline__ Right right(const f32x16& p) { return p; }
    __device__ static __forceinline__ f32x16 mac_t(const Turned& a, const Right& b, f32x16 acc) {
#pragma unroll
        for (int r = 0; r < 16; ++r) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.f[r], b[r], acc, 0, 0, 0);
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
__device__ __forceinline__ void dma16(unsigned voff, const i32x4& rsrc, unsigned soff, unsigned lds_addr) {   // 64 lanes x 16 B -> 1 KiB at lds_addr
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(rsrc), "s"(soff), "s"(__builtin_amdgcn_readfirstlane(lds_addr)) : "memory");
}
__device__ __forceinline__ void dma4(unsigned voff, const i32x4& rsrc, unsigned lds_addr) {            // 64 lanes x 4 B
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(lds_addr)) : "memory");
}
// this wave's DMA has landed and, behind the barrier, everybody's has; everybody is done with the buffer that is refilled next
__device__ __forceinline__ void dma_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ROWS token rows from `base` (row stride st bytes) into a tile; bit r of `valid`: row r is read, else zero.  NW > 0: the pieces are dealt evenly to that
// many waves, each the same number; NW = 0: waves first, first + step, ... take them in turn.
template <typename T, int DH, int ROWS, int NW>
__device__ __forceinline__ void load_tile(const char* base, unsigned st, unsigned long long valid, unsigned lds, int first, int step, int lane) {
    using L = Lay<T, DH>;
    const i32x4 rs = tile_rsrc(base);
    constexpr int P = ROWS / L::PIECE_ROWS;
    constexpr unsigned long long ALL = ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1;
    static_assert(ROWS % L::PIECE_ROWS == 0 && (NW == 0 || P % (NW ? NW : 1) == 0), "whole pieces, the same number for each wave");
    const unsigned off = (unsigned)L::dma_row(lane) * st + (unsigned)L::dma_chunk(lane) * 16u;
    auto one = [&](int piece, bool all) {
        const int row = piece * L::PIECE_ROWS;
        dma16(all || ((valid >> (row + L::dma_row(lane))) & 1ull) ? off : 0xfffffff0u, rs, (unsigned)row * st, lds + (unsigned)(piece * L::PS));
    };
    if constexpr (NW > 0) {
        if (valid == ALL) {
#pragma unroll
            for (int j = 0; j < P / NW; ++j) one(j * NW + first, true);
        } else {
#pragma unroll
            for (int j = 0; j < P / NW; ++j) one(j * NW + first, false);
        }
    } else if (valid == ALL)
        for (int piece = first; piece < P; piece += step) one(piece, true);
    else
        for (int piece = first; piece < P; piece += step) one(piece, false);
}
// The loads of `f` end here.  Left to their first use, inside the loop over tiles, the compiler's wait there would be for every load in flight, the next
// tiles' DMA among them (which it does not know of), in every turn.
template <typename F, int N> __device__ __forceinline__ void landed(F (&f)[N]) {
#pragma unroll
    for (int s = 0; s < N; ++s) asm volatile("" : "+v"(f[s]));
}
template <typename T, int DH>
__device__ __forceinline__ typename Mma<T>::Frag row_frag(const char* tile, int s, int lane) {
    return *(const typename Mma<T>::Frag*)(tile + Lay<T, DH>::row_base(lane) + Lay<T, DH>::step(s));
}

// An accumulated block (lane = row, registers = elements) times `mul` into a tensor: lane's row at `to`.
template <typename T, int DH> __device__ __forceinline__ void store_row(const f32x16 (&acc)[DH / 32], float mul, T* to, int hi) {
#pragma unroll
    for (int d = 0; d < DH / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) Mma<T>::st4(to + 32 * d + tok(r, hi), acc[d][r] * mul, acc[d][r + 1] * mul, acc[d][r + 2] * mul, acc[d][r + 3] * mul);
}
// The same through LDS (32 rows of ROWB + 16 bytes, the wave's own) into 32 rows, `rows` of them real: a store instruction then writes whole rows instead of
// 16 bytes of each of 32.  It takes registers and a barrier.  In the dk / dv kernel of 128 wide bf16 rows it pays where a workgroup has all keys of a head (whole
// backward passes: 600 key heads of 256 keys 256 us, without it 267; of 200 keys 244 and 254) and costs 1 to 3 per cent where it has four waves (4 x 2048
// rows, 16 query and 4 key heads: 417 and 405; the kernel alone at 2 x 4096 keys in windows of 1024: 169 and 165).  64 wide rows lose by it (117 -> 126 us);
// forward and dq, any type: no difference.
template <typename T, int DH> constexpr int OUT_ROW = Lay<T, DH>::ROWB + 16;
template <typename T, int DH> constexpr bool WHOLE_ROWS = sizeof(T) == 2 && DH == 128;
template <typename T, int DH>
__device__ __forceinline__ void store_rows(char* lds, const f32x16 (&acc)[DH / 32], float mul, T* to, long long stride, int rows, int lane) {
    using L = Lay<T, DH>;
    const int hi = lane >> 5;
    char* mine = lds + (lane & 31) * OUT_ROW<T, DH>;
#pragma unroll
    for (int d = 0; d < L::ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            Mma<T>::st4((T*)mine + 32 * d + tok(r, hi), acc[d][r] * mul, acc[d][r + 1] * mul, acc[d][r + 2] * mul, acc[d][r + 3] * mul);
#pragma unroll
    for (int e = 0; e < 32 * L::CH / 64; ++e) {
        const int row = (e * 64 + lane) / L::CH, c = (e * 64 + lane) % L::CH;
        const i32x4 v = *(const i32x4*)(lds + row * OUT_ROW<T, DH> + c * 16);
        if (row < rows) *(i32x4*)((char*)(to + row * stride) + c * 16) = v;
    }
}

__device__ __forceinline__ unsigned long long below(int x) { return x <= 0 ? 0ull : x >= 64 ? ~0ull : (1ull << x) - 1ull; }
__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// The position of a sequence's first query, and the keys that none of its queries sees, which count as absent: those from kvl on (they do not exist, or
// lie in front of everybody), and [sinks, from), behind everybody's window.
struct Seq { int kvl, pos, from; };
__device__ __forceinline__ Seq sequence(const WinArgs& a, int n) {
    Seq s;
    s.kvl = a.kv_len ? clampi(a.kv_len[n], 0, a.Tk) : a.Tk;
    s.pos = a.q_pos ? clampi(a.q_pos[n], -FAR_POS, FAR_POS) : 0;
    if (a.right >= 0) s.kvl = clampi(s.pos + a.Tq + a.right, 0, s.kvl);
    s.from = a.left < 0 ? 0 : max(0, s.pos - a.left);
    return s;
}
// Query at position t sees the keys [lo, hi) and [0, sk).
struct Span {
    int lo, hi, sk;
    __device__ __forceinline__ int keys() const { return max(0, hi - lo) + min(sk, lo); }        // (sinks inside the window are counted once)
};
__device__ __forceinline__ Span span_of(const WinArgs& a, int t, int kvl) {
    Span s;
    s.lo = a.left < 0 ? 0 : max(0, t - a.left);
    s.hi = a.right < 0 ? kvl : clampi(t + a.right + 1, 0, kvl);
    s.sk = a.left < 0 ? 0 : min(a.sinks, s.hi);
    return s;
}
__device__ __forceinline__ unsigned long long visible(const Span& s, int j0) { return (below(s.hi - j0) & ~below(s.lo - j0)) | below(s.sk - j0); }

// bits of the keys j0 .. j0 + 63 that somebody may see
__device__ __forceinline__ unsigned long long there(const WinArgs& a, int kvl, int from, int j0) { return below(kvl - j0) & (~below(from - j0) | below(a.sinks - j0)); }

// The key tiles that the queries at positions t0..t1 need: those of the sinks, then those of the windows.
struct Walk {
    int ns, w0, nt, kvl, from;
    __device__ __forceinline__ int j0(int t, int bn) const { return (t < ns ? t : w0 + t - ns) * bn; }
};
__device__ __forceinline__ Walk walk_of(const WinArgs& a, int t0, int t1, const Seq& sq, int bn) {
    Walk w;
    const int lo = span_of(a, t0, sq.kvl).lo;
    const Span e = span_of(a, t1, sq.kvl);
    w.kvl = sq.kvl;
    w.from = sq.from;
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

template <typename T> constexpr int MOST_WAVES = sizeof(T) == 2 ? 8 : 4;      // of a workgroup: fp32 operands need more than half of a SIMD's registers
// waves that a SIMD is to hold at once: what the registers of bf16 rows of 64 allow, 2 for rows of 256 bytes, 1 for rows of 512
template <typename T, int DH, int MOST> constexpr int RESIDENT = sizeof(T) * DH > 256 ? 1 : sizeof(T) * DH == 256 ? 2 : MOST;
constexpr int BQ = 32;                          // queries (or keys) per wave, and rows of a statistics tile
__host__ __device__ __forceinline__ long long stats_floats(long long N, long long H, long long Tq) { return N * H * ((Tq + BQ - 1) / BQ) * 2 * BQ; }
__device__ __forceinline__ long long stats_at(const WinArgs& a, int n, int h, int i0) { return stats_floats(1, (long long)n * a.H + h, a.Tq) + 2 * i0; }

// The key and value tiles of a workgroup's walk in LDS.  NW > 0: two turns of KS tiles, and that many waves fetch the next turn behind the barrier in front of
// one.  KS = 2: the first half of the waves takes the even tiles, the second the odd ones, for the same rows; they add up their results at the end.
// NW = 0: the walk has at most FEW_TILES, and whatever waves there are fetch all of them at the start.
constexpr int FEW_TILES = 4, MASK_RUN = 256;
template <typename T, int DH, int BN, int NW, int KS> struct KeyTiles {
    using L = Lay<T, DH>;
    static constexpr int TILE = L::bytes(BN), SLOTS = NW ? 2 * KS : FEW_TILES;
    const WinArgs& a;
    const Walk wk;
    const char *kb, *vb, *smem;
    const long long kst, vst;
    const int n, wave, nw, lane;
    unsigned long long* table;                                // with key_mask: the masks of the next tiles, a ring of 2 MASK_RUN
    __device__ __forceinline__ KeyTiles(const WinArgs& a, const Walk& wk, int n, int hk, char* smem, unsigned long long* table, int wave, int lane)
        : a(a), wk(wk), kb((const char*)((const T*)a.k + n * a.sk.n + hk * a.sk.h)), vb((const char*)((const T*)a.v + n * a.sv.n + hk * a.sv.h)), smem(smem),
          kst(a.sk.t * (long long)sizeof(T)), vst(a.sv.t * (long long)sizeof(T)), n(n), wave(wave), nw(NW ? NW : blockDim.x >> 6), lane(lane), table(table) {}
    // masks of the tiles t .. t + MASK_RUN - 1 (barriers around it)
    __device__ __forceinline__ void read_masks(int t) {
        for (int k = t + wave; k < min(t + MASK_RUN, wk.nt); k += nw) {
            const int j = wk.j0(k, BN) + lane;
            const unsigned long long v = __ballot(lane < BN && j < a.Tk && a.key_mask[(size_t)n * a.Tk + j] != 0);
            if (lane == 0) table[k & (2 * MASK_RUN - 1)] = v;
        }
    }
    // bits of the keys of tile t that exist and are not masked
    __device__ __forceinline__ unsigned long long valid(int t) const {
        unsigned long long v = there(a, wk.kvl, wk.from, wk.j0(t, BN)) & below(BN);
        if (a.key_mask) {
            const unsigned long long m = table[t & (2 * MASK_RUN - 1)];
            v &= (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)m) | (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(m >> 32)) << 32;
        }
        return v;
    }
    __device__ __forceinline__ void issue(int t) const {
        const int j0 = wk.j0(t, BN);
        const unsigned long long v = valid(t);
        const unsigned lds = (unsigned)(uintptr_t)(LDS_PTR(const char))smem + (t & (SLOTS - 1)) * 2 * TILE;
        load_tile<T, DH, BN, NW>(kb + j0 * kst, (unsigned)kst, v, lds, wave, nw, lane);
        load_tile<T, DH, BN, NW>(vb + j0 * vst, (unsigned)vst, v, lds + TILE, wave, nw, lane);
    }
    __device__ __forceinline__ void begin() {
        if (a.key_mask) { read_masks(0); __syncthreads(); }
        for (int t = 0; t < min(wk.nt, NW ? KS : FEW_TILES); ++t) issue(t);
        if constexpr (NW == 0) dma_barrier();
    }
    // the turn's tiles t .. t + KS - 1, as far as there are, are in LDS behind this call
    __device__ __forceinline__ void step(int t) {
        if constexpr (NW > 0) {
            dma_barrier();
            if (t + KS < wk.nt) {
                if (a.key_mask && ((t + KS) & (MASK_RUN - 1)) == 0) { read_masks(t + KS); __syncthreads(); }
#pragma unroll
                for (int k = 0; k < KS; ++k)
                    if (k == 0 || t + KS + k < wk.nt) issue(t + KS + k);
            }
        }
    }
    // the keys of tile t; its values lie TILE bytes further on
    __device__ __forceinline__ const char* at(int t) const { return smem + (t & (SLOTS - 1)) * 2 * TILE; }
};

// ------------------------------------------------------------------------------------------------ forward
// One pass over the keys with the running maximum and sum per query.  P is rounded to bf16 in front of its product, relative to its size, and the sums are fp32
// (l of the unrounded P: a product of bf16 operands is what the matrix unit has, and each P is off by half a step at most, evenly to both sides).
// Long spans are bound by the issue of matrix and vector instructions together (a 32 x 32 block is 16 of the former at 32 cycles a SIMD, and some 450 cycles of
// exponentials, masks, maxima and conversions; two or three waves a SIMD overlap them in part): 8192 rows that see 4096 keys, 16 heads of 128: 250 us, 825
// TFLOP/s of visible pairs, where a library matrix product reaches 1350; in windows of 1024, 2 x 4096 rows: 90 us, 670.  The matrix unit is busy 41 and 34 per
// cent of the CUs' time there, LDS reads 22 and 18, without a bank conflict: neither is the limit by itself.  Short ones are bound by moving their rows with
// little to compute meanwhile: 256 x 12 heads of 130 x 64: 197 MB in 66 us, 3.0 TB/s.  8 x 2050 rows in windows of 513, 12 heads of 64: 51 us.
template <typename T, int DH, int BN, int NW, int KS>
__global__ __launch_bounds__(64 * MOST_WAVES<T>, (DH == 128 && BN == 32 && sizeof(T) == 2 ? 3 : RESIDENT<T, DH, 4>)) void win_fwd_kernel(const WinArgs a) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    constexpr int NB = BN / 32, TILE = L::bytes(BN);
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5;
    constexpr int ROWS = NW / KS;                             // waves with rows of their own, or 0: all
    const int row_wave = KS > 1 ? wave % ROWS : wave, half = KS > 1 ? wave / ROWS : 0;
    const int bm = (NW ? ROWS : blockDim.x >> 6) * BQ, nqt = (a.Tq + bm - 1) / bm;
    int item = xcd_item();
    const int g = item % a.G; item /= a.G;
    const int qt = nqt - 1 - item % nqt; item /= nqt;         // long rows first
    const int hk = item % a.Hkv, n = item / a.Hkv, h = hk * a.G + g;
    const Seq sq = sequence(a, n);
    const int i0 = qt * bm + row_wave * BQ, i = i0 + (lane & 31), ic = min(i, a.Tq - 1);
    const Walk wk = walk_of(a, sq.pos + qt * bm, sq.pos + min(qt * bm + bm, a.Tq) - 1, sq, BN);
    const Span sp = span_of(a, sq.pos + ic, sq.kvl);
    const bool wave_rows = i0 < a.Tq;
    // what every row of this wave sees: [in_lo, in_hi)
    const int in_lo = span_of(a, sq.pos + min(i0 + 31, a.Tq - 1), sq.kvl).lo, in_hi = span_of(a, sq.pos + min(i0, a.Tq - 1), sq.kvl).hi;

    typename M::Frag qf[L::NF];
    {
        const char* p = (const char*)((const T*)a.q + n * a.sq.n + ic * a.sq.t + h * a.sq.h);
#pragma unroll
        for (int s = 0; s < L::NF; ++s) qf[s] = *(const typename M::Frag*)(p + 32 * s + 16 * hi);
        landed(qf);
    }
    __shared__ unsigned long long table[2 * MASK_RUN];
    KeyTiles<T, DH, BN, NW, KS> tiles(a, wk, n, hk, smem, table, wave, lane);
    tiles.begin();

    f32x16 acc[L::ND];
#pragma unroll
    for (int d = 0; d < L::ND; ++d) acc[d] = zero16();
    float m = -INFINITY, l = 0.f;
    // one step over `count` blocks of 32 keys of a tile, from block b0 on
    auto blocks = [&](auto count, int b0, const char* kt, const char* vt, unsigned long long bits, bool full) {
        constexpr int C = decltype(count)::value;
        f32x16 st[C];
        kt += b0 * L::bytes(32);
        vt += b0 * L::bytes(32);
#pragma unroll
        for (int b = 0; b < C; ++b) {
            st[b] = zero16();
#pragma unroll
            for (int s = 0; s < L::NF; ++s) st[b] = M::mac(row_frag<T, DH>(kt + L::bytes(32 * b), s, lane), qf[s], st[b]);
        }
        if (!full) {
#pragma unroll
            for (int b = 0; b < C; ++b) {
                const unsigned w = (unsigned)(bits >> (32 * (b0 + b))) >> (4 * hi);
#pragma unroll
                for (int r = 0; r < 16; ++r) st[b][r] = (w >> tok(r, 0)) & 1u ? st[b][r] : -INFINITY;
            }
        }
        float mt = st[0][0];
#pragma unroll
        for (int b = 0; b < C; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) mt = fmaxf(mt, st[b][r]);
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * a.c;
        // The reference point m of the exponentials follows the running maximum only when that is more than 2^8 above it: the sums are in 32 bits and
        // P's relative rounding does not depend on its size, and most tiles then leave the accumulators as they are.
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
        for (int b = 0; b < C; ++b) {
#pragma unroll
            for (int r = 0; r < 16; ++r) { st[b][r] = __builtin_amdgcn_exp2f(fmaf(st[b][r], a.c, -mm)); l += st[b][r]; }
#pragma unroll
            for (int d = 0; d < L::ND; ++d) acc[d] = M::mac_t(M::template turned<DH>(vt + L::bytes(32 * b), d, lane), M::right(st[b]), acc[d]);
        }
    };
    for (int t0 = 0; t0 < wk.nt; t0 += KS) {
        tiles.step(t0);
        const int t = t0 + half;
        if (KS > 1 && t >= wk.nt) break;                      // (the last turn)
        const int j0 = wk.j0(t, BN);
        const char* kt = tiles.at(t);
        const char* vt = kt + TILE;
        const unsigned long long valid = tiles.valid(t);
        unsigned long long bits = ~0ull;
        const bool full = j0 >= in_lo && j0 + BN <= in_hi && valid == below(BN);
        if (!full) bits = visible(sp, j0) & valid;
        if (wave_rows && (full || __any(bits != 0))) {
            // blocks of 32 keys that no row of the wave sees are left out
            if constexpr (NB == 1) blocks(std::integral_constant<int, 1>(), 0, kt, vt, bits, full);
            else {
                const bool first = full || __any((unsigned)bits != 0), second = full || __any((unsigned)(bits >> 32) != 0);
                if (first && second) blocks(std::integral_constant<int, 2>(), 0, kt, vt, bits, full);
                else blocks(std::integral_constant<int, 1>(), first ? 0 : 1, kt, vt, bits, full);
            }
        }
    }
    if constexpr (KS > 1) {
        float* const to = (float*)smem + row_wave * (L::ND * 16 + 2) * 64 + lane;
        __syncthreads();                                      // the tiles are done with
        if (half) {
#pragma unroll
            for (int d = 0; d < L::ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) to[(d * 16 + r) * 64] = acc[d][r];
            to[L::ND * 16 * 64] = m;
            to[(L::ND * 16 + 1) * 64] = l;
        }
        __syncthreads();
        if (half) return;
        const float m1 = to[L::ND * 16 * 64], mn = fmaxf(m, m1), mm = mn == -INFINITY ? 0.f : mn;
        const float f0 = __builtin_amdgcn_exp2f(m - mm), f1 = __builtin_amdgcn_exp2f(m1 - mm);
        m = mn;
        l = l * f0 + to[(L::ND * 16 + 1) * 64] * f1;
#pragma unroll
        for (int d = 0; d < L::ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = acc[d][r] * f0 + to[(d * 16 + r) * 64] * f1;
    }
    l += __shfl_xor(l, 32, 64);
    if (i < a.Tq) {
        store_row<T, DH>(acc, l == 0.f ? 0.f : 1.f / l, (T*)a.out + n * a.so.n + i * a.so.t + h * a.so.h, hi);
        if (a.lse && hi == 0) a.lse[((long long)n * a.H + h) * a.Tq + i] = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l)) * LN2;
    }
}

// ------------------------------------------------------------------------------------------------ backward: dq (and delta)
// Rows that see at most FEW_KEYS keys get the exact delta (dq_block): those of narrow windows and masks and the first ones of a causal text, whose gradients
// are the largest.  Beyond that, with logits of deviation 1, it changes less than a tenth of the rounding errors; where the weight of such a row rests on a few of
// its keys all the same, the rounded `out` shows (logits of deviation 5 over up to 900 keys: dq 3.7e-3 and dk 3.4e-3 of the norm off), as it is when `out` is all
// that the forward pass keeps.  The exact form costs a third more products, and carrying both the plain one its best schedule: 126 us for 121 (2 x 4096 rows,
// 16 heads of 128, windows of 1024), where a branch inside of one loop cost more.
template <typename T> constexpr bool BF16 = sizeof(T) == 2;
constexpr int FEW_KEYS = 256;
template <int ND> __device__ __forceinline__ float exactly(f32x16 (&acc)[ND], const f32x16 (&mean)[ND], float off) {        // acc with the exact delta; returns off of the row
    off += __shfl_xor(off, 32, 64);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = fmaf(-off, mean[d][r], acc[d][r]);
    return off;
}
// Does key_mask leave a row between those of the spans s0 (the first) and s1 (the last) at most FEW_KEYS keys?  Counts the keys that all of these rows see, so
// that no such row is missed; some rows with up to the workgroup's row count more then get the exact form, too.  Every wave counts for itself (the same bytes,
// the same answer), 512 keys to a round trip, and stops once there are enough: one or two round trips where most keys are there (masked backward pass, 2 x 4096 rows, 16 heads of
// 128, a tenth of the keys masked: windows of 1024 325 -> 329 us; of 341, whose rows share 214 keys, in the exact form now: 184 -> 196).
__device__ __forceinline__ bool mask_leaves_few(const WinArgs& a, int n, const Span& s0, const Span& s1) {
    const uint8_t* mask = a.key_mask + (size_t)n * a.Tk;
    const int lane = threadIdx.x & 63;
    int count = 0;
    auto add = [&](int lo, int hi) {
        for (int j0 = lo; j0 < hi && count <= FEW_KEYS; j0 += 512) {
            int byte[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) { const int j = j0 + 64 * e + lane; byte[e] = j < hi ? mask[j] : 0; }
#pragma unroll
            for (int e = 0; e < 8; ++e) count += __popcll(__ballot(byte[e] != 0));
        }
    };
    add(s1.lo, s0.hi);
    add(0, min(s0.sk, s1.lo));
    return count <= FEW_KEYS;
}
// acc += the part of dq / scale that 32 keys have; bit of `word`: the lane's query sees that key (`full`: all of them).
// EXACT (bf16): delta is dout . out with the ROUNDED out, off by e_i; where few keys share a row's weight that outweighs what rounding ds costs (windows of 3 keys in
// bf16: dq and dk 3.7e-3 off, in norm, of which rounding the results themselves is 1.7e-3).  Then `off` sums ds in 32 bits over the lane's keys, which is
// -e_i as the p_ij of a row sum to 1, and `mean` the rows p_ij k_j, so that dq = acc - off mean is what the exact delta gives (2.35e-3; a third more products:
// 4 texts of 2048 x 12 heads, windows of 256: 63 us for the backward pass, 61 without).
// With KEPT < NF the rest of the lane's dout row lies in LDS, 1 KiB apart.
template <typename T, int DH, bool EXACT, int KEPT>
__device__ __forceinline__ void dq_block(const char* kt, const char* vt, const typename Mma<T>::Frag (&qf)[Lay<T, DH>::NF], const typename Mma<T>::Frag (&df)[KEPT],
                                         const char* parked, float c, float l2, float delta, unsigned word, bool full, f32x16 (&acc)[DH / 32], f32x16 (&mean)[EXACT ? DH / 32 : 1], float& off, int lane) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    f32x16 st = zero16(), dp = zero16();
#pragma unroll
    for (int s = 0; s < L::NF; ++s) {
        st = M::mac(row_frag<T, DH>(kt, s, lane), qf[s], st);
        dp = M::mac(row_frag<T, DH>(vt, s, lane), s < KEPT ? df[s < KEPT ? s : 0] : *(const typename M::Frag*)(parked + (s - KEPT) * 1024), dp);
    }
    if constexpr (EXACT) __builtin_amdgcn_sched_barrier(0);
    const unsigned w = word >> (4 * (lane >> 5));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(st[r], c, -l2));
        st[r] = full || ((w >> tok(r, 0)) & 1u) ? p : 0.f;
        dp[r] = st[r] * (dp[r] - delta);
        if constexpr (EXACT) off += dp[r];
    }
#pragma unroll
    for (int d = 0; d < L::ND; ++d) {
        const typename M::Turned t = M::template turned<DH>(kt, d, lane);
        acc[d] = M::mac_t(t, M::right(dp), acc[d]);
        if constexpr (EXACT) mean[d] = M::mac_t(t, M::right(st), mean[d]);
    }
}
// Bound as the forward pass is, with three products a block for its two.  2 x 4096 rows in windows of 1024, 16 heads of 128: 126 us, 720 TFLOP/s of visible
// pairs, 4 registers spilled; fp32, 4 x 513 rows in windows of 257, 12 heads of 64: 44 us.  ds is rounded to bf16 in front of its product.
// The rows of one workgroup: query tile qt of query head h, key head hk, sequence n
template <typename T, int DH, int BN, int NW, int KS, bool EXACT>
__device__ __forceinline__ void dq_rows(const WinArgs& a, int n, int hk, int h, int qt, const Seq& sq, char* smem, unsigned long long* table) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    constexpr int NB = BN / 32, TILE = L::bytes(BN);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5;
    constexpr int ROWS = NW / KS;
    const int row_wave = KS > 1 ? wave % ROWS : wave, half = KS > 1 ? wave / ROWS : 0, bm = (NW ? ROWS : blockDim.x >> 6) * BQ;
    const int i0 = qt * bm + row_wave * BQ, i = i0 + (lane & 31), ic = min(i, a.Tq - 1);
    const Walk wk = walk_of(a, sq.pos + qt * bm, sq.pos + min(qt * bm + bm, a.Tq) - 1, sq, BN);
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
        landed(qf);
        landed(df);
    }
    // rows that see nothing, and those behind the last that fill a tile of statistics up, get lse = +inf: the dk / dv kernel's exponentials are then zero
    float l2 = a.lse[((long long)n * a.H + h) * a.Tq + ic] * LOG2E;
    if (l2 == -INFINITY || i >= a.Tq) l2 = INFINITY;
    asm volatile("" : "+v"(l2));

    KeyTiles<T, DH, BN, NW, KS> tiles(a, wk, n, hk, smem, table, wave, lane);
    tiles.begin();
    f32x16 acc[L::ND], mean[EXACT ? L::ND : 1];
    float off = 0.f;
#pragma unroll
    for (int d = 0; d < L::ND; ++d) acc[d] = zero16();
#pragma unroll
    for (int d = 0; d < (EXACT ? L::ND : 1); ++d) mean[d] = zero16();
    for (int t0 = 0; t0 < wk.nt; t0 += KS) {
        tiles.step(t0);
        const int t = t0 + half;
        if (KS > 1 && t >= wk.nt) break;                      // (the last turn)
        const int j0 = wk.j0(t, BN);
        const char* kt = tiles.at(t);
        const char* vt = kt + TILE;
        const unsigned long long valid = tiles.valid(t);
        unsigned long long bits = ~0ull;
        const bool full = j0 >= in_lo && j0 + BN <= in_hi && valid == below(BN);
        if (!full) bits = visible(sp, j0) & valid;
        if (wave_rows && (full || __any(bits != 0))) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (!full && !__any((unsigned)(bits >> (32 * b)) != 0)) continue;
                dq_block<T, DH, EXACT, L::NF>(kt + L::bytes(32 * b), vt + L::bytes(32 * b), qf, df, nullptr, a.c, l2, delta, (unsigned)(bits >> (32 * b)), full, acc, mean, off, lane);
            }
        }
    }
    if constexpr (KS > 1) {                                   // the halves' sums, one accumulator at a time
        float* const to = (float*)smem + row_wave * L::ND * 16 * 64 + lane;
        auto add = [&](auto& sums, int n) {
            __syncthreads();
            if (half)
#pragma unroll
                for (int d = 0; d < n; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) to[(d * 16 + r) * 64] = sums[d][r];
            __syncthreads();
            if (!half)
#pragma unroll
                for (int d = 0; d < n; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sums[d][r] += to[(d * 16 + r) * 64];
        };
        add(acc, L::ND);
        if constexpr (EXACT) {
            add(mean, L::ND);
            __syncthreads();
            if (half) *to = off;
            __syncthreads();
            if (!half) off += *to;
        }
        if (half) return;
    }
    if constexpr (EXACT) delta += exactly(acc, mean, off);
    if (wave_rows) a.stats[stats_at(a, n, h, i0) + lane] = hi ? (i < a.Tq ? delta : 0.f) : l2;
    if (i < a.Tq) store_row<T, DH>(acc, a.scale, (T*)a.dq + n * a.sdq.n + i * a.sdq.t + h * a.sdq.h, hi);
}
template <typename T, int DH, int BN, int NW, int KS>
__global__ __launch_bounds__(64 * MOST_WAVES<T>, (RESIDENT<T, DH, 3>)) void win_bwd_dq_kernel(const WinArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ unsigned long long table[2 * MASK_RUN];
    const int bm = (NW ? NW / KS : blockDim.x >> 6) * BQ, nqt = (a.Tq + bm - 1) / bm;
    int item = xcd_item();
    const int g = item % a.G; item /= a.G;
    const int qt = nqt - 1 - item % nqt; item /= nqt;
    const int hk = item % a.Hkv, n = item / a.Hkv, h = hk * a.G + g;
    const Seq sq = sequence(a, n);
    const Span s0 = span_of(a, sq.pos + qt * bm, sq.kvl), s1 = span_of(a, sq.pos + min(qt * bm + bm, a.Tq) - 1, sq.kvl);
    if (BF16<T> && (min(s0.keys(), s1.keys()) <= FEW_KEYS || (a.key_mask && mask_leaves_few(a, n, s0, s1)))) dq_rows<T, DH, BN, NW, KS, BF16<T>>(a, n, hk, h, qt, sq, smem, table);
    else dq_rows<T, DH, BN, NW, KS, false>(a, n, hk, h, qt, sq, smem, table);
}

// ------------------------------------------------------------------------------------------------ backward: dk, dv
// Fragments of a key group's values (in the short kernel below: also of dout's rows) that stay in LDS instead of registers: at 128 wide bf16 rows the accumulators and both operands take all 256 registers
// that two waves a SIMD leave each, and one that was reloaded from scratch memory in every turn made the turn wait for the next stage's DMA, too.
template <typename T, int DH> constexpr int PARKED = sizeof(T) == 2 && DH == 128 ? 4 : 0;
// Four products a block; P and ds are rounded to bf16 in front of theirs.  2 x 4096 rows in windows of 1024, 16 query and 4 key heads of 128: 169 us and 23 us
// for the sinks, 715 TFLOP/s of visible pairs: the accumulators and both operands leave two waves to a SIMD, and a wave of a 2 x 2 workgroup has one block
// between two barriers.  The matrix unit is busy 33 per cent of the CUs' time, LDS reads 23.  (64 wide bf16 rows: 5 registers spilled.)
// A workgroup owns kg groups of 32 keys and walks the queries that see them, 32 qh at a time: wave w takes key group w % kg and query rows 32 (w / kg).
// The qh partial sums of a key group are added through LDS at the end.  A stage holds u of those row groups for each; all queries in one stage, and one
// buffer, where they are few.
// SINK = false: the pairs inside the windows.  SINK = true, launched before it: the pairs of a sink key and a query whose window starts behind it.  Every
// query has those, so their walk is cut into `chunks` that leave fp32 partial sums in the workspace; the window pass adds them to the sink keys' rows
// in a fixed order.  (One workgroup that walks all queries for the sinks' tile alone took 1.9 ms where the window pass takes a tenth of that.)
template <typename T, int DH, bool SINK>
__global__ __launch_bounds__(64 * MOST_WAVES<T>, (RESIDENT<T, DH, 3>)) void win_bwd_dkv_kernel(const WinArgs a, int kg, int qh, int u, int buffers) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5, key_group = wave % kg, row_group = wave / kg, nw = kg * qh;
    const int bn = kg * BQ, groups = qh * u, bq = groups * BQ, tile = groups * L::bytes(BQ), stage = 2 * tile + groups * 256;        // Q, dout, statistics of bq queries
    const int keys = SINK ? a.sink_keys : a.Tk, nkt = (keys + bn - 1) / bn;
    int item = xcd_item();
    int chunk = 0;
    if (SINK) { chunk = item % a.chunks; item /= a.chunks; }
    const int kt = item % nkt; item /= nkt;
    const int hk = item % a.Hkv, n = item / a.Hkv;
    const Seq sq = sequence(a, n);
    const int jb = kt * bn, j = jb + key_group * BQ + (lane & 31), jc = min(j, a.Tk - 1);
    const bool seen = j < min(sq.kvl, keys) && (j >= sq.from || j < a.sinks) && (!a.key_mask || a.key_mask[(size_t)n * a.Tk + jc]);
    // rows of queries whose window holds key jj: [first_row, end_row); the rows behind them see it if it is a sink
    auto first_row = [&](int jj) { return a.right < 0 ? 0 : clampi(jj - a.right - sq.pos, 0, a.Tq); };
    auto end_row = [&](int jj) { return a.left < 0 || jj < a.near_sinks ? a.Tq : clampi(jj + a.left - sq.pos + 1, 0, a.Tq); };
    auto behind = [&](int jj) { return max(first_row(jj), end_row(jj)); };
    const int lo = !seen ? 0 : SINK ? behind(j) : first_row(j), end = !seen ? 0 : SINK ? a.Tq : end_row(j);
    const int last = min(min(jb + bn, keys), sq.kvl) - 1;                     // last key of the tile that exists
    int r0 = 0, r1 = 0;
    if (last >= jb) { r0 = (SINK ? behind(jb) : first_row(jb)) & ~(BQ - 1); r1 = SINK || jb < a.near_sinks ? a.Tq : end_row(last); }
    const int nq = r1 > r0 ? (r1 - r0 + bq - 1) / bq : 0;
    int t0 = 0, t1 = nq * a.G;                                                // tiles of queries, head by head
    if (SINK) { const int per = (t1 + a.chunks - 1) / a.chunks; t0 = min(chunk * per, t1); t1 = min(t0 + per, t1); }

    constexpr int PK = PARKED<T, DH>;
    typename M::Frag kf[L::NF], vf[L::NF - PK];
    char* parked = smem + buffers * stage + key_group * PK * 1024 + lane * 16;
    {
        const char* pk = (const char*)((const T*)a.k + n * a.sk.n + jc * a.sk.t + hk * a.sk.h);
        const char* pv = (const char*)((const T*)a.v + n * a.sv.n + jc * a.sv.t + hk * a.sv.h);
        const typename M::Frag zero = {};
#pragma unroll
        for (int s = 0; s < L::NF; ++s) {
            kf[s] = seen ? *(const typename M::Frag*)(pk + 32 * s + 16 * hi) : zero;
            const typename M::Frag v = seen ? *(const typename M::Frag*)(pv + 32 * s + 16 * hi) : zero;
            if (s < L::NF - PK) vf[s < L::NF - PK ? s : 0] = v;
            else *(typename M::Frag*)(parked + (s - (L::NF - PK)) * 1024) = v;        // (waves of one key group write the same)
        }
        landed(kf);
        landed(vf);
    }
    const long long qst = a.sq.t * (long long)sizeof(T), dst = a.sdo.t * (long long)sizeof(T);
    const unsigned lds = (unsigned)(uintptr_t)(LDS_PTR(char))smem;
    auto issue = [&](int t, int buf) {
        const int h = hk * a.G + t / nq, i0 = r0 + (t % nq) * bq;
        const unsigned at = lds + buf * stage;
        for (int r = 0; r < groups; ++r) {                                    // 32 rows at a time
            const int ir = i0 + r * BQ;
            if (ir >= a.Tq) break;                                            // (the rows of that group are masked out below)
            const unsigned long long valid = below(a.Tq - ir);
            load_tile<T, DH, BQ, 0>((const char*)((const T*)a.q + n * a.sq.n + h * a.sq.h) + ir * qst, (unsigned)qst, valid, at + r * L::bytes(BQ), wave, nw, lane);
            load_tile<T, DH, BQ, 0>((const char*)((const T*)a.dout + n * a.sdo.n + h * a.sdo.h) + ir * dst, (unsigned)dst, valid, at + tile + r * L::bytes(BQ), wave, nw, lane);
            if (wave == r % nw) dma4((unsigned)lane * 4u, tile_rsrc(a.stats + stats_at(a, n, h, ir)), at + 2 * tile + r * 256);
        }
    };
    f32x16 dk[L::ND], dv[L::ND];
#pragma unroll
    for (int d = 0; d < L::ND; ++d) { dk[d] = zero16(); dv[d] = zero16(); }
    if (t0 < t1) issue(t0, 0);
    for (int t = t0; t < t1; ++t) {
        dma_barrier();
        const int buf = (t - t0) & (buffers - 1);
        if (t + 1 < t1) issue(t + 1, buf ^ 1);
        for (int r = row_group; r < groups; r += qh) {
            const char* qt = smem + buf * stage + r * L::bytes(BQ);
            const char* dt = qt + tile;
            const float* st2 = (const float*)(smem + buf * stage + 2 * tile + r * 256);
            const int i0 = r0 + (t % nq) * bq + r * BQ;
            const unsigned bits = (unsigned)(below(min(end - i0, 32)) & ~below(lo - i0));
            if (!__any(bits != 0)) continue;
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int f = 0; f < L::NF; ++f) {
                s = M::mac(row_frag<T, DH>(qt, f, lane), kf[f], s);
                dp = M::mac(row_frag<T, DH>(dt, f, lane), f < L::NF - PK ? vf[f < L::NF - PK ? f : 0] : *(const typename M::Frag*)(parked + (f - (L::NF - PK)) * 1024), dp);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (!__all(bits == ~0u)) {
                const unsigned w = bits >> (4 * hi);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = (w >> tok(e, 0)) & 1u ? s[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const f32x4 l2 = *(const f32x4*)(st2 + tok(e, hi)), de = *(const f32x4*)(st2 + 32 + tok(e, hi));
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    s[e + x] = __builtin_amdgcn_exp2f(fmaf(s[e + x], a.c, -l2[x]));
                    dp[e + x] = s[e + x] * (dp[e + x] - de[x]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < L::ND; ++d) {
                dv[d] = M::mac_t(M::template turned<DH>(dt, d, lane), M::right(s), dv[d]);
                dk[d] = M::mac_t(M::template turned<DH>(qt, d, lane), M::right(dp), dk[d]);
            }
        }
    }
    if (qh > 1) {                                                             // add the row groups' sums: a lane's 16 ND values lie 64 apart
        auto add = [&](f32x16 (&acc)[L::ND]) {
            float* at = (float*)smem + key_group * 64 * 16 * L::ND + lane;
            const int group = kg * 64 * 16 * L::ND;
            __syncthreads();
            if (row_group > 0)
#pragma unroll
                for (int d = 0; d < L::ND; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) at[(row_group - 1) * group + (d * 16 + r) * 64] = acc[d][r];
            __syncthreads();
            if (row_group == 0)
                for (int g = 0; g + 1 < qh; ++g)
#pragma unroll
                    for (int d = 0; d < L::ND; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[d][r] += at[g * group + (d * 16 + r) * 64];
        };
        add(dk);
        add(dv);
    }
    const bool owner = row_group == 0;                                        // has its key group's sums
    if (SINK) {
        if (owner && j < a.sink_rows) {
            float* o = a.sinks_ws + (((long long)(n * a.Hkv + hk) * a.chunks + chunk) * a.sink_rows + j) * 2 * DH;
#pragma unroll
            for (int d = 0; d < L::ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    *(f32x4*)(o + 32 * d + tok(r, hi)) = f32x4{dk[d][r], dk[d][r + 1], dk[d][r + 2], dk[d][r + 3]};
                    *(f32x4*)(o + DH + 32 * d + tok(r, hi)) = f32x4{dv[d][r], dv[d][r + 1], dv[d][r + 2], dv[d][r + 3]};
                }
        }
        return;
    }
    if (owner && j < a.sink_keys) {
        for (int c = 0; c < a.chunks; ++c) {
            const float* o = a.sinks_ws + (((long long)(n * a.Hkv + hk) * a.chunks + c) * a.sink_rows + j) * 2 * DH;
#pragma unroll
            for (int d = 0; d < L::ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    const f32x4 x = *(const f32x4*)(o + 32 * d + tok(r, hi)), y = *(const f32x4*)(o + DH + 32 * d + tok(r, hi));
#pragma unroll
                    for (int e = 0; e < 4; ++e) { dk[d][r + e] += x[e]; dv[d][r + e] += y[e]; }
                }
        }
    }
    T* ok = (T*)a.dk + n * a.sdk.n + hk * a.sdk.h;
    T* ov = (T*)a.dv + n * a.sdv.n + hk * a.sdv.h;
    if constexpr (WHOLE_ROWS<T, DH>) {
        __syncthreads();                                                      // the stages are done with
        const int j0 = jb + key_group * BQ;
        if (owner && j0 < a.Tk) {
            char* mine = smem + key_group * 32 * OUT_ROW<T, DH>;
            store_rows<T, DH>(mine, dk, a.scale, ok + j0 * a.sdk.t, a.sdk.t, a.Tk - j0, lane);
            store_rows<T, DH>(mine, dv, 1.f, ov + j0 * a.sdv.t, a.sdv.t, a.Tk - j0, lane);
        }
    } else if (owner && j < a.Tk) {
        store_row<T, DH>(dk, a.scale, ok + j * a.sdk.t, hi);
        store_row<T, DH>(dv, 1.f, ov + j * a.sdv.t, hi);
    }
}

// ------------------------------------------------------------------------------------------------ backward of short sequences
// dk / scale and dv += the parts of 32 queries with the statistics st2; bit of `bits`: that query sees the lane's key.  (The dk / dv kernel above has the
// same steps in its loop: as a call of this function its 128 wide form spilled 19 registers there and took a quarter longer.)
template <typename T, int DH>
__device__ __forceinline__ void dkv_block(const char* qt, const char* dt, const float* st2, const typename Mma<T>::Frag (&kf)[Lay<T, DH>::NF],
                                          const typename Mma<T>::Frag (&vf)[Lay<T, DH>::NF - PARKED<T, DH>], const char* parked, float c, unsigned bits, f32x16 (&dk)[DH / 32],
                                          f32x16 (&dv)[DH / 32], int lane) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    constexpr int KEPT = L::NF - PARKED<T, DH>;
    const int hi = lane >> 5;
    f32x16 s = zero16(), dp = zero16();
#pragma unroll
    for (int f = 0; f < L::NF; ++f) {
        s = M::mac(row_frag<T, DH>(qt, f, lane), kf[f], s);
        dp = M::mac(row_frag<T, DH>(dt, f, lane), f < KEPT ? vf[f < KEPT ? f : 0] : *(const typename M::Frag*)(parked + (f - KEPT) * 1024), dp);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (!__all(bits == ~0u)) {
        const unsigned w = bits >> (4 * hi);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = (w >> tok(e, 0)) & 1u ? s[e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
        const f32x4 l2 = *(const f32x4*)(st2 + tok(e, hi)), de = *(const f32x4*)(st2 + 32 + tok(e, hi));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            s[e + x] = __builtin_amdgcn_exp2f(fmaf(s[e + x], c, -l2[x]));
            dp[e + x] = s[e + x] * (dp[e + x] - de[x]);
        }
    }
    const typename M::Right ps = M::right(s), pd = M::right(dp);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < L::ND; ++d) {
        dv[d] = M::mac_t(M::template turned<DH>(dt, d, lane), ps, dv[d]);
        dk[d] = M::mac_t(M::template turned<DH>(qt, d, lane), pd, dk[d]);
    }
}
// One workgroup has a head's queries and keys whole, wave w queries 32 w.. and keys 32 w.., and reads them once: keys and values lie in LDS and the wave's
// query rows in registers for dq; then they change places, and dk and dv follow without another read.  256 x 12 heads of 130 x 64 in bf16: 160 us (8 less
// without the exact delta), the two kernels 202; 8 tensors of 51 MB at 2.6 TB/s, where moving them alone would take 90 us: of 130 rows the fifth wave's 30
// are padding, and two workgroups of five waves share a CU (bounded to 128 registers, for three, it spilled 23 and was 17 us slower).
template <typename T, int DH>
__global__ __launch_bounds__(64 * MOST_WAVES<T>, (RESIDENT<T, DH, 3>)) void win_bwd_short_kernel(const WinArgs a) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    constexpr int TILE = L::bytes(BQ), PK = PARKED<T, DH>;
    extern __shared__ __attribute__((aligned(16))) char smem[];               // of every wave: two tiles, 64 statistics, parked values
    __shared__ unsigned words[MOST_WAVES<T>];                                 // the keys that exist
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5, row = lane & 31, nw = blockDim.x >> 6;
    const int item = xcd_item(), h = item % a.H, n = item / a.H;
    const Seq sq = sequence(a, n);
    const int i0 = wave * BQ, i = i0 + row, ic = min(i, a.Tq - 1);
    char* const mine = smem + wave * 2 * TILE;
    float* const stats = (float*)(smem + nw * 2 * TILE);
    char* const parked = smem + nw * (2 * TILE + 256) + wave * PK * 1024 + lane * 16;
    unsigned valid = 0;
    if (i0 < a.Tk) {
        const unsigned lds = (unsigned)(uintptr_t)(LDS_PTR(char))mine;
        const long long kst = a.sk.t * (long long)sizeof(T), vst = a.sv.t * (long long)sizeof(T);
        valid = (unsigned)(__ballot(mask_byte(a, n, i) != 0) & there(a, sq.kvl, sq.from, i0));
        load_tile<T, DH, BQ, 1>((const char*)((const T*)a.k + n * a.sk.n + h * a.sk.h) + i0 * kst, (unsigned)kst, valid, lds, 0, 1, lane);
        load_tile<T, DH, BQ, 1>((const char*)((const T*)a.v + n * a.sv.n + h * a.sv.h) + i0 * vst, (unsigned)vst, valid, lds + TILE, 0, 1, lane);
    }
    if (lane == 0) words[wave] = valid;
    f32x16 acc[L::ND];
    {
        typename M::Frag qf[L::NF] = {}, df[L::NF - PK] = {}, df_rest[PK ? PK : 1] = {};        // zeros behind the last query: nothing comes of them below
        float delta = 0.f, l2 = INFINITY;
        if (i < a.Tq) {
            const char* p = (const char*)((const T*)a.q + n * a.sq.n + i * a.sq.t + h * a.sq.h);
            const char* pd = (const char*)((const T*)a.dout + n * a.sdo.n + i * a.sdo.t + h * a.sdo.h);
            const char* po = (const char*)((const T*)a.o + n * a.so.n + i * a.so.t + h * a.so.h);
            l2 = a.lse[((long long)n * a.H + h) * a.Tq + i] * LOG2E;
#pragma unroll
            for (int s = 0; s < L::NF; ++s) {
                qf[s] = *(const typename M::Frag*)(p + 32 * s + 16 * hi);
                const typename M::Frag d = *(const typename M::Frag*)(pd + 32 * s + 16 * hi);
                delta += M::dot(d, *(const typename M::Frag*)(po + 32 * s + 16 * hi));
                if (s < L::NF - PK) df[s < L::NF - PK ? s : 0] = d;
                else df_rest[s < L::NF - PK ? 0 : s - (L::NF - PK)] = d;
            }
        }
#pragma unroll
        for (int s = 0; s < PK; ++s) *(typename M::Frag*)(parked + s * 1024) = df_rest[s];
        delta += __shfl_xor(delta, 32, 64);
        if (l2 == -INFINITY) l2 = INFINITY;                                   // the query sees nothing
        dma_barrier();
#pragma unroll
        for (int d = 0; d < L::ND; ++d) acc[d] = zero16();
        float off = 0.f;
        if (i0 < a.Tq) {
            f32x16 mean[BF16<T> ? L::ND : 1];
#pragma unroll
            for (int d = 0; d < (BF16<T> ? L::ND : 1); ++d) mean[d] = zero16();
            const Span sp = span_of(a, sq.pos + ic, sq.kvl);
            const int in_lo = span_of(a, sq.pos + min(i0 + 31, a.Tq - 1), sq.kvl).lo, in_hi = span_of(a, sq.pos + i0, sq.kvl).hi;
            for (int j0 = 0; j0 < a.Tk; j0 += BQ) {
                const unsigned keys = (unsigned)__builtin_amdgcn_readfirstlane((int)words[j0 / BQ]);
                const bool full = j0 >= in_lo && j0 + BQ <= in_hi && keys == ~0u;
                const unsigned bits = full ? ~0u : (unsigned)visible(sp, j0) & keys;
                if (!__any(bits != 0)) continue;
                const char* kt = smem + j0 / BQ * 2 * TILE;
                dq_block<T, DH, BF16<T>, L::NF - PK>(kt, kt + TILE, qf, df, parked, a.c, l2, delta, bits, full, acc, mean, off, lane);
            }
            if constexpr (BF16<T>) delta += exactly(acc, mean, off);
            if (i < a.Tq) store_row<T, DH>(acc, a.scale, (T*)a.dq + n * a.sdq.n + i * a.sdq.t + h * a.sdq.h, hi);
        }
#pragma unroll
        for (int s = 0; s < PK; ++s) df_rest[s] = *(const typename M::Frag*)(parked + s * 1024);
        typename M::Frag kf[L::NF], vf[L::NF - PK];
#pragma unroll
        for (int s = 0; s < L::NF; ++s) {
            kf[s] = row_frag<T, DH>(mine, s, lane);
            const typename M::Frag v = row_frag<T, DH>(mine + TILE, s, lane);
            if (s < L::NF - PK) vf[s < L::NF - PK ? s : 0] = v;
            else *(typename M::Frag*)(parked + (s - (L::NF - PK)) * 1024) = v;
        }
        __syncthreads();                                                      // nobody needs the keys' tiles any more
#pragma unroll
        for (int s = 0; s < L::NF; ++s) {
            *(typename M::Frag*)(mine + L::row_base(lane) + L::step(s)) = qf[s];
            *(typename M::Frag*)(mine + TILE + L::row_base(lane) + L::step(s)) = s < L::NF - PK ? df[s < L::NF - PK ? s : 0] : df_rest[s < L::NF - PK ? 0 : s - (L::NF - PK)];
        }
        stats[wave * 2 * BQ + lane] = hi ? delta : l2;
        __syncthreads();
        if (i0 >= a.Tk) return;
        const bool seen = (valid >> row) & 1u;
        const int lo = !seen || a.right < 0 ? 0 : clampi(i - a.right - sq.pos, 0, a.Tq);         // the queries that see key i: [lo, end)
        const int end = !seen ? 0 : a.left < 0 || i < a.sinks ? a.Tq : clampi(i + a.left - sq.pos + 1, 0, a.Tq);
        f32x16 dv[L::ND];
#pragma unroll
        for (int d = 0; d < L::ND; ++d) { acc[d] = zero16(); dv[d] = zero16(); }
        for (int r = 0; r < a.Tq; r += BQ) {
            const unsigned bits = (unsigned)(below(min(end - r, BQ)) & ~below(lo - r));
            if (!__any(bits != 0)) continue;
            const char* qt = smem + r / BQ * 2 * TILE;
            dkv_block<T, DH>(qt, qt + TILE, stats + 2 * r, kf, vf, parked, a.c, bits, acc, dv, lane);
        }
        if (i < a.Tk) {
            store_row<T, DH>(acc, a.scale, (T*)a.dk + n * a.sdk.n + i * a.sdk.t + h * a.sdk.h, hi);
            store_row<T, DH>(dv, 1.f, (T*)a.dv + n * a.sdv.n + i * a.sdv.t + h * a.sdv.h, hi);
        }
    }
}

// ------------------------------------------------------------------------------------------------ few query rows against many keys
// The G Tq <= 32 rows of one key head as one 32-column tile, the keys in 32-row tiles that the workgroup's waves take in turn, each with its own running
// maximum and sum and its own pair of LDS tiles (no barrier: a wave waits for its own DMA, counted, while the next tile is in flight).  The waves are
// merged through LDS; with `splits` > 1 several workgroups share the keys and win_merge_kernel joins their partial results.  Bound by memory, so P is kept
// as the sum of two bf16 numbers: the second product costs nothing.  One token of 64 sequences, 8 key heads, 4096 of 16384 keys of 128: 1.08 GB in 182 us, 5.9
// TB/s (a copy moves 4.8, half of it writes).
constexpr int FEW = 32;
template <int N> __device__ __forceinline__ void wait_dma() { asm volatile("s_waitcnt vmcnt(%c0)" ::"i"(N) : "memory"); }
template <typename T, int DH> struct Few {
    using L = Lay<T, DH>;
    static constexpr int TILE = L::bytes(FEW), PIECES = 2 * FEW / L::PIECE_ROWS, NW = PIECES <= 16 ? 4 : 2;
    static constexpr int MERGE = NW * FEW * (DH + 2) * 4, STAGES = NW * 4 * TILE, LDS = MERGE > STAGES ? MERGE : STAGES;
};
template <typename T, int DH>
__global__ __launch_bounds__((64 * Few<T, DH>::NW), 1) void win_few_kernel(const WinArgs a, int splits) {
    using L = Lay<T, DH>;
    using M = Mma<T>;
    using F = Few<T, DH>;
    constexpr int NW = F::NW, TILE = F::TILE;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), hi = lane >> 5, r = lane & 31, rows = a.G * a.Tq;
    int item = blockIdx.x;
    const int split = item % splits; item /= splits;
    const int hk = item % a.Hkv, n = item / a.Hkv;
    const Seq sq = sequence(a, n);
    const int rc = min(r, rows - 1), g = rc / a.Tq, i = rc - g * a.Tq, h = hk * a.G + g;
    Walk wk = walk_of(a, sq.pos, sq.pos + a.Tq - 1, sq, FEW);
    Span sp = span_of(a, sq.pos + i, sq.kvl);
    const Span s0 = span_of(a, sq.pos, sq.kvl), s1 = span_of(a, sq.pos + a.Tq - 1, sq.kvl);           // every row sees [s1.lo, s0.hi)
    const int per = (wk.nt + splits - 1) / splits, t0 = min(split * per, wk.nt), t1 = min(t0 + per, wk.nt);

    typename M::Frag qf[L::NF];
    {
        const char* p = (const char*)((const T*)a.q + n * a.sq.n + i * a.sq.t + h * a.sq.h);
#pragma unroll
        for (int s = 0; s < L::NF; ++s) qf[s] = *(const typename M::Frag*)(p + 32 * s + 16 * hi);
        landed(qf);
    }
    const char* kb = (const char*)((const T*)a.k + n * a.sk.n + hk * a.sk.h);
    const char* vb = (const char*)((const T*)a.v + n * a.sv.n + hk * a.sv.h);
    const long long kst = a.sk.t * (long long)sizeof(T), vst = a.sv.t * (long long)sizeof(T);
    char* mine = smem + wave * 4 * TILE;
    const unsigned lds = (unsigned)(uintptr_t)(LDS_PTR(char))mine;
    auto valid_of = [&](int byte, int j0) { return __ballot(byte != 0) & there(a, wk.kvl, wk.from, j0) & below(FEW); };
    auto issue = [&](int j0, unsigned long long valid, int buf) {
        load_tile<T, DH, FEW, 1>(kb + j0 * kst, (unsigned)kst, valid, lds + buf * 2 * TILE, 0, 1, lane);
        load_tile<T, DH, FEW, 1>(vb + j0 * vst, (unsigned)vst, valid, lds + buf * 2 * TILE + TILE, 0, 1, lane);
    };
    f32x16 acc[L::ND];
#pragma unroll
    for (int d = 0; d < L::ND; ++d) acc[d] = zero16();
    float m = -INFINITY, l = 0.f;
    int t = t0 + wave, buf = 0, byte = 1;
    unsigned long long valid = 0, next = 0;
    if (t < t1) {
        valid = valid_of(mask_byte(a, n, wk.j0(t, FEW) + r), wk.j0(t, FEW));
        issue(wk.j0(t, FEW), valid, 0);
        if (t + NW < t1) byte = mask_byte(a, n, wk.j0(t + NW, FEW) + r);
    }
    for (; t < t1; t += NW) {
        const int j0 = wk.j0(t, FEW);
        const bool more = t + NW < t1;
        if (more) {
            next = valid_of(byte, wk.j0(t + NW, FEW));
            if (t + 2 * NW < t1) byte = mask_byte(a, n, wk.j0(t + 2 * NW, FEW) + r);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");       // this wave has read the tile that is refilled
            issue(wk.j0(t + NW, FEW), next, buf ^ 1);
            wait_dma<F::PIECES>();
        } else wait_dma<0>();
        const char* kt = mine + buf * 2 * TILE;
        const char* vt = kt + TILE;
        f32x16 st = zero16();
#pragma unroll
        for (int s = 0; s < L::NF; ++s) st = M::mac(row_frag<T, DH>(kt, s, lane), qf[s], st);
        if (!(j0 >= s1.lo && j0 + FEW <= s0.hi && valid == below(FEW))) {
            const unsigned w = (unsigned)(visible(sp, j0) & valid) >> (4 * hi);
#pragma unroll
            for (int e = 0; e < 16; ++e) st[e] = (w >> tok(e, 0)) & 1u ? st[e] : -INFINITY;
        }
        float mt = st[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mt = fmaxf(mt, st[e]);
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * a.c;
        if (__any(mt > m + 8.f)) {
            const float mn = fmaxf(m, mt), f = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < L::ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[d][e] *= f;
        }
        const float mm = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int e = 0; e < 16; ++e) { st[e] = __builtin_amdgcn_exp2f(fmaf(st[e], a.c, -mm)); l += st[e]; }
#pragma unroll
        for (int d = 0; d < L::ND; ++d) acc[d] = M::mac_t(M::template turned<DH>(vt, d, lane), M::right(st), acc[d]);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int e = 0; e < 16; ++e) st[e] -= bf2f(f2bf(st[e]));
#pragma unroll
            for (int d = 0; d < L::ND; ++d) acc[d] = M::mac_t(M::template turned<DH>(vt, d, lane), M::right(st), acc[d]);
        }
        valid = next;
        buf ^= 1;
    }
    l += __shfl_xor(l, 32, 64);
    __syncthreads();                                                          // the tiles are done with: their LDS takes the waves' results
    float* part = (float*)smem;                                               // [NW][32][DH], then [NW][32] of m and of l
    float* pm = part + NW * FEW * DH;
    float* pl = pm + NW * FEW;
#pragma unroll
    for (int d = 0; d < L::ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            *(f32x4*)(part + (wave * FEW + r) * DH + 4 * (((32 * d + tok(e, hi)) >> 2) ^ (r & 7))) = f32x4{acc[d][e], acc[d][e + 1], acc[d][e + 2], acc[d][e + 3]};
    if (hi == 0) { pm[wave * FEW + r] = m; pl[wave * FEW + r] = l; }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * (DH / 4); e += 64 * NW) {
        const int row = e / (DH / 4), d = e - row * (DH / 4), gg = row / a.Tq, ii = row - gg * a.Tq, hh = hk * a.G + gg;
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, pm[w * FEW + row]);
        const float base = top == -INFINITY ? 0.f : top;
        f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(pm[w * FEW + row] - base);
            total += f * pl[w * FEW + row];
            o = o + *(const f32x4*)(part + (w * FEW + row) * DH + 4 * (d ^ (row & 7))) * f;
        }
        if (splits > 1) {
            const long long at = (((long long)n * a.Hkv + hk) * splits + split) * rows + row;
            *(f32x4*)(a.parts + at * DH + 4 * d) = o;
            if (d == 0) { float* ml = a.parts + (long long)a.N * a.Hkv * splits * rows * DH + 2 * at; ml[0] = top; ml[1] = total; }
        } else {
            const float inv = total == 0.f ? 0.f : 1.f / total;
            M::st4((T*)a.out + n * a.so.n + ii * a.so.t + hh * a.so.h + 4 * d, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
            if (d == 0 && a.lse) a.lse[((long long)n * a.H + hh) * a.Tq + ii] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * LN2;
        }
    }
}
// one row per wave: the splits' partial results into out and lse
template <typename T, int DH>
__global__ __launch_bounds__(256) void win_merge_kernel(const WinArgs a, int splits) {
    const int lane = threadIdx.x & 63, rows = a.G * a.Tq;
    const long long units = (long long)a.N * a.Hkv, at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= units * rows) return;
    const long long unit = at / rows;
    const int row = (int)(at - unit * rows), g = row / a.Tq, i = row - g * a.Tq, n = (int)(unit / a.Hkv), h = (int)(unit % a.Hkv) * a.G + g;
    const float* ml = a.parts + units * splits * rows * DH;
    float top = -INFINITY, total = 0.f, o[DH / 64];
    for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[2 * ((unit * splits + s) * rows + row)]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int e = 0; e < DH / 64; ++e) o[e] = 0.f;
    for (int s = 0; s < splits; ++s) {
        const long long k = (unit * splits + s) * rows + row;
        const float f = __builtin_amdgcn_exp2f(ml[2 * k] - base);
        total += f * ml[2 * k + 1];
#pragma unroll
        for (int e = 0; e < DH / 64; ++e) o[e] += f * a.parts[k * DH + 64 * e + lane];
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    T* p = (T*)a.out + n * a.so.n + i * a.so.t + h * a.so.h;
#pragma unroll
    for (int e = 0; e < DH / 64; ++e) Elem<T>::st(p + 64 * e + lane, o[e] * inv);
    if (lane == 0 && a.lse) a.lse[((long long)n * a.H + h) * a.Tq + i] = total == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(total)) * LN2;
}

// ------------------------------------------------------------------------------------------------ host side
// The stride of a dimension of one element is never used, and may be anything.
Strides st(const DicStrides& s, int N, int T, int H) { return Strides{N > 1 ? s.n : 0, T > 1 ? s.t : 0, H > 1 ? s.h : 0}; }
bool fits(const DicStrides& d, int N, int T, int H, int size) {
    // 16-byte rows, and 64 rows of a tile inside a descriptor's 31-bit range
    const Strides s = st(d, N, T, H);
    const int per = 16 / size;
    constexpr long long MOST = 1ll << 52;                        // elements that a dimension spans (what the sums of offsets are sure to hold)
    return s.n % per == 0 && s.t % per == 0 && s.h % per == 0 && s.n >= 0 && s.t >= 0 && s.h >= 0 && s.t <= (1ll << 24) / size
           && s.n <= MOST / (N > 0 ? N : 1) && s.h <= MOST / (H > 0 ? H : 1);
}
bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// The bytes of an argument: rows of w at p + v_0 s_0 + v_1 s_1 + v_2 s_2 with 0 <= v_i < n_i (as far as n_i > 1).
struct Area { const char* p; long long s[3], n[3], w; };
struct Term { long long s, lo, hi; };                            // v s with lo <= v <= hi, s > 0
enum { NO = 0, YES = 1, UNTOLD = 2 };
// Can a sum of the terms, sorted by falling s, lie in [from, to]?  Depth first, over the values that the smaller terms can still make up for: where a stride
// spans what lies inside of it, one to three for each term.  Interleaved layouts of other orders take more, and are given up on after `steps` sums.
int reaches(const Term* t, int count, long long from, long long to, int& steps) {
    if (count == 0) return from <= 0 && to >= 0 ? YES : NO;
    long long lo = 0, hi = 0;                                    // of the terms behind this one
    for (int i = 1; i < count; ++i) { lo += t[i].lo * t[i].s; hi += t[i].hi * t[i].s; }
    auto down = [](long long a, long long b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
    const long long v0 = -down(hi - from, t->s), v1 = down(to - lo, t->s);
    for (long long v = v0 > t->lo ? v0 : t->lo; v <= (v1 < t->hi ? v1 : t->hi); ++v) {
        if (--steps < 0) return UNTOLD;
        if (int r = reaches(t + 1, count - 1, from - v * t->s, to - v * t->s, steps)) return r;
    }
    return NO;
}
long long extent(const Area& a) { return (a.n[0] - 1) * a.s[0] + (a.n[1] - 1) * a.s[1] + (a.n[2] - 1) * a.s[2] + a.w; }
int overlap(const Area& a, const Area& b) {
    if (!a.p || !b.p || a.n[0] * a.n[1] * a.n[2] * a.w == 0 || b.n[0] * b.n[1] * b.n[2] * b.w == 0) return NO;
    if (a.p + extent(a) <= b.p || b.p + extent(b) <= a.p) return NO;
    Term t[6];
    int count = 0;
    auto add = [&](long long s, long long lo, long long hi) {
        if (s == 0 || lo == hi) return;
        int i = 0;
        while (i < count && t[i].s > s) ++i;
        if (i < count && t[i].s == s) { t[i].lo += lo; t[i].hi += hi; return; }
        for (int k = count++; k > i; --k) t[k] = t[k - 1];
        t[i] = Term{s, lo, hi};
    };
    for (int i = 0; i < 3; ++i) { add(a.s[i], 0, a.n[i] - 1); add(b.s[i], 1 - b.n[i], 0); }
    // a row of a begins less than b.w behind and less than a.w in front of one of b
    const long long d = b.p - a.p;
    int steps = 1 << 16;
    return reaches(t, count, d - a.w + 1, d + b.w - 1, steps);
}
// Are an output's rows of dh elements apart from each other?
bool apart(const DicStrides& d, int N, int T, int H, int dh) {
    if (N == 0 || T == 0 || H == 0) return true;
    const long long s[3] = {d.n, d.t, d.h}, n[3] = {N, T, H};
    Term t[3];
    int count = 0;
    for (int i = 0; i < 3; ++i) {
        if (n[i] <= 1) continue;
        int k = count++;
        for (; k > 0 && t[k - 1].s < s[i]; --k) t[k] = t[k - 1];
        t[k] = Term{s[i], 1 - n[i], n[i] - 1};
        if (s[i] < dh || (k > 0 && t[k - 1].s == s[i])) return false;
    }
    for (int i = 0; i < count; ++i) {                            // two rows that differ in t[i] first: either way round, so forwards
        long long inside = dh;
        for (int k = i + 1; k < count; ++k) inside += t[k].hi * t[k].s;
        int steps = 1 << 16;
        t[i].lo = 1;
        if (t[i].s < inside && reaches(t + i, count - i, 1 - dh, dh - 1, steps) != NO) return false;
        t[i].lo = -t[i].hi;
    }
    return true;
}
int check_areas(const DicWinAttnParams* p, int size, bool bwd, size_t ws) {
    auto rows = [&](const void* at, const DicStrides& d, int T, int H) {
        const Strides s = st(d, p->N, T, H);
        return Area{(const char*)at, {s.n * size, s.t * size, s.h * size}, {p->N, T, H}, (long long)p->dh * size};
    };
    auto flat = [](const void* at, long long bytes) { return Area{(const char*)at, {0, 0, 0}, {1, 1, 1}, bytes}; };
    const Area q = rows(p->q, p->q_stride, p->Tq, p->H), k = rows(p->k, p->k_stride, p->Tk, p->Hkv), v = rows(p->v, p->v_stride, p->Tk, p->Hkv);
    const Area out = rows(p->out, p->out_stride, p->Tq, p->H), lse = flat(p->lse, 4ll * p->N * p->H * p->Tq), work = flat(p->ws, (long long)ws);
    const Area mask = flat(p->key_mask, (long long)p->N * p->Tk), len = flat(p->kv_len, 4ll * p->N), pos = flat(p->q_pos, 4ll * p->N);
    Area in[8] = {q, k, v, mask, len, pos}, written[4] = {out, lse, work};
    int ni = 6, nw = 3;
    if (bwd) {
        in[ni++] = out; in[ni++] = lse;
        written[0] = work;
        written[1] = rows(p->dq, p->dq_stride, p->Tq, p->H); written[2] = rows(p->dk, p->dk_stride, p->Tk, p->Hkv); written[3] = rows(p->dv, p->dv_stride, p->Tk, p->Hkv);
        nw = 4;
    }
    const Area dout = rows(bwd ? p->dout : nullptr, p->dout_stride, p->Tq, p->H);
    auto apart = [](int r) {
        DIC_REQUIRE(r != YES, "dic_win_attn: an output overlaps an input or another output");
        DIC_REQUIRE(r == NO, "dic_win_attn: an output and an input or another output share memory with strides that leave open whether they overlap");
        return 0;
    };
    for (int i = 0; i < nw; ++i) {
        for (int j = 0; j < ni; ++j) if (int rc = apart(overlap(written[i], in[j]))) return rc;
        if (int rc = apart(overlap(written[i], dout))) return rc;
        for (int j = 0; j < i; ++j) if (int rc = apart(overlap(written[i], written[j]))) return rc;
    }
    return 0;
}

int check(int dtype, const DicWinAttnParams* p, bool bwd, bool pointers = true) {
    DIC_REQUIRE(p != nullptr, "dic_win_attn: no parameters");
    DIC_REQUIRE(dtype == DIC_F32 || dtype == DIC_BF16, "dic_win_attn: dtype must be DIC_F32 or DIC_BF16");
    const int size = dtype == DIC_BF16 ? 2 : 4;
    DIC_REQUIRE(p->dh == 64 || p->dh == 128, "dic_win_attn: head dim must be 64 or 128");
    DIC_REQUIRE(p->N >= 0 && p->Tq >= 0 && p->Tk >= 0 && p->Tq <= (1 << 28) && p->Tk <= (1 << 28), "dic_win_attn: sizes out of range");
    DIC_REQUIRE(p->H > 0 && p->Hkv > 0 && p->H % p->Hkv == 0, "dic_win_attn: the number of heads must be a multiple of the number of key heads");
    DIC_REQUIRE(p->sinks >= 0 && std::isfinite(p->scale * LOG2E) && p->scale > 0.f, "dic_win_attn: sinks >= 0 and a positive scale, finite times log2(e), are needed");
    const long long heads = (long long)p->N * p->H, most = 1ll << 31;          // (heads >= N Hkv; bounded by itself first, as three factors may pass 64 bits)
    DIC_REQUIRE(heads < most && heads * (p->Tq / 32 + 1) < most && (long long)p->N * p->Hkv * (p->Tk / 32 + 1) < most, "dic_win_attn: too many tiles for one launch");
    if (!pointers) return 0;
    const bool nq = p->N && p->Tq, nk = p->N && p->Tk;
    DIC_REQUIRE(!nq || (p->q && (bwd ? p->out && p->lse && p->dout && p->dq : p->out != nullptr)), "dic_win_attn: null query-side pointer");
    DIC_REQUIRE(!nk || (p->k && p->v && (!bwd || (p->dk && p->dv))), "dic_win_attn: null key-side pointer");
    DIC_REQUIRE(aligned(p->q) && aligned(p->k) && aligned(p->v) && aligned(p->out) && (!bwd || (aligned(p->dout) && aligned(p->dq) && aligned(p->dk) && aligned(p->dv))),
                "dic_win_attn: pointers must be 16-byte aligned");
    auto rows_q = [&](const DicStrides& d) { return fits(d, p->N, p->Tq, p->H, size); };
    auto rows_k = [&](const DicStrides& d) { return fits(d, p->N, p->Tk, p->Hkv, size); };
    DIC_REQUIRE((!nq || (rows_q(p->q_stride) && rows_q(p->out_stride) && (!bwd || (rows_q(p->dout_stride) && rows_q(p->dq_stride)))))
                && (!nk || (rows_k(p->k_stride) && rows_k(p->v_stride) && (!bwd || (rows_k(p->dk_stride) && rows_k(p->dv_stride))))),
                "dic_win_attn: strides must be non-negative multiples of 16 bytes, and a token stride at most 16 MiB");
    const void *in[5] = {p->q, p->k, p->v, bwd ? p->out : nullptr, bwd ? p->dout : nullptr}, *written[3] = {bwd ? p->dq : p->out, bwd ? p->dk : nullptr, bwd ? p->dv : nullptr};
    for (int i = 0; i < 3; ++i) {
        for (const void* x : in) DIC_REQUIRE(!written[i] || written[i] != x, "dic_win_attn: an output in place of an input");
        DIC_REQUIRE(!written[i] || (written[i] != written[(i + 1) % 3]), "dic_win_attn: two outputs in one place");
    }
    DIC_REQUIRE(bwd ? apart(p->dq_stride, p->N, p->Tq, p->H, p->dh) && apart(p->dk_stride, p->N, p->Tk, p->Hkv, p->dh) && apart(p->dv_stride, p->N, p->Tk, p->Hkv, p->dh)
                    : apart(p->out_stride, p->N, p->Tq, p->H, p->dh), "dic_win_attn: rows of an output overlap");
    return 0;
}
// The dk / dv kernel's workgroup: kg groups of 32 keys and qh groups of 32 query rows.  All keys where they are few and the heads many (600 key heads of 200
// x 128: 242 us, cut in two 270); else four waves, as 4 x 1, 2 x 2 or 1 x 4 as there are workgroups for two, or most of one, on every CU: whole backward passes
// of 128 wide rows, 4 x 2048 rows, 16 query and 4 key heads: 589 / 527 us with 256 / 512 workgroups of 4 x 1 / 2 x 2; 1 x 2048, 12 heads: 197 / 181 / 245 with
// 192 / 384 / 768; 2 x 700, 8 heads: 63 / 55 / 71 with 96 / 176 / 352; 1 x 700, 8 heads: 52 / 47 for 2 x 2 / 1 x 4 with 88 / 176.
struct Shape { int kg, qh; };
Shape shape_of(const WinArgs& a, int waves, int most, int most_rows) {
    const int tiles = (a.Tk + BQ - 1) / BQ;
    const long long heads = (long long)a.N * a.Hkv;
    if (tiles <= most && heads >= 256) return {tiles, 1};
    int kg = waves;
    while (kg > 1 && heads * ((tiles + kg - 1) / kg) < (kg > 2 ? 512 : 160) && waves / kg < most_rows) kg >>= 1;
    return {kg, waves / kg};
}
// Row groups at most: with 2, the stages of fp32 rows of 256 bytes let two workgroups share a CU (4 x 513 rows, 12 heads: 75 us, with 4 87), and those of 512
// bytes fit at all.
template <typename T, int DH> constexpr int ROW_GROUPS = sizeof(T) == 2 ? 4 : 2;
// Pieces of the sink pass: about 256 workgroups, and no more than 16 partial sums for the window pass to add.
void plan_sinks(WinArgs& a) {
    a.near_sinks = a.left >= 0 ? (a.sinks < a.Tk ? a.sinks : a.Tk) : 0;
    // The sinks' tile walks Tq rows, another one about left + right + 128 of them: it needs no pass of its own while the card has as much else to do
    // (130 rows in windows of 129, 256 x 12 heads, before other steps: that pass took 43 us beside the window pass of 150).
    const long long others = a.right < 0 ? a.Tq : (long long)a.left + a.right + 128, all = (long long)a.N * a.Hkv * ((a.Tk + 127) / 128) * (others < a.Tq ? others : a.Tq);
    if (a.near_sinks > 0 && a.Tq > 2 * others && a.Tq > all / 256) { a.sink_keys = a.near_sinks; a.near_sinks = 0; }
    a.sink_rows = (a.sink_keys + BQ - 1) / BQ * BQ;
    const long long tiles = (long long)a.N * a.Hkv * (a.sink_rows / BQ), most = (long long)a.G * ((a.Tq + 4 * BQ - 1) / (4 * BQ));
    const long long want = tiles ? (256 + tiles - 1) / tiles : 1;
    a.chunks = (int)(want < most ? want : most);
    if (a.chunks > 16) a.chunks = 16;
    if (a.chunks < 1) a.chunks = 1;
}
long long sink_floats(const WinArgs& a, int dh) { return (long long)a.N * a.Hkv * a.chunks * a.sink_rows * 2 * dh; }
// Few query rows: one workgroup per key head and sequence, or several that share the keys while that fills the card and leaves each 8 tiles to read.  One token,
// 32 query and 8 key heads of 128: 64 sequences of 1000 keys 44 us, a wave for each query head's tile 114, of 128 keys 11 and 29; one sequence of 16384 keys
// 43 us in 64 pieces, 173 in one workgroup a head.
bool few_rows(const WinArgs& a) { return a.G * (long long)a.Tq <= FEW && a.Tk > 64; }
// Keys that the rows of one key head see together when they are few, at most (where the host can tell: no lengths, no masks).
long long span_keys(const WinArgs& a) {
    const long long seen = a.left < 0 || a.right < 0 ? a.Tk : (long long)a.left + a.right + 1 + (a.sinks < a.Tk ? a.sinks : a.Tk);
    return seen < a.Tk ? seen : a.Tk;
}
int splits_of(const WinArgs& a) {
    const long long seen = span_keys(a) + a.Tq + 2 * FEW;
    const long long tiles = ((seen < a.Tk ? seen : a.Tk) + FEW - 1) / FEW, units = (long long)a.N * a.Hkv, want = (512 + units - 1) / units, most = tiles / 8;
    const long long s = want < most ? want : most;
    return s > 1 ? (int)s : 1;
}
long long parts_floats(const WinArgs& a, int dh) {
    const int s = few_rows(a) ? splits_of(a) : 1;
    return s > 1 ? (long long)a.N * a.Hkv * s * a.G * a.Tq * (dh + 2) : 0;
}
size_t ws_bytes(const WinArgs& a, int dh, bool backward) {
    if (!backward) return (size_t)parts_floats(a, dh) * sizeof(float);
    return (size_t)(stats_floats(a.N, a.H, a.Tq) + sink_floats(a, dh)) * sizeof(float);
}

WinArgs args_of(const DicWinAttnParams* p) {
    WinArgs a{};
    a.q = p->q; a.k = p->k; a.v = p->v; a.o = p->out; a.out = p->out; a.dout = p->dout;
    a.dq = p->dq; a.dk = p->dk; a.dv = p->dv; a.lse = p->lse;
    auto rows_q = [&](const DicStrides& d) { return st(d, p->N, p->Tq, p->H); };
    auto rows_k = [&](const DicStrides& d) { return st(d, p->N, p->Tk, p->Hkv); };
    a.sq = rows_q(p->q_stride); a.sk = rows_k(p->k_stride); a.sv = rows_k(p->v_stride); a.so = rows_q(p->out_stride);
    a.sdo = rows_q(p->dout_stride); a.sdq = rows_q(p->dq_stride); a.sdk = rows_k(p->dk_stride); a.sdv = rows_k(p->dv_stride);
    a.key_mask = p->key_mask; a.kv_len = p->kv_len; a.q_pos = p->q_pos;
    a.N = p->N; a.Tq = p->Tq; a.Tk = p->Tk; a.H = p->H; a.Hkv = p->Hkv; a.G = p->H / p->Hkv;
    a.left = p->left < 0 ? -1 : (p->left < FAR ? p->left : FAR);
    a.right = p->right < 0 ? -1 : (p->right < FAR ? p->right : FAR);
    a.sinks = p->sinks; a.scale = p->scale; a.c = p->scale * LOG2E;
    plan_sinks(a);
    return a;
}
constexpr int MOST_LDS = 150 << 10;                              // of a workgroup, beside what kernels hold under a name
// A call goes through its launches twice: once to see that each can be made (a grid holds less than 2^32 threads), so that none runs in front of one that cannot.
struct Where { hipStream_t st; bool look; };
template <auto KERNEL, typename... More> int launch(long long blocks, int threads, size_t lds, Where w, More... more) {
    if (w.look) {
        DIC_REQUIRE(blocks < (1ll << 31) && blocks * threads < (1ll << 32), "dic_win_attn: too many workgroups for one launch");
        return 0;
    }
    if (lds > (64 << 10)) {                     // once for each device: the attribute belongs to its copy of the kernel
        static std::atomic<unsigned long long> allowed{0};
        int dev = 0;
        hipError_t e = hipGetDevice(&dev);
        if (e == hipSuccess && !((allowed.load(std::memory_order_relaxed) >> (dev & 63)) & 1)) {
            e = hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, MOST_LDS);
            if (e == hipSuccess) allowed.fetch_or(1ull << (dev & 63), std::memory_order_relaxed);
        }
        if (e != hipSuccess) { dic_set_error(hipGetErrorString(e)); return (int)e; }
    }
    hipLaunchKernelGGL(KERNEL, dim3((unsigned)blocks), dim3(threads), lds, w.st, more...);
    DIC_CHECK_LAUNCH();
    return 0;
}
// With that few workgroups of 128 rows (a CU has one at most, a SIMD one wave) a workgroup takes 64 rows instead, and its wave pairs share the keys of 32: one
// text of 4096 rows read from left to right, 8 heads of 128, forward: 72 us for 142, backward 240 for 292; 4 x 513 rows in windows of 257, 12 heads, fp32: 30
// for 37 and 96 for 104.  With 512 workgroups, 128 wide, it fills the LDS of a CU by itself: 54 us for 33 (2 x 2048 rows, windows of 501, 16 heads).
constexpr long long SPLIT = 256;
constexpr size_t SHARED_CU_LDS = 75 << 10;                       // two workgroups fit a CU's 160 KB
// The workgroups of a kernel that walks the keys.  Few keys: all of them in LDS at once (unless that keeps a second workgroup off the CU) and the query rows
// of a sequence in one workgroup where they fit (130 rows x 130 keys x 12 heads x 256 sequences, forward, before its other steps: 5 waves 86 us, 4 waves and a second workgroup 113).
template <typename T, int DH, int BN, typename F> int over_keys(const WinArgs& a, F&& go) {
    constexpr int MOST = MOST_WAVES<T>;
    const int rows = (a.Tq + BQ - 1) / BQ, tiles = (a.Tk + BN - 1) / BN;
    const size_t all = (size_t)tiles * 2 * Lay<T, DH>::bytes(BN);
    const bool few = tiles <= FEW_TILES && all <= SHARED_CU_LDS;
    const int waves = few && rows <= MOST ? rows : 4;
    const long long heads = (long long)a.N * a.H, blocks = heads * ((rows + waves - 1) / waves);
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    if (few) return go(std::integral_constant<int, 0>(), one, waves, blocks, all);
    constexpr std::integral_constant<int, 4> four;
    const size_t turns = (size_t)4 * Lay<T, DH>::bytes(BN), sums = (size_t)2 * (DH / 2 + 2) * 256;
    if (blocks <= SPLIT) return go(four, two, 4, heads * ((rows + 1) / 2), 2 * turns > sums ? 2 * turns : sums);
    return go(four, one, 4, blocks, turns);
}
template <typename T, int DH> int fwd(const WinArgs& a, Where w) {
    constexpr int BN = sizeof(T) == 2 ? 64 : 32;
    if (few_rows(a)) {
        const int splits = splits_of(a);
        if (int rc = launch<win_few_kernel<T, DH>>((long long)a.N * a.Hkv * splits, 64 * Few<T, DH>::NW, Few<T, DH>::LDS, w, a, splits)) return rc;
        return splits > 1 ? launch<win_merge_kernel<T, DH>>(((long long)a.N * a.H * a.Tq + 3) / 4, 256, 0, w, a, splits) : 0;
    }
    // 128 wide rows that see many keys: tiles of 32, which take the registers and LDS of three workgroups a CU instead of two (one text of 8192 rows, 4096 keys
    // each, 16 heads: 249 us against 277; rows of 1024 keys, 2 x 4096 rows: 104 us against 96)
    if constexpr (sizeof(T) == 2 && DH == 128)
        if (span_keys(a) >= 2048 && (long long)a.N * a.H * ((a.Tq + 4 * BQ - 1) / (4 * BQ)) > SPLIT)
            return launch<win_fwd_kernel<T, DH, 32, 4, 1>>((long long)a.N * a.H * ((a.Tq + 4 * BQ - 1) / (4 * BQ)), 256, 
                          (size_t)4 * Lay<T, DH>::bytes(32), w, a);
    return over_keys<T, DH, BN>(a, [&](auto nw, auto ks, int waves, long long blocks, size_t lds) { return launch<win_fwd_kernel<T, DH, BN, decltype(nw)::value, decltype(ks)::value>>(blocks, 64 * waves, lds, w, a); });
}
template <typename T, int DH> size_t dkv_lds(int kg, int qh, int u, int buffers) {
    const size_t stages = (size_t)buffers * qh * u * (2 * Lay<T, DH>::bytes(BQ) + 256) + kg * PARKED<T, DH> * 1024, sums = (size_t)(qh - 1) * kg * BQ * DH * sizeof(float);
    const size_t out = WHOLE_ROWS<T, DH> ? (size_t)kg * 32 * OUT_ROW<T, DH> : 0, most = stages > sums ? stages : sums;
    return most > out ? most : out;
}
template <typename T, int DH> int bwd(const WinArgs& a, Where w) {
    constexpr int BN = sizeof(T) == 2 ? 64 : 32;
    const int waves = ((a.Tq > a.Tk ? a.Tq : a.Tk) + BQ - 1) / BQ;
    const size_t whole = (size_t)waves * (2 * Lay<T, DH>::bytes(BQ) + 256 + PARKED<T, DH> * 1024);
    // A head to a workgroup where there is one for every CU (128 wide bf16 rows, 1024 heads of 146: 137 us against 157 in two passes; 32 heads of 224: 33 against
    // 28; fp32, 768 heads of 128 x 64: 116 against 142, 24 heads: 39 against 34), and always for rows of 128 bytes, of which a wave holds and multiplies the
    // least (256 x 12 heads of 130: 168 against 202 us; 12 heads of 146: 16 against 19, of 256: 23.5 against 23).
    if (a.G == 1 && a.Tq > 0 && a.Tk > 0 && waves <= MOST_WAVES<T> && whole <= MOST_LDS && ((long long)a.N * a.H >= 256 || Lay<T, DH>::ROWB == 128))
        return launch<win_bwd_short_kernel<T, DH>>((long long)a.N * a.H, 64 * waves, whole, w, a);
    if (a.Tq > 0)
        if (int rc = over_keys<T, DH, BN>(a, [&](auto nw, auto ks, int waves, long long blocks, size_t lds) { return launch<win_bwd_dq_kernel<T, DH, BN, decltype(nw)::value, decltype(ks)::value>>(blocks, 64 * waves, lds, w, a); }))
            return rc;
    if (a.Tk == 0) return 0;
    if (a.sink_keys > 0)
        if (int rc = launch<win_bwd_dkv_kernel<T, DH, true>>((long long)a.N * a.Hkv * (a.sink_rows / BQ) * a.chunks, 64 * ROW_GROUPS<T, DH>,
                            dkv_lds<T, DH>(1, ROW_GROUPS<T, DH>, 1, 2), w, a, 1, ROW_GROUPS<T, DH>, 1, 2)) return rc;
    constexpr int WAVES = 4;
    const Shape s = shape_of(a, WAVES, MOST_WAVES<T>, ROW_GROUPS<T, DH>);
    // all queries in one stage where they take no more LDS than lets two workgroups share a CU; else as many to a stage (barriers) as two buffers hold
    const int all = s.qh == 1 && a.G == 1 ? (a.Tq + BQ - 1) / BQ : 0;
    int u = WAVES / 2 / s.qh > 1 ? WAVES / 2 / s.qh : 1, buffers = 2;
    if (all > 0 && dkv_lds<T, DH>(s.kg, 1, all, 1) <= SHARED_CU_LDS) { u = all; buffers = 1; }
    return launch<win_bwd_dkv_kernel<T, DH, false>>((long long)a.N * a.Hkv * ((a.Tk + s.kg * BQ - 1) / (s.kg * BQ)), 64 * s.kg * s.qh, dkv_lds<T, DH>(s.kg, s.qh, u, buffers), w, a,
                  s.kg, s.qh, u, buffers);
}
int fwd(int dtype, int dh, const WinArgs& a, Where w) {
    if (dtype == DIC_BF16) return dh == 64 ? fwd<bf16_t, 64>(a, w) : fwd<bf16_t, 128>(a, w);
    return dh == 64 ? fwd<float, 64>(a, w) : fwd<float, 128>(a, w);
}
int bwd(int dtype, int dh, const WinArgs& a, Where w) {
    if (dtype == DIC_BF16) return dh == 64 ? bwd<bf16_t, 64>(a, w) : bwd<bf16_t, 128>(a, w);
    return dh == 64 ? bwd<float, 64>(a, w) : bwd<float, 128>(a, w);
}
}  // namespace

extern "C" size_t dic_win_attn_ws_bytes(int dtype, int backward, const DicWinAttnParams* p) {
    if (check(dtype, p, false, false)) return 0;
    return ws_bytes(args_of(p), p->dh, backward != 0);
}

extern "C" int dic_win_attn_fwd(int dtype, const DicWinAttnParams* p, void* stream) {
    if (int rc = check(dtype, p, false)) return rc;
    if (p->N == 0 || p->Tq == 0) return 0;
    WinArgs a = args_of(p);
    if (int rc = fwd(dtype, p->dh, a, Where{nullptr, true})) return rc;
    const size_t need = ws_bytes(a, p->dh, false);
    if (int rc = check_areas(p, dtype == DIC_BF16 ? 2 : 4, false, need)) return rc;
    DIC_REQUIRE(need == 0 || (p->ws && aligned(p->ws) && p->ws_bytes >= need), "dic_win_attn_fwd: workspace missing or too small (dic_win_attn_ws_bytes)");
    a.parts = (float*)p->ws;
    return fwd(dtype, p->dh, a, Where{(hipStream_t)stream, false});
}

extern "C" int dic_win_attn_bwd(int dtype, const DicWinAttnParams* p, void* stream) {
    if (int rc = check(dtype, p, true)) return rc;
    if (p->N == 0) return 0;
    WinArgs a = args_of(p);
    if (int rc = bwd(dtype, p->dh, a, Where{nullptr, true})) return rc;
    const size_t need = ws_bytes(a, p->dh, true);
    if (int rc = check_areas(p, dtype == DIC_BF16 ? 2 : 4, true, need)) return rc;
    DIC_REQUIRE(need == 0 || (p->ws && aligned(p->ws) && p->ws_bytes >= need), "dic_win_attn_bwd: workspace missing or too small (dic_win_attn_ws_bytes)");
    a.stats = (float*)p->ws;
    a.sinks_ws = a.stats + stats_floats(p->N, p->H, p->Tq);
    return bwd(dtype, p->dh, a, Where{(hipStream_t)stream, false});
}
