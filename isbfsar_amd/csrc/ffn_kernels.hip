// Gated feed-forward block y = (act(x Wg^T + bg) o (x Wu^T + bu)) Wd^T + bd and its gradients.
//
// One matrix-product kernel carries all of it: C[m][n] = sum_k A(m, k) B(n, k), 16-bit operands, f32 sums, each operand either with k
// contiguous (layout 0: LDS rows are m or n, fragments are 16-byte reads) or with m / n contiguous (layout 1: LDS rows are k, fragments
// are transposing reads), so no operand is ever transposed in memory. The product is formed transposed (accumulator rows = n), so a lane
// owns four neighbouring n of one m. The epilogues:
//   GATE  both projections at once: every wave holds the gate and the up columns of the same features; h = act(g) o u (g, u kept in f32
//         for the backward pass: rounded to 16 bits they would put a second rounding into every gradient);
//   OUT   + bias, rounded (or the f32 partial sums of a split of k);
//   DH    dh stays in registers: dG = dh o u o act'(g) and dU = dh o act(g) are what is stored.
#include <algorithm>
#include <cmath>

#include "blocks.h"

namespace isb {
namespace {

enum { EPI_GATE = 0, EPI_OUT = 1, EPI_DH = 2 };
enum { FFN_SILU = 0, FFN_GELU = 1, FFN_RELU = 2, FFN_SIGMOID = 3 };
constexpr int BK = 64, KS = BK / 16;     // k per tile, its steps

struct MmArgs {
    const uint16_t *A, *B, *B2;          // B2: GATE: the up weights; else the operand of the second k segment
    int64_t lda, ldb;
    int M, N, K;                         // GATE: N = 2 F (32 gate columns, 32 up columns, ...)
    int nseg;                            // segments of K (A continues at column K)
    int splits, kt_per_split;
    const uint16_t *bias, *bias2;
    uint16_t* C;
    int64_t ldc;
    float *g, *u;                        // GATE: saved (or null); DH: read
    float* part;                         // OUT with splits > 1: [split][M][N]
    float* cs;                           // DH: column sums of dG | dU over 32 rows, [ceil(M / 32)][2 F], or null
    int8_t* ex;                          // fp16 (Powers): exponents of h (GATE), of dG | dU (DH)
    uint16_t* h;                         // fp16, DH: the saved h, for dWd, and its exponents
    int8_t* ex_h;
    const int8_t *xa, *xb;               // fp16, OUT: exponents of A's, B's values, or null
    int F, act;
    int tiles_m, tiles_n, n_items;
    int full, tail, tail_splits, tail_per, kt_per_tail;   // OUT: the last `tail` tiles, behind `full` whole rounds of the chip, split k (0: none)
};

// Bands of GM m tiles with the n tiles side by side: the 32 or 64 items that an XCD runs at a time are a block of 8 x 4 or 8 x 8 tiles, whose
// operands its L2 fetches once (one n tile with every m tile instead: 384 us for 355, 7680 x 1280 x 5120)
__device__ __forceinline__ void tile_at_item(int lin, int tiles_m, int tiles_n, int& tm, int& tn) {
    constexpr int GM = 8;
    const int band = lin / (GM * tiles_n), bm = min(GM, tiles_m - band * GM), r = lin - band * GM * tiles_n;
    tm = band * GM + r % bm;
    tn = r / bm;
}

__device__ __forceinline__ float sigmoid_(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * x)); }
// The normal distribution's integral, e = exp(-g g / 2) on the side. Below 0 as e R(|g|): 1 + erf would lose its digits there (from -6 on all of
// them). R(x) = exp(x x / 2) Phi(-x) runs from 1/2 to 1 / (x sqrt(2 pi)) and is a polynomial in t = 1 / (1 + 0.3 x), t the factor of all terms: the
// least largest relative deviation over 0 .. 14.5 (a fit in 64 bits) is 1.7e-7.
__device__ __forceinline__ float normal_(float g, float& e) {
    e = __builtin_amdgcn_exp2f(-0.5f * LOG2E * g * g);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3f, fabsf(g), 1.0f));
    constexpr float C[8] = {0.11963200649944483f, 0.12071214884664003f, 0.10017585937116391f, 0.1276920947382172f,
                            -0.052034684618224844f, 0.20455757001720992f, -0.15615893604636474f, 0.0354238594837955f};
    float r = C[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) r = __builtin_fmaf(r, t, C[i]);
    r *= t * e;
    return g < 0.f ? r : 1.0f - r;
}
__device__ __forceinline__ float act_of(int act, float g) {
    if (act == FFN_SILU) return g * sigmoid_(g);
    if (act == FFN_GELU) {
        float e;
        return g * normal_(g, e);
    }
    if (act == FFN_RELU) return g < 0.f ? 0.f : g;             // (a NaN stays one)
    return sigmoid_(g);
}
__device__ __forceinline__ void act_and_slope(int act, float g, float& f, float& d) {
    if (act == FFN_GELU) {
        float e;
        const float phi = normal_(g, e);
        f = g * phi;
        d = __builtin_fmaf(g * 0.3989422804014327f, e, phi);
    } else if (act == FFN_RELU) {
        f = g < 0.f ? 0.f : g;
        d = g > 0.f ? 1.f : 0.f;
    } else {
        const float t = __builtin_amdgcn_exp2f(-LOG2E * g), s = __builtin_amdgcn_rcpf(1.0f + t);
        const float c = g < 0.f ? 1.0f - s : t * s;            // 1 - s: by subtraction only where s is the smaller one
        f = act == FFN_SILU ? g * s : s;
        d = act == FFN_SILU ? s * __builtin_fmaf(g, c, 1.0f) : s * c;
    }
}

// requests of one operand tile. Layout 0: ROWS rows of 64 k (row valid below `rows`); layout 1: 64 k rows of ROWS values (value valid
// below `rows`). PAIR: rows 0-31 gate, 32-63 up, ... of ROWS / 2 features.
template <int LAY, int ROWS, int NW, bool PAIR>
struct OpLoad {
    static constexpr int PIECES = ROWS * BK * 2 / 1024 / NW, W = LAY == 0 ? BK : ROWS;
    static_assert(PIECES >= 1 && PIECES * NW * 1024 == ROWS * BK * 2 && W >= 64, "whole pieces per wave, rows that tile_xor covers");
    uint32_t voff[PIECES];
    int kk[PIECES];                                   // first k (layout 0) or k (layout 1) of the lane's chunk
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int rows) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int byte = (wave * PIECES + j) * 1024 + lane * 16, r = byte / (W * 2);
            const int c = ((byte % (W * 2)) >> 4) ^ tile_xor<W>(r);
            if constexpr (LAY == 0) {
                const int row = PAIR ? (r >> 6) * 32 + (r & 31) : r;
                kk[j] = 8 * c;
                voff[j] = row < rows ? (uint32_t)(row * (int)ld * 2 + c * 16) : DMA_NONE;
            } else {
                kk[j] = r;
                voff[j] = 8 * c < rows ? (uint32_t)(r * (int)ld * 2 + c * 16) : DMA_NONE;
            }
        }
    }
    // where the next tile comes from and goes to; its pieces can then be requested one by one
    i32x4 d, d2;
    int k_left;
    uint32_t to;
    __device__ __forceinline__ void aim(const uint16_t* base, const uint16_t* base2, int left, uint32_t lds, int wave) {
        d = dma_desc(base);
        d2 = PAIR ? dma_desc(base2) : d;
        k_left = left;
        to = lds + wave * PIECES * 1024;
    }
    __device__ __forceinline__ void piece(int j, int wave) const {
        const uint32_t v = kk[j] < k_left ? voff[j] : DMA_NONE;
        const bool up = PAIR && (((wave * PIECES + j) >> 2) & 1);          // a piece is 8 rows: 4 pieces per 32-row group (wave-uniform)
        dma16_desc(up ? d2 : d, v, to + j * 1024);
    }
};

// ---- fp16 between two products. h = act(g) o u, dG and dU may lie past 65504, or far below fp16's normal numbers, where y, dx and the weights'
// gradients do not. So a group of 8 rows x 32 features carries a power of two of its own: what is stored is value 2^-e, e = 0 while the group's largest magnitude lies in [2^-10, 65504] -- as
// good as always --, above just enough to bring it below 2^15, below in steps of 16. Exponents: a byte per group, [ceil(F / 32)][4 ceil(rows / 32)];
// EXP_NONE: nothing but zeros, infinities and NaN.
constexpr int EXP_NONE = -128;
// Whether groups that a wave has stored as they are should have carried a power of two: the common case has no branch, so that the steps of an
// epilogue stay side by side (with one in every step: GATE 56 -> 65 us, DH 48 -> 59 at 4111 rows, 640 x 2560). MARGIN: a little sooner.
template <bool MARGIN>
struct GroupCheck {
    static constexpr float LOW = MARGIN ? 0x1.01p-10f : 0x1p-10f, HIGH = MARGIN ? 65248.f : 65504.f;
    float hi = 0.f;
    uint64_t seen = 0;
    bool tiny = false;
    // a step's values; `fresh`: of new groups. Then, groups complete: which lanes hold each, and which of them are part of the matrix (uniform)
    __device__ __forceinline__ void add(const float (&v)[4], bool fresh) {
        const float mx = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
        hi = fmaxf(hi, mx);
        const uint64_t b = __ballot(mx >= LOW);
        seen = fresh ? b : seen | b;
    }
    __device__ __forceinline__ void close(uint64_t lanes, bool live) { tiny |= live && (seen & lanes) == 0; }
    // (of the whole wave: not behind a branch that some of its lanes take)
    __device__ __forceinline__ bool zero() const { return __ballot(hi > 0.f) == 0; }                      // (or NaN)
    __device__ __forceinline__ bool odd() const { return (tiny && !zero()) || __ballot(hi > HIGH) != 0; }
};
constexpr uint64_t ALL_LANES = ~0ull, LOW_COLUMNS = 0x00ff00ff00ff00ffull;         // the wave; of every 16 lanes the first 8
__device__ __forceinline__ float finite_max(const float (&v)[4], float mx = 0.f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = fabsf(v[i]) < __builtin_inff() ? fmaxf(mx, fabsf(v[i])) : mx;
    return mx;
}
__device__ __forceinline__ int exp_of(float mx) {
    const int x = __builtin_amdgcn_frexp_expf(mx);                        // mx = f 2^x, f in [1/2, 1)
    return mx == 0.f ? EXP_NONE : mx > 65504.f ? x - 15 : mx >= 0x1p-10f ? 0 : -16 * min((-10 - x) / 16 + 1, 7);
}
// over the lanes that hold 32 features: 8 of every 16
__device__ __forceinline__ float half_max(float mx) {
#pragma unroll
    for (int k : {1, 2, 4, 16, 32}) mx = fmaxf(mx, __shfl_xor(mx, k));
    return mx;
}
// N groups' bytes at once: all of them e
template <int N>
__device__ __forceinline__ void store_exps(int8_t* to, int e) {
    const uint32_t w = 0x01010101u * (uint8_t)e;
    static_assert(N == 1 || N == 4, "a wave's rows of a block: 8 or 32");
    if constexpr (N == 1) *to = (int8_t)w;
    else *reinterpret_cast<uint32_t*>(to) = w;
}
__device__ __forceinline__ float stored_by(int e) { return e == 0 || e == EXP_NONE ? 1.0f : __builtin_ldexpf(1.0f, -e); }

// What a wave of the product that reads such values knows of their exponents. BY_ROW (layout 0): lane l holds rows row0 + 32 i + (l & 31) of the
// matrix, and k runs over its columns; else (layout 1) lane l holds columns, k runs over the rows. A wave looks its part of the table over
// while its first tiles travel; nothing but zeros (the rule) costs no more than that. Else every lane's fragments are brought to the largest of the
// exponents that it will meet (2^(e - largest): exact down to subnormal numbers), whose power the sums get at the end.
template <int N, bool BY_ROW>
struct Powers {
    static constexpr int RG = 8, CG = 32, PER = 32 / RG;
    const int8_t* at;
    int stride, groups, blocks, first, half, width;                       // bytes per column block, those in use; column blocks; the wave's first row (column)
    int e[N], lane_;
    bool any, uneven;
    // rows x cols: the matrix. half_: columns of its first half (dG | dU), whose column blocks are counted apart, or cols
    __device__ __forceinline__ void init(const int8_t* table, int rows, int cols, int first_, int half_) {
        at = table;
        any = uneven = false;
        if (!at) return;
        stride = (rows + 31) / 32 * PER;
        groups = (rows + RG - 1) / RG;
        first = first_;
        half = half_;
        width = cols;
        blocks = (half + CG - 1) / CG * (cols > half ? 2 : 1);
    }
    __device__ __forceinline__ int block_of(int c) const {
        c = min(c, width - 1);
        return c < half ? c / CG : (half + CG - 1) / CG + (c - half) / CG;
    }
    __device__ __forceinline__ int exp_at(int block, int group) const { return block < blocks && group < groups ? at[(int64_t)block * stride + group] : EXP_NONE; }
    // BY_ROW: the column block of k-step ks of tile t (a half's last tile may be part full: zeros, whatever their exponent)
    __device__ __forceinline__ int block_of_k(int t, int ks) const {
        const int kts = (half + BK - 1) / BK, seg = t >= kts, b = 2 * (t - seg * kts) + (ks >> 1), per = (half + CG - 1) / CG;
        return seg * per + min(b, per - 1);
    }
    // tiles t0 .. t1 of 64 k
    __device__ __forceinline__ void look(int t0, int t1, int lane) {
        if (!at) return;
        lane_ = lane;
        uint32_t bits = 0;
        const int c0 = BY_ROW ? block_of_k(t0, 0) : block_of(first), c9 = 1 + (BY_ROW ? block_of_k(t1 - 1, KS - 1) : block_of(first + 32 * N - 1));
        const int r0 = BY_ROW ? first / 32 : t0 * 2, r9 = min(stride / PER, BY_ROW ? first / 32 + N : t1 * 2);
        const auto take = [&](int c, int r) { bits |= *reinterpret_cast<const uint32_t*>(at + (int64_t)c * stride + r * PER); };
        if constexpr (BY_ROW) {
            for (int c = c0 + lane; c < c9; c += 64)
                for (int r = r0; r < r9; ++r) take(c, r);
        } else {
            for (int c = c0; c < c9; ++c)
                for (int r = r0 + lane; r < r9; r += 64) take(c, r);
        }
        any = __any((bits & 0x7f7f7f7fu) != 0);
        if (!any) return;
        // the largest and smallest exponent per lane: every lane takes its share of the words, byte k of which (BY_ROW: of row group k) it keeps apart
        bool differ = false;
#pragma unroll 1
        for (int i = 0; i < N; ++i) {
            const int mine = first + 32 * i + (lane & 31), b0 = BY_ROW ? 0 : block_of(first + 32 * i), b1 = BY_ROW ? 0 : block_of(first + 32 * i + 31);
            int top = 0;
#pragma unroll 1
            for (int b = b0; b <= b1; ++b) {                              // (32 columns lie in at most two blocks)
                int hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) { hi[k] = EXP_NONE; lo[k] = 127; }
                const int r = first / 32 + i;
                if (!BY_ROW || r < stride / PER) {
                    for (int n = (BY_ROW ? c0 : r0) + lane; n < (BY_ROW ? c9 : r9); n += 64) {
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(at + (int64_t)(BY_ROW ? n : b) * stride + (BY_ROW ? r : n) * PER);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int x = (int8_t)(w >> (8 * k));
                            if (x != EXP_NONE && (BY_ROW ? r : n) * PER + k < groups) { hi[k] = max(hi[k], x); lo[k] = min(lo[k], x); }
                        }
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int o = 1; o < 64; o <<= 1) { hi[k] = max(hi[k], __shfl_xor(hi[k], o)); lo[k] = min(lo[k], __shfl_xor(lo[k], o)); }
                int h = hi[0], l = lo[0];
#pragma unroll
                for (int k = 1; k < 4; ++k) {
                    if (!BY_ROW) { h = max(h, hi[k]); l = min(l, lo[k]); }
                    else if ((mine / RG) % PER == k) { h = hi[k]; l = lo[k]; }
                }
                if (BY_ROW || block_of(mine) == b) {
                    top = h == EXP_NONE ? 0 : h;
                    differ |= h != EXP_NONE && l < h;
                }
            }
#pragma unroll
            for (int k = 0; k < N; ++k) e[k] = k == i ? top : e[k];
        }
        uneven = __any(differ);
    }
    // the exponents of tile t for a lane's fragment i: a byte per k-step (BY_ROW), or per half a k-step
    __device__ __forceinline__ uint2 of_tile(int i, int t) const {
        const int mine = first + 32 * i + (lane_ & 31);
        if constexpr (BY_ROW) {
            const int a = exp_at(block_of_k(t, 0), mine / RG) & 0xff, b = exp_at(block_of_k(t, 2), mine / RG) & 0xff;
            return make_uint2(a * 0x101u | b * 0x1010000u, 0u);
        } else {
            const int g = t * (BK / RG);                                  // (past the last row: zeros, whatever their exponent)
            const uint32_t* w = reinterpret_cast<const uint32_t*>(at + (int64_t)block_of(mine) * stride + g);
            return make_uint2(g < stride ? w[0] : 0u, g + 4 < stride ? w[1] : 0u);
        }
    }
    // 2^d in both halves of a word, -24 <= d <= 0
    static __device__ __forceinline__ uint32_t half_power(int d) {
        const uint32_t h = d >= -14 ? (uint32_t)(15 + d) << 10 : 1u << (24 + d);
        return h | h << 16;
    }
    static __device__ __forceinline__ uint32_t times(uint32_t w, uint32_t f) { return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, w) * __builtin_bit_cast(f16x2_t, f)); }
    // fragment i of k-step ks, brought to the lane's common exponent (8 rows or 16 features of one group); x: of_tile
    __device__ __forceinline__ uint4 level(uint4 f, int i, uint2 x, int ks) const {
        const uint32_t w = BY_ROW || ks < 2 ? x.x : x.y;
        const int at_byte = BY_ROW ? ks : 2 * (ks & 1) + (lane_ >> 5);
        // in two factors: 2^d reaches below fp16's smallest number where the value does not. -48 leaves nothing of a finite one; an infinity stays one
        const int d = min(max((int)(int8_t)(w >> (8 * at_byte)) - e[i], -48), 0), d0 = d >> 1;
        const uint32_t h0 = half_power(d0), h1 = half_power(d - d0);
        return make_uint4(times(times(f.x, h0), h1), times(times(f.y, h0), h1), times(times(f.z, h0), h1), times(times(f.w, h0), h1));
    }
};

// ROWS x 64 operand tile in LDS -> fragment of 32 rows (columns) at r0, k-step ks
template <int LAY, int ROWS>
__device__ __forceinline__ uint4 op_frag(const unsigned char* t, int r0, int ks, int lane) {
    if constexpr (LAY == 0) return frag_rows<BK>(t, r0, ks, lane);
    else return frag_cols<ROWS, 8, 4>(t, 16 * ks, r0, lane);
}

// this wave's requests have landed, all but the newest N (`newest`: that many are known to be on their way), and its LDS reads are done
template <int N>
__device__ __forceinline__ void wait_landed(bool newest) {
    if (newest) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
}
__device__ __forceinline__ void meet() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// what this wave's lanes wrote to LDS is there for its other lanes (a wave's LDS accesses are done in order; this keeps the compiler to it)
__device__ __forceinline__ void corner_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <bool F16, int BM, int BN, int NWM, int NWN, int NWK, int NBUF, int LA, int LB, int EPI>
__global__ __launch_bounds__(NWM * NWN * NWK * 64, NWM * NWN >= 8 ? 2 : 1) void ffn_mm_kernel(MmArgs p) {
    constexpr int NW = NWM * NWN * NWK, WM = BM / NWM, WN = BN / NWN, IM = WM / 32, IN = WN / 32;
    constexpr bool PAIR = EPI == EPI_GATE;
    static_assert(!PAIR || (IN % 2 == 0 && LB == 0), "a wave owns gate and up columns of the same features");
    constexpr int ABYTES = BM * BK * 2, STAGE = ABYTES + BN * BK * 2;
    int item, split = 0, tm, tn;
    bool tail = false;
    if (EPI == EPI_OUT && p.tail > 0) {
        // every XCD takes its eighth of the whole rounds, then its eighth of the tail's parts
        const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, per = p.full >> 3;
        tail = slot >= per;
        item = xcd * per + slot;
        if (tail) {
            const int t = xcd * p.tail_per + slot - per;
            if (t >= p.tail * p.tail_splits) return;
            item = p.full + t / p.tail_splits;
            split = t % p.tail_splits;
        }
        tile_at_item(item, p.tiles_m, p.tiles_n, tm, tn);
    } else {
        item = xcd_item(blockIdx.x, p.n_items);
        if (item >= p.n_items) return;
        split = item / (p.tiles_m * p.tiles_n);
        tile_at_item(item - split * p.tiles_m * p.tiles_n, p.tiles_m, p.tiles_n, tm, tn);
    }
    const int m0 = tm * BM, n0 = tn * BN;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    const int wm = wave % NWM, wn = wave / NWM % NWN, wk = wave / (NWM * NWN);

    const int kts = (p.K + BK - 1) / BK, total = kts * p.nseg;
    const int kt_per = tail ? p.kt_per_tail : p.kt_per_split, t0 = split * kt_per, t1 = min(total, t0 + kt_per);
    OpLoad<LA, BM, NW, false> la;
    OpLoad<LB, BN, NW, PAIR> lb;
    la.init(wave, lane, p.lda, p.M - m0);
    lb.init(wave, lane, p.ldb, PAIR ? p.F - n0 / 2 : p.N - n0);
    const uint32_t lds0 = lds_addr_of(conv_lds_dyn);
    auto aim = [&](int t, int buf) {
        const int seg = t >= kts, kt = t - seg * kts;
        const int k0 = kt * BK;
        const uint16_t* a = LA == 0 ? p.A + (int64_t)m0 * p.lda + seg * p.K + k0 : p.A + (int64_t)k0 * p.lda + m0;
        const uint16_t* bb = PAIR || !seg ? p.B : p.B2;
        const int64_t off = LB == 0 ? (int64_t)(PAIR ? n0 / 2 : n0) * p.ldb + k0 : (int64_t)k0 * p.ldb + n0;
        la.aim(a, nullptr, p.K - k0, lds0 + buf * STAGE, wave);
        lb.aim(bb + off, PAIR ? p.B2 + off : nullptr, p.K - k0, lds0 + buf * STAGE + ABYTES, wave);
    };
    constexpr int PA = decltype(la)::PIECES, PIECES = PA + decltype(lb)::PIECES;
    auto piece = [&](int j) { if (j < PA) la.piece(j, wave); else lb.piece(j - PA, wave); };
    f32x16 acc[IM][IN];
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    // Fragments run one k-step ahead of the products, also over the edge of a tile: the workgroup meets BEFORE the last k-step's products, when
    // every wave holds its fragments of the old tile; the buffer is then free for the tile NBUF ahead, whose requests have NBUF - 1 tiles'
    // products to land (the wait counts the requests of the tiles that may still be on their way: the loop has no other memory access).
    // Fragment reads and requests are issued one by one BETWEEN the products (the matrix pipe takes 32 cycles each).
    uint4 fa[2][IM], fb[2][IN];
    auto fetch = [&](int buf, int ks, int i) {
        const unsigned char* at = conv_lds_dyn + buf * STAGE;
        if (i < IN) fb[ks & 1][i] = op_frag<LB, BN>(at + ABYTES, wn * WN + 32 * i, ks, lane);
        else fa[ks & 1][i - IN] = op_frag<LA, BM>(at, wm * WM + 32 * (i - IN), ks, lane);
    };
    // fp16 operands with powers of two: A's rows (down, dx), A's columns (dW gate, up) or B's (dW down)
    constexpr bool POWERS = F16 && EPI == EPI_OUT;
    Powers<IM, LA == 0> pa;
    Powers<IN, false> pb;
    if constexpr (POWERS) {
        if constexpr (LA == 0) pa.init(p.xa, p.M, p.K * p.nseg, m0 + wm * WM, p.K);
        else pa.init(p.xa, p.K, p.M, m0 + wm * WM, p.F);
        pb.init(LA == 1 ? p.xb : nullptr, p.K, p.N, n0 + wn * WN, p.N);
    }
    auto look = [&] {
        if constexpr (POWERS) {
            pa.look(t0, t1, lane);
            if constexpr (LA == 1) pb.look(t0, t1, lane);
        }
    };
    auto uneven = [&] { return pa.uneven || (LA == 1 && pb.uneven); };
    // (the loop over the tiles exists twice, with and without this: its waits and meetings are the same, so a wave chooses for itself)
    uint2 xa[IM], xb[IN], xa_next[IM], xb_next[IN];                       // exponents of this tile and of the next one
    auto exps = [&](auto on, int t, uint2 (&a)[IM], uint2 (&b)[IN]) {
        if constexpr (decltype(on)::value) {
            if (pa.uneven) {
#pragma unroll
                for (int i = 0; i < IM; ++i) a[i] = pa.of_tile(i, t);
            }
            if constexpr (LA == 1)
                if (pb.uneven) {
#pragma unroll
                    for (int j = 0; j < IN; ++j) b[j] = pb.of_tile(j, t);
                }
        }
    };
    auto turn = [&](auto on) {
        if constexpr (decltype(on)::value) {
#pragma unroll
            for (int i = 0; i < IM; ++i) xa[i] = xa_next[i];
#pragma unroll
            for (int j = 0; j < IN; ++j) xb[j] = xb_next[j];
        }
    };
    auto level = [&](auto on, uint4 (&a)[IM], uint4 (&b)[IN], int ks) {
        if constexpr (decltype(on)::value) {
            if (pa.uneven) {
#pragma unroll
                for (int i = 0; i < IM; ++i) a[i] = pa.level(a[i], i, xa[i], ks);
            }
            if constexpr (LA == 1)
                if (pb.uneven) {
#pragma unroll
                    for (int j = 0; j < IN; ++j) b[j] = pb.level(b[j], j, xb[j], ks);
                }
        }
    };
    constexpr int SLOTS = IM * IN, FETCH = IM + IN;
    static_assert(KS % 2 == 0, "k-step 0 of the next tile takes the other half of the fragment registers");
    if constexpr (NWK > 1) {
        // few rows: the waves share out the k-steps of a tile (their sums meet below), so a tile costs a wave its share of the requests, one
        // step's fragments and its products
        static_assert(KS % NWK == 0 && NWM == 1 && NWN == 1 && (NBUF - 1) * PIECES < 64, "whole steps per wave");
#pragma unroll
        for (int n = 0; n < NBUF - 1; ++n)
            if (t0 + n < t1) {
                aim(t0 + n, n);
#pragma unroll
                for (int j = 0; j < PIECES; ++j) piece(j);
            }
        look();
        const auto walk = [&](auto leveled) {
        int buf = 0, free = NBUF - 1;
        if (t0 < t1) exps(leveled, t0, xa_next, xb_next);
        for (int t = t0; t < t1; ++t) {
            turn(leveled);
            if (t + 1 < t1) exps(leveled, t + 1, xa_next, xb_next);
            wait_landed<(NBUF - 2) * PIECES>(t + NBUF - 1 <= t1);
            meet();                                                            // tile t is there, and nobody reads tile t - 1 any more
            if (t + NBUF - 1 < t1) {
                aim(t + NBUF - 1, free);
#pragma unroll
                for (int j = 0; j < PIECES; ++j) piece(j);
            }
#pragma unroll
            for (int k = 0; k < KS / NWK; ++k) {
                const unsigned char* at = conv_lds_dyn + buf * STAGE;
                const int ks = wk * (KS / NWK) + k;
#pragma unroll
                for (int j = 0; j < IN; ++j) fb[0][j] = op_frag<LB, BN>(at + ABYTES, 32 * j, ks, lane);
#pragma unroll
                for (int i = 0; i < IM; ++i) fa[0][i] = op_frag<LA, BM>(at, 32 * i, ks, lane);
                level(leveled, fa[0], fb[0], ks);
#pragma unroll
                for (int j = 0; j < IN; ++j)
#pragma unroll
                    for (int i = 0; i < IM; ++i) acc[i][j] = T16<F16>::mfma32(fb[0][j], fa[0][i], acc[i][j]);
            }
            free = buf;
            buf = buf + 1 == NBUF ? 0 : buf + 1;
        }
        };
        if (POWERS && uneven()) walk(std::bool_constant<POWERS>());
        else walk(std::false_type());
    } else {
    static_assert((NBUF - 2) * PIECES < 64, "vmcnt counts to 63");
    if (t0 < t1) {
#pragma unroll
        for (int n = 0; n < NBUF; ++n)
            if (t0 + n < t1) {
                aim(t0 + n, n);
#pragma unroll
                for (int j = 0; j < PIECES; ++j) piece(j);
            }
        look();
        wait_landed<(NBUF - 1) * PIECES>(t0 + NBUF <= t1);
        meet();
#pragma unroll
        for (int i = 0; i < FETCH; ++i) fetch(0, 0, i);
    }
    const auto walk = [&](auto leveled) {
    int buf = 0;
    if (t0 < t1) exps(leveled, t0, xa_next, xb_next);
    for (int t = t0; t < t1; ++t) {
        const int nbuf = buf + 1 == NBUF ? 0 : buf + 1;
        turn(leveled);
        if (t + 1 < t1) exps(leveled, t + 1, xa_next, xb_next);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bool edge = ks + 1 == KS, more = edge && t + NBUF < t1;
            if (edge) {
                if (t + 1 < t1) {
                    wait_landed<(NBUF - 2) * PIECES>(t + NBUF <= t1);
                    meet();
                }
                if (more) aim(t + NBUF, buf);
            }
            level(leveled, fa[ks & 1], fb[ks & 1], ks);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) {
                acc[s / IN][s % IN] = T16<F16>::mfma32(fb[ks & 1][s % IN], fa[ks & 1][s / IN], acc[s / IN][s % IN]);
#pragma unroll
                for (int i = s * FETCH / SLOTS; i < (s + 1) * FETCH / SLOTS; ++i) {
                    if (!edge) fetch(buf, ks + 1, i);
                    else if (t + 1 < t1) fetch(nbuf, 0, i);
                }
                if (more) {
#pragma unroll
                    for (int j = s * PIECES / SLOTS; j < (s + 1) * PIECES / SLOTS; ++j) piece(j);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        buf = nbuf;
    }
    };
    if (POWERS && uneven()) walk(std::bool_constant<POWERS>());
    else walk(std::false_type());
    }

    if constexpr (POWERS) {
        if (pa.any || (LA == 1 && pb.any)) {
#pragma unroll
            for (int i = 0; i < IM; ++i)
#pragma unroll
                for (int j = 0; j < IN; ++j) {                            // (32 columns of B are one column block: e[j] is the wave's)
                    const float f = __builtin_ldexpf(1.0f, (pa.any ? pa.e[i] : 0) + (LA == 1 && pb.any ? pb.e[j] : 0));
#pragma unroll
                    for (int k = 0; k < 16; ++k) acc[i][j][k] *= f;
                }
        }
    }

    // The accumulators hold 32 rows m a lane column each; memory wants whole rows. Each wave turns its 32 x WN blocks round in its own corner of
    // the operand buffers (free now), so that WN / 4 lanes write one row: full lines instead of 32-byte pieces.
    constexpr int LN = WN / 4, RS = WN + 4, STEP = 64 / LN;           // lanes per row, LDS row (floats), rows per step
    static_assert(NW * 32 * RS * 4 <= NBUF * STAGE, "the corners fit");
    wait_all_and_meet();
    float* corner = reinterpret_cast<float*>(conv_lds_dyn) + wave * 32 * RS;
    const int cl = lane % LN, rl = lane / LN;
    // (GATE, DH: one copy of what follows: unrolled over the blocks the activations do not fit the instruction cache)
    int guess_g = 0, guess_u = 0;                                          // DH, fp16: the exponents that the next block's dG and dU are stored with first
    constexpr int BLOCKS_AT_ONCE = EPI == EPI_OUT ? IM : 1, STEPS_AT_ONCE = EPI == EPI_OUT ? 4 : 1;
#pragma unroll BLOCKS_AT_ONCE
    for (int i = 0; i < IM; ++i) {
#pragma unroll
        for (int k = 0; k < IM; ++k) {
            if (k != i) continue;
#pragma unroll
            for (int j = 0; j < IN; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4*>(corner + (lane & 31) * RS + 32 * j + 8 * q + 4 * h) =
                        make_float4(acc[k][j][4 * q], acc[k][j][4 * q + 1], acc[k][j][4 * q + 2], acc[k][j][4 * q + 3]);
        }
        // NWK waves hold parts of the same sums: each adds up 32 / NWK rows over the corners, in wave order, and goes on with those
        constexpr int RN = 32 / NWK;
        const int R0 = wk * RN;
        float* rows = corner;
        if constexpr (NWK > 1) {
            __syncthreads();
            rows = reinterpret_cast<float*>(conv_lds_dyn);
#pragma unroll
            for (int r = 0; r < RN; r += STEP) {
                float* at = rows + (R0 + r + rl) * RS + 4 * cl;
                float4 t = *reinterpret_cast<const float4*>(at);
#pragma unroll
                for (int w = 1; w < NWK; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(at + w * 32 * RS);
                    t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
                }
                *reinterpret_cast<float4*>(at) = t;
            }
        }
        corner_done();
        // fp16 results saturate; the switch is set behind the products (saturate_from_here) and before anything read from the corner is converted
        saturate_from_here<F16>();
        corner_done();
        const int mb = m0 + wm * WM + 32 * i;
        float sg[4] = {}, su[4] = {};                                         // DH: column sums over the block's rows
        if constexpr (EPI == EPI_GATE) {
            // half the lanes of a row: 4 features each, gate columns in the first 32 of every 64, up columns 32 further on
            constexpr int LF = LN / 2, SF = 64 / LF;
            const int c2 = lane % LF, r2 = lane / LF;
            const int gc = (c2 >> 3) * 64 + (c2 & 7) * 4, f = (n0 + wn * WN) / 2 + 4 * c2;
            float bg[4] = {}, bu[4] = {};
            if (f < p.F) {
                if (p.bias) {
                    const uint2 w = *reinterpret_cast<const uint2*>(p.bias + f);
                    bg[0] = T16<F16>::lo(w.x); bg[1] = T16<F16>::hi(w.x); bg[2] = T16<F16>::lo(w.y); bg[3] = T16<F16>::hi(w.y);
                }
                if (p.bias2) {
                    const uint2 w = *reinterpret_cast<const uint2*>(p.bias2 + f);
                    bu[0] = T16<F16>::lo(w.x); bu[1] = T16<F16>::hi(w.x); bu[2] = T16<F16>::lo(w.y); bu[3] = T16<F16>::hi(w.y);
                }
            }
            // fp16: a wave's step is a group of 8 rows x 32 features
            static_assert(!F16 || (SF == 8 && WN == 64), "8 rows x 32 features");
            GroupCheck<false> check;
            const bool live = (n0 + wn * WN) / 2 < p.F;
            const auto hidden = [&](auto whole, int r, float (&g)[4], float (&u)[4], float (&o)[4]) {
                const float4 g4 = *reinterpret_cast<const float4*>(rows + (r + r2) * RS + gc), u4 = *reinterpret_cast<const float4*>(rows + (r + r2) * RS + gc + 32);
                const bool in = decltype(whole)::value || (mb + r + r2 < p.M && f < p.F);
                g[0] = g4.x + bg[0]; g[1] = g4.y + bg[1]; g[2] = g4.z + bg[2]; g[3] = g4.w + bg[3];
                u[0] = u4.x + bu[0]; u[1] = u4.y + bu[1]; u[2] = u4.z + bu[2]; u[3] = u4.w + bu[3];
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = F16 && !in ? 0.f : act_of(p.act, g[e]) * u[e];
                return in;
            };
            const auto put = [&](int r, const float (&o)[4], float by) {
                *reinterpret_cast<uint2*>(p.C + (int64_t)(mb + r + r2) * p.F + f) = make_uint2(T16<F16>::pack2(o[0] * by, o[1] * by), T16<F16>::pack2(o[2] * by, o[3] * by));
            };
            // (a block that lies in the matrix as a whole has no masks between its steps)
            const auto store = [&](auto whole) {
#pragma unroll
            for (int r = R0; r < R0 + RN; r += SF) {
                float g[4], u[4], o[4];
                const bool in = hidden(whole, r, g, u, o);
                if constexpr (F16) {
                    check.add(o, true);
                    check.close(ALL_LANES, decltype(whole)::value || (live && mb + r < p.M));
                }
                if (!in) continue;
                if (p.g) {
                    const int64_t at = (int64_t)(mb + r + r2) * p.F + f;
                    *reinterpret_cast<float4*>(p.g + at) = make_float4(g[0], g[1], g[2], g[3]);
                    *reinterpret_cast<float4*>(p.u + at) = make_float4(u[0], u[1], u[2], u[3]);
                }
                put(r, o, 1.0f);
            }
            };
            if (mb + 32 <= p.M && (n0 + wn * WN) / 2 + 32 <= p.F) store(std::true_type());
            else store(std::false_type());
            if constexpr (F16) {
                int8_t* ex = p.ex + (int64_t)(f / 32) * ((p.M + 31) / 32 * 4) + (mb + R0) / 8;
                const bool first = lane == 0 && live && mb < p.M;
                const int plain = check.zero() ? EXP_NONE : 0;
                if (!check.odd()) {
                    if (first) store_exps<RN / SF>(ex, plain);
                } else {
#pragma unroll 1
                    for (int r = R0; r < R0 + RN; r += SF) {
                        float g[4], u[4], o[4];
                        const bool in = hidden(std::false_type(), r, g, u, o);
                        float mx = finite_max(o);
#pragma unroll
                        for (int k = 1; k < 64; k <<= 1) mx = fmaxf(mx, __shfl_xor(mx, k));
                        const int x = exp_of(mx);
                        if (in) put(r, o, stored_by(x));
                        if (first) ex[(r - R0) / SF] = (int8_t)x;
                    }
                }
            }
        } else {
            const int n = n0 + wn * WN + 4 * cl;
            float bias[4] = {};
            if constexpr (EPI == EPI_OUT)
                if (p.bias && p.splits == 1 && n < p.N) {
                    const uint2 w = *reinterpret_cast<const uint2*>(p.bias + n);
                    bias[0] = T16<F16>::lo(w.x); bias[1] = T16<F16>::hi(w.x); bias[2] = T16<F16>::lo(w.y); bias[3] = T16<F16>::hi(w.y);
                }
            // DH, fp16: two steps of a wave are two groups of 8 rows x 32 features, side by side
            static_assert(!(F16 && EPI == EPI_DH) || (STEP == 4 && WN == 64 && RN % 8 == 0), "8 rows x 64 features");
            // dG and dU are tried with the exponent (0 or below) of the last group that needed one: small gradients are small all over, and a block is
            // stored anew only where that changes
            const float by_g = stored_by(guess_g), by_u = stored_by(guess_u);
            GroupCheck<false> cg, cu;
            GroupCheck<true> ch;                                              // (h: what GATE has scaled has to be found again)
            const bool live = n0 + wn * WN < p.N, live2 = n0 + wn * WN + 32 < p.N;
            const auto in_range = [&](int r) { return mb + r + rl < p.M && n < p.N; };
            const auto grads = [&](auto whole, int r, float (&dg)[4], float (&du)[4], float (&hh)[4]) {         // (outside: all 0)
                const int64_t at = (int64_t)(mb + r + rl) * p.F + n;
                float4 g4 = make_float4(0.f, 0.f, 0.f, 0.f), u4 = g4, o = g4;          // (a zero row's product with an infinite weight is none)
                if (decltype(whole)::value || in_range(r)) {
                    o = *reinterpret_cast<const float4*>(rows + (r + rl) * RS + 4 * cl);
                    g4 = *reinterpret_cast<const float4*>(p.g + at);
                    u4 = *reinterpret_cast<const float4*>(p.u + at);
                }
                const float g[4] = {g4.x, g4.y, g4.z, g4.w}, u[4] = {u4.x, u4.y, u4.z, u4.w}, d[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float f, s;
                    act_and_slope(p.act, g[e], f, s);
                    dg[e] = d[e] * u[e] * s;
                    du[e] = d[e] * f;
                    hh[e] = f * u[e];
                }
            };
            const auto put_d = [&](uint16_t* c, int r, const float (&d)[4], float by) {
                *reinterpret_cast<uint2*>(c + (int64_t)(mb + r + rl) * p.ldc + n) = make_uint2(T16<F16>::pack2(d[0] * by, d[1] * by), T16<F16>::pack2(d[2] * by, d[3] * by));
            };
            const auto put_h = [&](int r, const float (&hh)[4], float by) {
                *reinterpret_cast<uint2*>(p.h + (int64_t)(mb + r + rl) * p.F + n) =
                    make_uint2(T16<F16>::pack2(hh[0] * by, hh[1] * by), T16<F16>::pack2(hh[2] * by, hh[3] * by));
            };
            const auto store = [&](auto whole_) {
            constexpr bool whole = decltype(whole_)::value;
#pragma unroll STEPS_AT_ONCE
            for (int r8 = R0; r8 < R0 + RN; r8 += 8)
#pragma unroll
            for (int r = r8; r < r8 + 8; r += STEP) {
                const int m = mb + r + rl;
                if constexpr (EPI == EPI_DH) {
                    if (!F16 && !whole && !in_range(r)) continue;
                    float dg[4], du[4], hh[4];
                    grads(whole_, r, dg, du, hh);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sg[e] += dg[e];
                        su[e] += du[e];
                    }
                    if constexpr (F16) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            dg[e] *= by_g;
                            du[e] *= by_u;
                        }
                        cg.add(dg, r == r8);
                        cu.add(du, r == r8);
                        ch.add(hh, r == r8);
                        if (r != r8)
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint64_t lanes = k == 0 ? LOW_COLUMNS : ~LOW_COLUMNS;
                                const bool in = whole || ((k == 0 ? live : live2) && mb + r - 4 < p.M);
                                cg.close(lanes, in);
                                cu.close(lanes, in);
                                ch.close(lanes, in);
                            }
                        if (!whole && !in_range(r)) continue;
                    }
                    put_d(p.C, r, dg, 1.0f);
                    put_d(p.C + p.F, r, du, 1.0f);
                } else {
                    if (!whole && !in_range(r)) continue;
                    const float4 o = *reinterpret_cast<const float4*>(rows + (r + rl) * RS + 4 * cl);
                    if (p.splits > 1) {
                        *reinterpret_cast<float4*>(p.part + ((int64_t)split * p.M + m) * p.N + n) = o;
                    } else if (EPI == EPI_OUT && tail) {
                        *reinterpret_cast<float4*>(p.part + ((int64_t)((item - p.full) * p.tail_splits + split) * BM + m - m0) * BN + n - n0) = o;
                    } else {
                        *reinterpret_cast<uint2*>(p.C + (int64_t)m * p.ldc + n) =
                            make_uint2(T16<F16>::pack2(o.x + bias[0], o.y + bias[1]), T16<F16>::pack2(o.z + bias[2], o.w + bias[3]));
                    }
                }
            }
            };
            if (mb + 32 <= p.M && n0 + wn * WN + WN <= p.N) store(std::true_type());
            else store(std::false_type());
            if constexpr (F16 && EPI == EPI_DH) {
                const int64_t ex = (int64_t)(n / 32) * ((p.M + 31) / 32 * 4) + (mb + R0) / 8;
                const bool first = (lane & ~8) == 0 && n < p.N && mb < p.M;
                const int64_t up = (int64_t)((p.F + 31) / 32) * ((p.M + 31) / 32 * 4);         // dU's column blocks follow dG's
                const bool og = cg.odd(), ou = cu.odd(), oh = ch.odd();
                const int zg = cg.zero() ? EXP_NONE : guess_g, zu = cu.zero() ? EXP_NONE : guess_u, zh = ch.zero() ? EXP_NONE : 0;
                if (first) {
                    if (!og) store_exps<RN / 8>(p.ex + ex, zg);
                    if (!ou) store_exps<RN / 8>(p.ex + up + ex, zu);
                    if (!oh) store_exps<RN / 8>(p.ex_h + ex, zh);
                }
                // (one of the three at a time: a wave's registers are taken)
                const auto anew = [&](int8_t* to, auto pick, auto put) {
                    int last = 0;
#pragma unroll 1
                    for (int r = R0; r < R0 + RN; r += 8) {
                        float v[2][4];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            float dg[4], du[4], hh[4];
                            grads(std::false_type(), r + 4 * k, dg, du, hh);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[k][e] = pick(dg[e], du[e], hh[e]);
                        }
                        const int x = exp_of(half_max(finite_max(v[1], finite_max(v[0]))));
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            if (in_range(r + 4 * k)) put(r + 4 * k, v[k], stored_by(x));
                        if (first) to[ex + (r - R0) / 8] = (int8_t)x;
                        last = x == EXP_NONE ? last : min(x, 0);
                    }
                    return __builtin_amdgcn_readfirstlane(last);
                };
                if (og) guess_g = anew(p.ex, [](float a, float, float) { return a; }, [&](int r, const float (&v)[4], float by) { put_d(p.C, r, v, by); });
                if (ou) guess_u = anew(p.ex + up, [](float, float a, float) { return a; }, [&](int r, const float (&v)[4], float by) { put_d(p.C + p.F, r, v, by); });
                if (oh) anew(p.ex_h, [](float, float, float a) { return a; }, put_h);
            }
        }
        if constexpr (EPI == EPI_DH) {
            if (p.cs) {                                       // the block's column sums: the STEP lanes of a column, then one row of cs per 32 rows
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int o = LN; o < 64; o <<= 1) { sg[e] += __shfl_xor(sg[e], o); su[e] += __shfl_xor(su[e], o); }
                const int n = n0 + wn * WN + 4 * cl;
                if constexpr (NWK > 1) {
                    float* part = reinterpret_cast<float*>(conv_lds_dyn) + NW * 32 * RS;       // [NWK][2][WN], behind the corners
                    static_assert((NW * 32 * RS + NWK * 2 * WN) * 4 <= NBUF * STAGE, "the sums fit");
                    if (rl == 0) {
                        *reinterpret_cast<float4*>(part + wk * 2 * WN + 4 * cl) = make_float4(sg[0], sg[1], sg[2], sg[3]);
                        *reinterpret_cast<float4*>(part + wk * 2 * WN + WN + 4 * cl) = make_float4(su[0], su[1], su[2], su[3]);
                    }
                    __syncthreads();
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sg[e] = su[e] = 0.f;
#pragma unroll
                        for (int w = 0; w < NWK; ++w) { sg[e] += part[w * 2 * WN + 4 * cl + e]; su[e] += part[w * 2 * WN + WN + 4 * cl + e]; }
                    }
                }
                if (wk == 0 && rl == 0 && mb < p.M && n < p.N) {
                    float* c = p.cs + (int64_t)(mb / 32) * 2 * p.F + n;
                    *reinterpret_cast<float4*>(c) = make_float4(sg[0], sg[1], sg[2], sg[3]);
                    *reinterpret_cast<float4*>(c + p.F) = make_float4(su[0], su[1], su[2], su[3]);
                }
            }
        }
        corner_done();
    }
}

// sums of the splits of k in their order, + bias; four values per thread. The three products of a backward pass may share one launch (BwdParts)
struct Sums {
    struct One { const float* part; const uint16_t* bias; uint16_t* C; int64_t n4; int N, splits, blocks; } of[3];
    int blocks() const { return of[0].blocks + of[1].blocks + of[2].blocks; }
};
template <bool F16>
__global__ __launch_bounds__(256) void ffn_sum_kernel(Sums all) {
    T16<F16>::enter();
    int b = blockIdx.x, k = 0;
    while (b >= all.of[k].blocks) b -= all.of[k++].blocks;
    const Sums::One p = all.of[k];
    const int64_t i = (int64_t)b * 256 + threadIdx.x;
    if (i >= p.n4) return;
    float o[4] = {};
    for (int s = 0; s < p.splits; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(p.part + (s * p.n4 + i) * 4);
        o[0] += v.x; o[1] += v.y; o[2] += v.z; o[3] += v.w;
    }
    if (p.bias) {
        const uint2 w = *reinterpret_cast<const uint2*>(p.bias + i * 4 % p.N);
        o[0] += T16<F16>::lo(w.x); o[1] += T16<F16>::hi(w.x); o[2] += T16<F16>::lo(w.y); o[3] += T16<F16>::hi(w.y);
    }
    *reinterpret_cast<uint2*>(p.C + i * 4) = make_uint2(T16<F16>::pack2(o[0], o[1]), T16<F16>::pack2(o[2], o[3]));
}

// the same for the tail's tiles: part [tail tile][split][BM][BN]; a workgroup takes 1024 values of a tile
template <bool F16, int BM, int BN>
__global__ __launch_bounds__(256) void ffn_tail_kernel(MmArgs p) {
    T16<F16>::enter();
    constexpr int PER = BM * BN / 1024;
    const int t = blockIdx.x / PER, i = (blockIdx.x % PER * 256 + threadIdx.x) * 4;
    int tm, tn;
    tile_at_item(p.full + t, p.tiles_m, p.tiles_n, tm, tn);
    const int m = tm * BM + i / BN, n = tn * BN + i % BN;
    if (m >= p.M || n >= p.N) return;
    float o[4] = {};
    for (int s = 0; s < p.tail_splits; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(p.part + (int64_t)(t * p.tail_splits + s) * BM * BN + i);
        o[0] += v.x; o[1] += v.y; o[2] += v.z; o[3] += v.w;
    }
    if (p.bias) {
        const uint2 w = *reinterpret_cast<const uint2*>(p.bias + n);
        o[0] += T16<F16>::lo(w.x); o[1] += T16<F16>::hi(w.x); o[2] += T16<F16>::lo(w.y); o[3] += T16<F16>::hi(w.y);
    }
    *reinterpret_cast<uint2*>(p.C + (int64_t)m * p.ldc + n) = make_uint2(T16<F16>::pack2(o[0], o[1]), T16<F16>::pack2(o[2], o[3]));
}

// ------------------------------------------------------------------------------------------------------------------------------------
// At most TOKENS rows: the weights are the work, each read once in whole 1-KiB rows of a wave; dot products on the vector ALU.
// PER waves share a weight row (pair of rows); their sums are added in wave order. Between the two launches h stays in f32 (a few KB), so
// that y is rounded once. One row, 1280 x 5120: 6.1 us for 26 MB, 4.5 us for 13 MB (the weights partly in the last-level cache), two launches.
// ------------------------------------------------------------------------------------------------------------------------------------
constexpr int TOKENS = 4;
template <bool F16, int MT, int PER, bool GATE>
__global__ __launch_bounds__(256) void ffn_token_kernel(MmArgs p, float* h) {
    T16<F16>::enter();
    __shared__ float sums[4][2 * MT];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int n = blockIdx.x * (4 / PER) + wave / PER, part = wave % PER;
    const int N = GATE ? p.F : p.N;
    float s[GATE ? 2 : 1][MT] = {};
    if (n < N) {
        const uint16_t* w0 = p.B + (int64_t)n * p.ldb;
        const uint16_t* w1 = GATE ? p.B2 + (int64_t)n * p.ldb : nullptr;
#pragma unroll 4
        for (int k = (part * 64 + lane) * 8; k < p.K; k += PER * 512) {
            const uint4 a = *reinterpret_cast<const uint4*>(w0 + k);
            uint4 b = a;
            if constexpr (GATE) b = *reinterpret_cast<const uint4*>(w1 + k);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if constexpr (GATE) {
                    const uint4 x = *reinterpret_cast<const uint4*>(p.A + (int64_t)min(t, p.M - 1) * p.lda + k);
                    s[0][t] = T16<F16>::dot2(x.w, a.w, T16<F16>::dot2(x.z, a.z, T16<F16>::dot2(x.y, a.y, T16<F16>::dot2(x.x, a.x, s[0][t]))));
                    s[1][t] = T16<F16>::dot2(x.w, b.w, T16<F16>::dot2(x.z, b.z, T16<F16>::dot2(x.y, b.y, T16<F16>::dot2(x.x, b.x, s[1][t]))));
                } else {
                    const float4* x = reinterpret_cast<const float4*>(h + (int64_t)min(t, p.M - 1) * p.K + k);
                    const float4 x0 = x[0], x1 = x[1];
                    float v = s[0][t];
                    v = __builtin_fmaf(x0.x, T16<F16>::lo(a.x), v); v = __builtin_fmaf(x0.y, T16<F16>::hi(a.x), v);
                    v = __builtin_fmaf(x0.z, T16<F16>::lo(a.y), v); v = __builtin_fmaf(x0.w, T16<F16>::hi(a.y), v);
                    v = __builtin_fmaf(x1.x, T16<F16>::lo(a.z), v); v = __builtin_fmaf(x1.y, T16<F16>::hi(a.z), v);
                    v = __builtin_fmaf(x1.z, T16<F16>::lo(a.w), v); v = __builtin_fmaf(x1.w, T16<F16>::hi(a.w), v);
                    s[0][t] = v;
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < (GATE ? 2 : 1); ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int o = 32; o; o >>= 1) s[j][t] += __shfl_xor(s[j][t], o);
    if constexpr (PER > 1) {
        if (lane == 0) {
#pragma unroll
            for (int t = 0; t < MT; ++t) { sums[wave][t] = s[0][t]; if constexpr (GATE) sums[wave][MT + t] = s[1][t]; }
        }
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int w = 1; w < PER; ++w)
#pragma unroll
            for (int t = 0; t < MT; ++t) { s[0][t] += sums[wave + w][t]; if constexpr (GATE) s[1][t] += sums[wave + w][MT + t]; }
    }
    if (n >= N || lane != 0) return;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        if (t >= p.M) break;
        float o = s[0][t] + (p.bias ? T16<F16>::to_f32(p.bias[n]) : 0.f);
        if constexpr (GATE) {
            const float u = s[1][t] + (p.bias2 ? T16<F16>::to_f32(p.bias2[n]) : 0.f);
            if (p.g) { p.g[(int64_t)t * p.F + n] = o; p.u[(int64_t)t * p.F + n] = u; }
            o = act_of(p.act, o) * u;
            h[(int64_t)t * p.F + n] = o;
        }
        if (!GATE || p.C) p.C[(int64_t)t * (GATE ? p.F : p.ldc) + n] = T16<F16>::from_f32(o);      // (GATE: only if h is saved)
    }
}

// column sums over 32 rows of a 16-bit matrix: part [ceil(M / 32)][N]; 64 columns x 8 at a time, 4 row lanes
template <bool F16>
__global__ __launch_bounds__(256) void ffn_colsum_kernel(const uint16_t* x, int64_t ld, int M, int N, float* part) {
    __shared__ float red[4][512];
    const int c = threadIdx.x & 63, rl = threadIdx.x >> 6, n = blockIdx.y * 512 + 8 * c, m0 = blockIdx.x * 32;
    float s[8] = {};
    if (n < N) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int m = m0 + 4 * r + rl;
            if (m >= M) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(x + m * ld + n);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) { s[2 * e] += T16<F16>::lo(w[e]); s[2 * e + 1] += T16<F16>::hi(w[e]); }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) red[rl][8 * c + e] = s[e];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int l = threadIdx.x + 256 * k, col = blockIdx.y * 512 + l;
        if (col < N) part[(int64_t)blockIdx.x * N + col] = red[0][l] + red[1][l] + red[2][l] + red[3][l];
    }
}
// bias gradients from the sums over 32 rows: columns of cs [parts][2 F] (gate, up), then of cd [parts][D] (down); 16 columns x 16 part lanes
template <bool F16>
__global__ __launch_bounds__(256) void ffn_bias_kernel(const float* cs, const float* cd, int parts, int F, int D, uint16_t* dbg, uint16_t* dbu, uint16_t* dbd) {
    T16<F16>::enter();
    __shared__ float red[16][16];
    const int cl = threadIdx.x & 15, pl = threadIdx.x >> 4, i = blockIdx.x * 16 + cl, n2 = dbg ? 2 * F : 0;
    const bool down = i >= n2;
    const int n = down ? D : 2 * F, c = down ? i - n2 : i;
    const float* p = (down ? cd : cs) + c;
    const bool in = c < n && (!down || dbd);
    float t = 0.f;
    if (in)
        for (int k = pl; k < parts; k += 16) t += p[(int64_t)k * n];
    red[pl][cl] = t;
    __syncthreads();
    if (pl != 0 || !in) return;
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) t += red[k][cl];
    (down ? dbd[c] : c < F ? dbg[c] : dbu[c - F]) = T16<F16>::from_f32(t);
}

// ------------------------------------------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------------------------------------------
// tile shapes: thin (32 x 64, four waves on the k-steps of a tile, four tiles in flight: the weights are the work, and many small workgroups
// read them; us forward, D = 1280, F = 5120: 32 rows 18 for mid's 30, 256 rows 36 for 41, at 600 rows it loses, 63 for 50), mid (128 x 128,
// two workgroups per CU), big (256 x 256, one workgroup of eight waves; half the LDS and L2 bytes per product, but only where its tiles
// fill the 256 CUs), tall (fused_tile)
enum { TILE_THIN, TILE_MID, TILE_BIG, TILE_TALL };
int tile_of(int la, int M, int N) {
    if (M <= 256 && la == 0) return TILE_THIN;         // (layout 1 keeps whole 128-byte rows of m in LDS: no thin form)
    return (int64_t)cdiv(M, 256) * cdiv(N, 256) >= 200 ? TILE_BIG : TILE_MID;
}
// GATE and DH finish a tile in their epilogue: k cannot be split, and a last round of the chip that is part full costs a whole one. They take
// the tile whose rounds together are shortest -- rounds x a CU's work per round, with mid's products a quarter dearer than big's; tall (192 x
// 256) is there for what leaves big a nearly empty round (us, forward with saving + backward, before and with this rule: 4111 rows, 640 x 2560:
// 254 and 241; 2000, 1280 x 5120: 366 and 335; 12000, 256 x 1024: 182 and 175; 8192, 512 x 2048, where big fits: 300 and 295).
int fused_tile(int M, int N) {
    if (M <= 256) return TILE_THIN;
    const auto rounds = [&](int bm, int bn, int places) { return ((int64_t)cdiv(M, bm) * cdiv(N, bn) + places - 1) / places; };
    const int64_t mid = rounds(128, 128, 512) * 10, big = rounds(256, 256, 256) * 16, tall = rounds(192, 256, 256) * 12;
    return mid < big && mid < tall ? TILE_MID : tall < big ? TILE_TALL : TILE_BIG;
}
// How an OUT product shares out k. Tiles that do not fill the chip once: every tile in `splits` parts. Tiles that leave a part round behind
// whole ones: the tail's tiles in as many parts as fill it, if that is at most 5 / 8 full (7680 x 1280 from 5120: 600 tiles on 512 places,
// 148 -> 125 us).
struct OutPlan { int splits = 1, full = 0, tail = 0, tail_splits = 0; size_t bytes = 0; };
OutPlan plan_out(int la, int M, int N, int kts) {
    const int t = tile_of(la, M, N), bm = t == TILE_THIN ? 32 : t == TILE_MID ? 128 : 256, bn = t == TILE_BIG ? 256 : t == TILE_THIN ? 64 : 128;
    const int64_t tiles = (int64_t)cdiv(M, bm) * cdiv(N, bn);
    const int places = t == TILE_BIG ? 256 : 512;
    OutPlan p;
    int s = (int)std::min<int64_t>(t == TILE_BIG ? 1 : places / tiles, std::max(1, kts / (t == TILE_THIN ? 16 : 4)));
    s = std::max(1, std::min(s, 16));
    p.splits = cdiv(kts, cdiv(kts, s));
    if (p.splits > 1) {
        p.bytes = (size_t)p.splits * M * N * 4;
        return p;
    }
    const int tail = (int)(tiles % places);
    if (t == TILE_THIN || tiles < places || tail == 0 || tail > places * 5 / 8) return p;
    const int ts = std::min(std::min(places / tail, kts / 8), 8);
    if (ts < 2) return p;
    p.tail = tail;
    p.full = (int)(tiles - tail);
    p.tail_splits = cdiv(kts, cdiv(kts, ts));
    p.bytes = (size_t)p.tail * p.tail_splits * bm * bn * 4;
    return p;
}

template <bool F16, int BM, int BN, int NWM, int NWN, int NWK, int NBUF, int LA, int LB, int EPI>
int mm_run(MmArgs p, const char* name, hipStream_t st) {
    constexpr size_t lds = NBUF * (BM + BN) * BK * 2;
    p.tiles_m = cdiv(p.M, BM);
    p.tiles_n = cdiv(p.N, BN);
    const int64_t n = p.tail > 0 ? p.full + 8 * cdiv(p.tail * p.tail_splits, 8) : (int64_t)p.tiles_m * p.tiles_n * p.splits;
    ISB_REQUIRE((n + 7) * (NWM * NWN * NWK * 64) < (1ll << 32), ISB_ERR_INVALID, "gated feed-forward: %lld workgroups are more than one launch holds", (long long)n);
    p.n_items = (int)n;
    const int kts = cdiv(p.K, BK) * p.nseg;
    p.kt_per_split = cdiv(kts, p.splits);
    if (p.tail > 0) {
        p.tail_per = cdiv(p.tail * p.tail_splits, 8);
        p.kt_per_tail = cdiv(kts, p.tail_splits);
    }
    ISB_TRY((allow_lds<ffn_mm_kernel<F16, BM, BN, NWM, NWN, NWK, NBUF, LA, LB, EPI>>(lds)));
    ffn_mm_kernel<F16, BM, BN, NWM, NWN, NWK, NBUF, LA, LB, EPI><<<(unsigned)(8 * ((n + 7) / 8)), NWM * NWN * NWK * 64, lds, st>>>(p);
    ISB_LAUNCHED(name, st);
    if constexpr (EPI == EPI_OUT && BM >= 128) {
        if (p.tail > 0) {
            ffn_tail_kernel<F16, BM, BN><<<(unsigned)p.tail * (BM * BN / 1024), 256, 0, st>>>(p);
            ISB_LAUNCHED("ffn_tail", st);
        }
    }
    return ISB_OK;
}
template <bool F16, int LA, int LB, int EPI>
int mm(const MmArgs& p, const char* name, hipStream_t st) {
    const int t = EPI == EPI_OUT ? tile_of(LA, p.M, p.N) : fused_tile(p.M, p.N);
    if constexpr (EPI != EPI_OUT)
        if (t == TILE_TALL) return mm_run<F16, 192, 256, 2, 4, 1, 2, LA, LB, EPI>(p, name, st);
    if constexpr (LA == 0)
        if (t == TILE_THIN) return mm_run<F16, 32, 64, 1, 1, 4, 4, LA, LB, EPI>(p, name, st);
    if (t == TILE_MID) return mm_run<F16, 128, 128, 2, 2, 1, 2, LA, LB, EPI>(p, name, st);
    return mm_run<F16, 256, 256, 2, 4, 1, 2, LA, LB, EPI>(p, name, st);
}
// C = A B^T (+ bias), k split where the tiles alone leave CUs idle: into `part`, to be added up as `sum` says
template <bool F16, int LA, int LB>
int mm_out(MmArgs p, unsigned char* part, Sums::One& sum, const char* name, hipStream_t st) {
    const OutPlan plan = plan_out(LA, p.M, p.N, cdiv(p.K, BK) * p.nseg);
    p.splits = plan.splits;
    p.full = plan.full;
    p.tail = plan.tail;
    p.tail_splits = plan.tail_splits;
    p.part = reinterpret_cast<float*>(part);
    ISB_TRY((mm<F16, LA, LB, EPI_OUT>(p, name, st)));
    const int64_t n4 = (int64_t)p.M * p.N / 4;
    sum = {p.part, p.bias, p.C, n4, p.N, p.splits, p.splits > 1 ? (int)((n4 + 255) / 256) : 0};
    return ISB_OK;
}
template <bool F16>
int add_up(Sums& s, hipStream_t st) {
    if (s.blocks() == 0) return ISB_OK;
    ffn_sum_kernel<F16><<<(unsigned)s.blocks(), 256, 0, st>>>(s);
    ISB_LAUNCHED("ffn_sum", st);
    s = Sums{};
    return ISB_OK;
}
size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t part_bytes(int la, int M, int N, int kts) { return up256(plan_out(la, M, N, kts).bytes); }
// the exponents of [rows, cols] values (Powers)
size_t exp_bytes(int rows, int cols) { return up256((size_t)cdiv(cols, 32) * cdiv(rows, 32) * 4); }

template <bool F16, int MT, bool GATE>
int token(const MmArgs& p, float* h, hipStream_t st) {
    const int n = GATE ? p.F : p.N;
    if (p.K > 2048) ffn_token_kernel<F16, MT, 4, GATE><<<n, 256, 0, st>>>(p, h);
    else ffn_token_kernel<F16, MT, 1, GATE><<<cdiv(n, 4), 256, 0, st>>>(p, h);
    ISB_LAUNCHED("ffn_token", st);
    return ISB_OK;
}

// Where the partial sums of the backward pass's three products lie. Together, one launch adds them all up (us of the pass, a launch each and
// together: 600 rows, 512 x 2048: 74, 63; 1030, 640 x 2560: 91, 84) -- as long as they and what else passes between the launches (14 bytes for
// each value of h) stay well inside the 256 MB last-level cache: at 4111 rows, 237 MB, dh takes 52 for 44 us and the shared launch gains 3.
struct BwdParts {
    size_t at[3] = {}, bytes = 0;
    bool together = false;
    explicit BwdParts(const FfnArgs& a) {
        const size_t n[3] = {part_bytes(0, a.M, a.D, 2 * cdiv(a.F, BK)), part_bytes(1, 2 * a.F, a.D, cdiv(a.M, BK)), part_bytes(1, a.D, a.F, cdiv(a.M, BK))};
        together = 14 * (size_t)a.M * a.F + n[0] + n[1] + n[2] <= (160u << 20);
        if (together) { at[1] = n[0]; at[2] = n[0] + n[1]; }
        for (int i = 0; i < 3; ++i) bytes = std::max(bytes, at[i] + n[i]);
    }
};

template <bool F16>
int fwd(const FfnArgs& a, unsigned char* ws, hipStream_t st) {
    uint16_t* h = a.h;
    if (!h && a.M > TOKENS) {
        h = reinterpret_cast<uint16_t*>(ws);
        ws += up256((size_t)a.M * a.F * 2);
    }
    int8_t* ex = nullptr;
    if (F16 && a.M > TOKENS) {
        ex = reinterpret_cast<int8_t*>(ws);
        ws += exp_bytes(a.M, a.F);
    }
    MmArgs g{};
    g.A = a.x; g.B = a.wg; g.B2 = a.wu; g.lda = a.x_s; g.ldb = a.D;
    g.M = a.M; g.N = 64 * cdiv(a.F, 32); g.K = a.D; g.F = a.F; g.nseg = 1; g.splits = 1;
    g.bias = a.bg; g.bias2 = a.bu; g.C = h; g.g = a.g; g.u = a.u; g.act = a.act; g.ex = ex;
    MmArgs d{};
    d.A = h; d.B = a.wd; d.lda = a.F; d.ldb = a.F;
    d.M = a.M; d.N = a.D; d.K = a.F; d.nseg = 1; d.splits = 1;
    d.bias = a.bd; d.C = a.y; d.ldc = a.D; d.xa = ex;
    if (a.M <= TOKENS) {
        float* hf = reinterpret_cast<float*>(ws);
        if (a.M == 1) {
            ISB_TRY((token<F16, 1, true>(g, hf, st)));
            return token<F16, 1, false>(d, hf, st);
        }
        ISB_TRY((token<F16, TOKENS, true>(g, hf, st)));
        return token<F16, TOKENS, false>(d, hf, st);
    }
    ISB_TRY((mm<F16, 0, 0, EPI_GATE>(g, "ffn gate + up", st)));
    Sums s{};
    ISB_TRY((mm_out<F16, 0, 0>(d, ws, s.of[0], "ffn down", st)));
    return add_up<F16>(s, st);
}

template <bool F16>
int bwd(const FfnArgs& a, unsigned char* ws, hipStream_t st) {
    uint16_t* dgu = reinterpret_cast<uint16_t*>(ws);
    unsigned char* rest = ws + up256((size_t)a.M * 2 * a.F * 2);
    // fp16: DH finds the groups of the saved h that carry powers of two, or were cut off at 65504 (one to four rows), from the pre-activations -- with
    // a margin for its own rounding, so none is missed --, and puts its own value in their place. The table is not saved: the next call finds the same.
    int8_t *ex_h = nullptr, *ex_d = nullptr;
    if (F16) {
        ex_h = reinterpret_cast<int8_t*>(rest);
        rest += exp_bytes(a.M, a.F);
        ex_d = reinterpret_cast<int8_t*>(rest);
        rest += 2 * exp_bytes(a.M, a.F);
    }
    float* part = reinterpret_cast<float*>(rest);
    MmArgs p{};
    // dG, dU from dh = dy Wd
    p.A = a.dy; p.B = a.wd; p.lda = a.dy_s; p.ldb = a.F; p.M = a.M; p.N = a.F; p.K = a.D; p.nseg = 1; p.splits = 1;
    p.g = a.g; p.u = a.u; p.F = a.F; p.act = a.act; p.C = dgu; p.ldc = 2 * (int64_t)a.F;
    p.h = a.h; p.ex_h = ex_h; p.ex = ex_d;
    // (the bias gradients' partial sums use the place of the products' partial results before those need it)
    const int parts = cdiv(a.M, 32);
    float* down = part + (a.dbg ? (int64_t)parts * 2 * a.F : 0);
    p.cs = a.dbg ? part : nullptr;
    ISB_TRY((mm<F16, 0, 1, EPI_DH>(p, "ffn dh", st)));
    if (a.dbd) {
        ffn_colsum_kernel<F16><<<dim3(parts, cdiv(a.D, 512)), 256, 0, st>>>(a.dy, a.dy_s, a.M, a.D, down);
        ISB_LAUNCHED("ffn_colsum", st);
    }
    if (a.dbg || a.dbd) {
        const int cols = (a.dbg ? 2 * a.F : 0) + (a.dbd ? a.D : 0);
        ffn_bias_kernel<F16><<<cdiv(cols, 16), 256, 0, st>>>(part, down, parts, a.F, a.D, a.dbg, a.dbu, a.dbd);
        ISB_LAUNCHED("ffn_bias", st);
    }
    // dx = dG Wg + dU Wu
    p = MmArgs{};
    p.A = dgu; p.B = a.wg; p.B2 = a.wu; p.lda = 2 * (int64_t)a.F; p.ldb = a.D; p.M = a.M; p.N = a.D; p.K = a.F; p.nseg = 2;
    p.C = a.dx; p.ldc = a.D; p.xa = ex_d;
    const BwdParts parts_at(a);
    Sums s{};
    ISB_TRY((mm_out<F16, 0, 1>(p, rest + parts_at.at[0], s.of[0], "ffn dx", st)));
    if (!parts_at.together) ISB_TRY(add_up<F16>(s, st));
    // [dWg; dWu] = [dG | dU]^T x
    p = MmArgs{};
    p.A = dgu; p.B = a.x; p.lda = 2 * (int64_t)a.F; p.ldb = a.x_s; p.M = 2 * a.F; p.N = a.D; p.K = a.M; p.nseg = 1;
    p.C = a.dwgu; p.ldc = a.D; p.xa = ex_d; p.F = a.F;
    ISB_TRY((mm_out<F16, 1, 1>(p, rest + parts_at.at[1], s.of[1], "ffn dW gate, up", st)));
    if (!parts_at.together) ISB_TRY(add_up<F16>(s, st));
    // dWd = dy^T h
    p = MmArgs{};
    p.A = a.dy; p.B = a.h; p.xb = ex_h; p.lda = a.dy_s; p.ldb = a.F; p.M = a.D; p.N = a.F; p.K = a.M; p.nseg = 1;
    p.C = a.dwd; p.ldc = a.F;
    ISB_TRY((mm_out<F16, 1, 1>(p, rest + parts_at.at[2], s.of[2], "ffn dW down", st)));
    return add_up<F16>(s, st);
}
}  // namespace

size_t ffn_workspace(const FfnArgs& a, bool f16, bool backward) {
    const size_t M = a.M, F = a.F;
    if (!backward) {
        if (a.M <= TOKENS) return M * F * 4;
        const size_t h = a.h ? 0 : up256(M * F * 2);
        return h + (f16 ? exp_bytes(a.M, a.F) : 0) + part_bytes(0, a.M, a.D, cdiv(a.F, BK));
    }
    const size_t sums = (size_t)cdiv(a.M, 32) * ((a.dbg ? 2 * F : 0) + (a.dbd ? a.D : 0)) * 4;
    const size_t part = std::max(sums, BwdParts(a).bytes);
    return up256(M * 2 * F * 2) + (f16 ? 3 * exp_bytes(a.M, a.F) : 0) + part;
}
int launch_ffn_fwd(const FfnArgs& a, bool f16, unsigned char* ws, hipStream_t st) { return f16 ? fwd<true>(a, ws, st) : fwd<false>(a, ws, st); }
int launch_ffn_bwd(const FfnArgs& a, bool f16, unsigned char* ws, hipStream_t st) { return f16 ? bwd<true>(a, ws, st) : bwd<false>(a, ws, st); }

}  // namespace isb
