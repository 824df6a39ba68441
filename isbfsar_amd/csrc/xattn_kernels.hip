// Cross attention of query rows to an encoder's states of another length: forward (rows in tiles, or few rows with the states split over
// waves and workgroups) and backward. Softmax statistics, sums and partial results are 32-bit; the attention weights and dS are rounded to
// the tensors' 16-bit type where they enter a matrix product (half a step, the same size as the rounding of the results).
//
// One identity carries all kernels: a 32x32x16 product's accumulator holds, per lane, ONE column and the 16 rows 8 (i / 4) + 4 h + i % 4
// (h = lane / 32). Computing S^T = K Q^T (column = query row) makes the softmax lane-local, and its registers 8 s ... 8 s + 7 ARE the B
// operand of the next product over the states if the other operand lists the summed index in the same order -- which the transposing LDS
// read does for free (frag_cols<W, 4, 8>). P never leaves its registers.
#include <algorithm>
#include <cmath>

#include "blocks.h"

namespace isb {
namespace {

constexpr int KT = 64;                    // states per tile
constexpr int FEW_STATES = KT;            // up to these many P and dS enter products with their rests (rest8)
constexpr float NEG_INF = -__builtin_inff();

// element offset of row r of group (bk, hk) in a [B, Lq, Hq, .] tensor with strides sb, sl, sh
struct RowAt { int b, i, hq; };
__device__ __forceinline__ RowAt row_at(const XattnArgs& a, int bk, int hk, int r) {
    const uint32_t s = a.by_lqg.div(r), rem = r - s * a.by_lqg.d, i = a.by_g.div(rem);
    return {bk * a.nb + (int)s, (int)i, hk * a.G + (int)(rem - i * a.by_g.d)};
}
__device__ __forceinline__ int64_t off_at(const RowAt& p, int64_t sb, int64_t sl, int64_t sh) { return p.b * sb + p.i * sl + p.hq * sh; }
__device__ __forceinline__ int64_t off_out(const XattnArgs& a, const RowAt& p) { return (((int64_t)p.b * a.Lq + p.i) * a.Hq + p.hq) * a.D; }
__device__ __forceinline__ int64_t off_lse(const XattnArgs& a, const RowAt& p) { return ((int64_t)p.b * a.Hq + p.hq) * a.Lq + p.i; }

__device__ __forceinline__ int states_of(const XattnArgs& a, int bk) { return a.kv_len ? min(max(a.kv_len[bk], 0), a.Lk) : a.Lk; }

// byte of lane's state in the mask (0 = masked or absent); the ballot of tile_bits makes the tile's validity one scalar
__device__ __forceinline__ uint32_t mask_byte(const XattnArgs& a, int bk, int key, int k1) {
    if (key >= k1) return 0;
    return a.mask ? a.mask[bk * a.mask_sb + key] : 1u;
}

// fragment of a row held in global memory (zeros past D): lane half h, k-step ks
__device__ __forceinline__ uint4 row_frag(const uint16_t* p, int ks, int h, int D, bool ok) {
    const int c = 16 * ks + 8 * h;
    return ok && c < D ? *reinterpret_cast<const uint4*>(p + c) : make_uint4(0, 0, 0, 0);
}

// ---- requests of one tile of ROWS states x DT values by NW waves; voff[] holds the lane's byte offsets (DMA_NONE past D)
template <int DT, int ROWS, int NW>
struct TileLoad {
    static constexpr int PIECES = ROWS * DT * 2 / 1024 / NW;      // 1-KiB requests per wave
    uint32_t voff[PIECES];
    int row[PIECES];
    __device__ __forceinline__ void init(int wave, int lane, int64_t sl, int D) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
            const int byte = (wave * PIECES + j) * 1024 + lane * 16, r = byte / (DT * 2);
            const int c = ((byte % (DT * 2)) >> 4) ^ tile_xor<DT>(r);
            row[j] = r;
            voff[j] = c * 8 < D ? (uint32_t)(r * (int)sl * 2 + c * 16) : DMA_NONE;
        }
    }
    // all: every state of the tile is valid
    __device__ __forceinline__ void request(const uint16_t* base, bool all, uint64_t bits, uint32_t lds, int wave) const {
        const i32x4 d = dma_desc(base);
        if (all) {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) dma16_desc(d, voff[j], lds + (wave * PIECES + j) * 1024);
        } else {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                const uint32_t none = (uint32_t)((bits >> row[j]) & 1) - 1u;         // all ones where the state is masked: past the buffer's end
                dma16_desc(d, voff[j] | none, lds + (wave * PIECES + j) * 1024);
            }
        }
    }
};

// Masked states enter as the accumulators' start: their lane of `bias` (LDS, a float per state of the tile) holds -inf, the others 0, so a
// masked score costs the softmax no instruction (masked K rows are zeros: -inf + 0 stays).
__device__ __forceinline__ void start_scores(f32x16& s, const float* bias, bool all, int h) {
    if (all) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 0.f;
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float4 v = *reinterpret_cast<const float4*>(bias + 8 * q + 4 * h);
            s[4 * q] = v.x; s[4 * q + 1] = v.y; s[4 * q + 2] = v.z; s[4 * q + 3] = v.w;
        }
    }
}
__device__ __forceinline__ void put_bias(float* bias, int n, uint32_t byte, bool all, int lane) {
    if (!all && lane < n) bias[lane] = byte ? 0.f : NEG_INF;
}

// LDS reads and matrix products keep the order they are written in (vector and scalar arithmetic may move): a fragment is read several
// products before its own, which hides the read's latency also where a SIMD has only one or two waves. Left to itself the compiler reads one
// product ahead.
__device__ __forceinline__ void reads_stay() { __builtin_amdgcn_sched_barrier(0x6); }

// fp16: P is formed as 2^12 P, so that weights down to 2^-26 of a row's largest stay normal numbers (many small ones can make up the result, next to
// a large one with a small value: rounded to steps of 2^-24, 20000 weights of 2^-24.5 came out 44 % too large). bf16 has f32's range.
template <bool F16> constexpr float P_UP = F16 ? 12.0f : 0.0f;              // log2 of the factor on P
template <bool F16> constexpr float P_LAG = F16 ? 3.0f : 8.0f;

template <bool F16>
__device__ __forceinline__ uint4 pack8(const f32x16& x, int t) {
    return t == 0 ? make_uint4(T16<F16>::pack2(x[0], x[1]), T16<F16>::pack2(x[2], x[3]), T16<F16>::pack2(x[4], x[5]), T16<F16>::pack2(x[6], x[7]))
                  : make_uint4(T16<F16>::pack2(x[8], x[9]), T16<F16>::pack2(x[10], x[11]), T16<F16>::pack2(x[12], x[13]), T16<F16>::pack2(x[14], x[15]));
}
// What that rounds off, as a second operand. Where a sum has few terms (up to FEW_STATES states; up to 32 rows for dQ, 64 for dK, dV) the roundings of P and dS do not average
// out: they scale whole rows of V, K, dout or Q, and the results are as far off as with roundings of their own, or further. There both operands
// enter (hi + lo: 2^-16 or better), which costs a few products of a launch that waits for its loads. An infinity of V or dout times a rest of 0 would be
// a NaN: where one comes out (any_nan) the wave adds up once more without the rests.
template <bool F16>
__device__ __forceinline__ uint4 rest8(const f32x16& x, int t, const uint4& hi) {
    const uint32_t w[4] = {hi.x, hi.y, hi.z, hi.w};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float a = t == 0 ? x[2 * i] : x[8 + 2 * i], b = t == 0 ? x[2 * i + 1] : x[9 + 2 * i];
        r[i] = T16<F16>::pack2(a - T16<F16>::lo(w[i]), b - T16<F16>::hi(w[i]));
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

template <int NA>
__device__ __forceinline__ bool any_nan(const f32x16 (&acc)[NA]) {
    bool n = false;
#pragma unroll
    for (int d = 0; d < NA; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) n |= acc[d][i] != acc[d][i];
    return __any(n);
}
template <int NA>
__device__ __forceinline__ void clear(f32x16 (&acc)[NA]) {
#pragma unroll
    for (int d = 0; d < NA; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
}

// One block of NB x 32 states for 32 rows (a column of S^T each): scores, running maximum (m: less P_UP) and sum, O^T += V^T P^T.
// The maximum follows lazily: O^T is rescaled only when a row's maximum grows by more than P_LAG (base-2 units), so P <= 2^15 (fp16), 2^8.
// FEW: with the rest of P (rest8).
template <bool F16, int DT, int NB, bool FEW = false>
__device__ __forceinline__ void attend(const unsigned char* kt, const unsigned char* vt, const uint4 (&qf)[DT / 16], f32x16 (&acc)[DT / 32],
                                       float& m, float& l, float c, const float* bias, bool all, int lane) {
    const int h = lane >> 5;
    constexpr int KS = DT / 16;
    f32x16 s[NB];
    uint4 kf[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) kf[ks] = frag_rows<DT>(kt, 0, ks, lane);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        start_scores(s[b], bias + 32 * b, all, h);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            s[b] = T16<F16>::mfma32(kf[ks], qf[ks], s[b]);
            if (b + 1 < NB) kf[ks] = frag_rows<DT>(kt, 32 * (b + 1), ks, lane);       // the next block's fragment behind this one's product
            reads_stay();
        }
    }
    float mx = NEG_INF;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[b][i]);
    mx = max_halves(mx) * c;
    if (__any(mx > m + (P_UP<F16> + P_LAG<F16>))) {
        const float mn = fmaxf(m, mx - P_UP<F16>);
        const float al = __builtin_amdgcn_exp2f(m - (mn == NEG_INF ? 0.f : mn));
        l *= al;
#pragma unroll
        for (int d = 0; d < DT / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] *= al;
        m = mn;
    }
    // the first fragments of V^T travel while the weights are formed
    constexpr int NT = 2 * NB, NV = NT * (DT / 32), AHEAD = 4;
    uint4 vf[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) vf[i] = frag_cols<DT, 4, 8>(vt, 16 * (i % NT), 32 * (i / NT), lane);
    reads_stay();
    const float mu = m == NEG_INF ? 0.f : m;
    uint4 p[2 * NB];
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s[b][8 * t + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][8 * t + i], c, -mu));
                sum += s[b][8 * t + i];
            }
            p[2 * b + t] = pack8<F16>(s[b], t);
        }
    l += sum;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        acc[i / NT] = T16<F16>::mfma32(vf[i % AHEAD], p[i % NT], acc[i / NT]);
        if constexpr (FEW) acc[i / NT] = T16<F16>::mfma32(vf[i % AHEAD], rest8<F16>(s[i % NT / 2], i % 2, p[i % NT]), acc[i / NT]);
        if (i + AHEAD < NV) vf[i % AHEAD] = frag_cols<DT, 4, 8>(vt, 16 * ((i + AHEAD) % NT), 32 * ((i + AHEAD) / NT), lane);
        reads_stay();
    }
}

// four columns of a row's results (and, `first`, what goes with the row): out and lse, or (splits) its unnormalised sums with maximum and sum
template <bool F16, int DT>
__device__ __forceinline__ void store_piece(const XattnArgs& a, int bk, int hk, int split, int r, int c, float4 o, float m, float l, bool first, float one) {
    if (r >= a.M) return;
    if (a.splits > 1) {
        const int64_t at = ((int64_t)split * a.Bk * a.Hk + bk * a.Hk + hk) * a.M + r;
        *reinterpret_cast<float4*>(a.part + at * DT + c) = o;
        if (first) *reinterpret_cast<float2*>(a.part2 + at * 2) = make_float2(m, l);
        return;
    }
    const RowAt w = row_at(a, bk, hk, r);
    const float inv = l == 0.f ? 0.f : one / l;
    if (c < a.D) *reinterpret_cast<uint2*>(a.out + off_out(a, w) + c) = make_uint2(T16<F16>::pack2(o.x * inv, o.y * inv), T16<F16>::pack2(o.z * inv, o.w * inv));
    if (first) a.lse[off_lse(a, w)] = l == 0.f ? NEG_INF : (m + __builtin_amdgcn_logf(l)) * LN2;
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Forward, many rows: a workgroup takes 128 rows (32 per wave) of one group and walks the states in tiles of 64; K and V tiles arrive by
// LDS-DMA, the next ones while this one is used (two buffers, one barrier per tile). Two workgroups per CU: one's softmax stands beside the
// other's products. 2 x 16 heads, 4096 rows and states: 292 us 128 wide (940 TFLOP/s, bf16), 179 us 64 wide (770, fp16: as many exponentials
// for half the products); no single unit bounds it (without the exponentials 1087, the requests 1067, P V 1244).
// ------------------------------------------------------------------------------------------------------------------------------------
template <bool F16, int DT>
__global__ __launch_bounds__(256, 2) void xattn_fwd_kernel(XattnArgs a) {
    const int item = xcd_item(blockIdx.x, a.n_items);
    if (item >= a.n_items) return;
    const int rt = item % a.tiles, split = item / a.tiles % a.splits, grp = item / a.tiles / a.splits, bk = grp / a.Hk, hk = grp % a.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    const int r = rt * 128 + wave * 32 + (lane & 31);
    constexpr int TB = KT * DT * 2, STAGE = 2 * TB + KT * 4;

    const int len = states_of(a, bk), k0 = split * a.chunk, k1 = min(len, k0 + a.chunk);
    int nt = k1 > k0 ? (k1 - k0 + KT - 1) / KT : 0;

    uint4 qf[DT / 16];
    {
        const RowAt w = row_at(a, bk, hk, min(r, a.M - 1));
        const uint16_t* q = a.q + off_at(w, a.q_sb, a.q_sl, a.q_sh);
#pragma unroll
        for (int ks = 0; ks < DT / 16; ++ks) qf[ks] = row_frag(q, ks, h, a.D, r < a.M);
    }
    f32x16 acc[DT / 32];
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    float m = NEG_INF, l = 0.f;

    const uint16_t* kb = a.k + bk * a.k_sb + hk * a.k_sh + (int64_t)k0 * a.k_sl;
    const uint16_t* vb = a.v + bk * a.v_sb + hk * a.v_sh + (int64_t)k0 * a.v_sl;
    const uint32_t lds0 = lds_addr_of(conv_lds_dyn);
    TileLoad<DT, KT, 4> lk, lv;
    lk.init(wave, lane, a.k_sl, a.D);
    lv.init(wave, lane, a.v_sl, a.D);
    uint64_t bits = 0, next = 0;
    uint32_t byte = 0;
    auto request = [&](int t, uint64_t valid, uint32_t at) {
        const bool all = valid == ~0ull;
        lk.request(kb + (int64_t)t * KT * a.k_sl, all, valid, lds0 + at, wave);
        lv.request(vb + (int64_t)t * KT * a.v_sl, all, valid, lds0 + at + TB, wave);
        if (wave == 0) put_bias(reinterpret_cast<float*>(conv_lds_dyn + at + 2 * TB), KT, byte, all, lane);
        byte = mask_byte(a, bk, k0 + (t + 1) * KT + lane, k1);
    };
    if (nt > 0) {
        byte = mask_byte(a, bk, k0 + lane, k1);
        bits = __ballot(byte != 0);
        request(0, bits, 0);
    }
    if (nt == 1 && len <= FEW_STATES) {
        wait_all_and_meet();
        const auto few = [&](auto rests) {
            for (int b = 0; b < 2; ++b)
                if (bits >> (32 * b) & 0xffffffffu)
                    attend<F16, DT, 1, decltype(rests)::value>(conv_lds_dyn + 32 * b * DT * 2, conv_lds_dyn + TB + 32 * b * DT * 2, qf, acc, m, l, a.c,
                                                               reinterpret_cast<const float*>(conv_lds_dyn + 2 * TB) + 32 * b, bits == ~0ull, lane);
        };
        few(std::true_type());
        if (any_nan(acc)) {
            clear(acc);
            m = NEG_INF;
            l = 0.f;
            few(std::false_type());
        }
        nt = 0;
    }
    for (int t = 0; t < nt; ++t) {
        next = __ballot(byte != 0);
        wait_all_and_meet();
        const uint32_t cur = (t & 1) * STAGE, oth = STAGE - cur;
        if (t + 1 < nt) request(t + 1, next, oth);
        const float* bias = reinterpret_cast<const float*>(conv_lds_dyn + cur + 2 * TB);
        if (bits != 0) attend<F16, DT, 2>(conv_lds_dyn + cur, conv_lds_dyn + cur + TB, qf, acc, m, l, a.c, bias, bits == ~0ull, lane);
        bits = next;
    }
    const float one = saturate_from_here<F16>();
    l = sum_halves(l);
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            store_piece<F16, DT>(a, bk, hk, split, r, 32 * d + 8 * q + 4 * h, make_float4(acc[d][4 * q], acc[d][4 * q + 1], acc[d][4 * q + 2], acc[d][4 * q + 3]),
                                 m, l, d == 0 && q == 0 && h == 0, one);
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Forward, tiles of 32 rows (single tokens, grouped heads; a few windows): the states are the work. Eight waves walk their own blocks of 32
// states, each through its own LDS and without a barrier in the loop -- a wave waits for its block while the others use theirs --, and their
// sums meet at the end (few_rows says when). Up to 2048 states one workgroup does all of a group in one launch (4 heads x 1800 states x 64: 10.0 us, as long as five
// splits and their join; four waves with two buffers each: 9.6 in two launches, 28.9 for 24.0 where 128 groups of 128 wide fill the chip).
// ------------------------------------------------------------------------------------------------------------------------------------
constexpr int TOKEN_WAVES = 8;
template <bool F16, int DT>
__global__ __launch_bounds__(TOKEN_WAVES * 64, TOKEN_WAVES / 4) void xattn_token_kernel(XattnArgs a) {
    constexpr int NW = TOKEN_WAVES;
    const int item = xcd_item(blockIdx.x, a.n_items);
    if (item >= a.n_items) return;
    const int rt = item % a.tiles, split = item / a.tiles % a.splits, grp = item / a.tiles / a.splits, bk = grp / a.Hk, hk = grp % a.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5, r = lane & 31, row = rt * 32 + r;
    constexpr int TB = 32 * DT * 2;

    const int len = states_of(a, bk), k0 = split * a.chunk, k1 = min(len, k0 + a.chunk);
    const int nt = k1 > k0 ? (k1 - k0 + 31) / 32 : 0;                        // blocks of the workgroup; wave w takes w, w + NW, ...
    uint4 qf[DT / 16];
    {
        const RowAt w = row_at(a, bk, hk, min(row, a.M - 1));
        const uint16_t* q = a.q + off_at(w, a.q_sb, a.q_sl, a.q_sh);
#pragma unroll
        for (int ks = 0; ks < DT / 16; ++ks) qf[ks] = row_frag(q, ks, h, a.D, row < a.M);
    }
    f32x16 acc[DT / 32];
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    float m = NEG_INF, l = 0.f;

    const uint16_t* kb = a.k + bk * a.k_sb + hk * a.k_sh + (int64_t)k0 * a.k_sl;
    const uint16_t* vb = a.v + bk * a.v_sb + hk * a.v_sh + (int64_t)k0 * a.v_sl;
    unsigned char* own = conv_lds_dyn + wave * (2 * TB + 128);
    float* bias = reinterpret_cast<float*>(own + 2 * TB);
    const uint32_t lds0 = lds_addr_of(own);
    TileLoad<DT, 32, 1> lk, lv;
    lk.init(0, lane, a.k_sl, a.D);
    lv.init(0, lane, a.v_sl, a.D);
    uint32_t byte = 0, bits = 0;
    auto valid = [&](int t) -> uint32_t { return t < nt ? mask_byte(a, bk, k0 + 32 * t + (lane & 31), k1) : 0u; };
    auto request = [&](int t) {
        bits = (uint32_t)__ballot(byte != 0);
        const bool all = bits == ~0u;
        lk.request(kb + (int64_t)t * 32 * a.k_sl, all, bits, lds0, 0);
        lv.request(vb + (int64_t)t * 32 * a.v_sl, all, bits, lds0 + TB, 0);
        put_bias(bias, 32, byte, all, lane);
        byte = valid(t + NW);
    };
    byte = valid(wave);
    if (wave < nt) request(wave);
    int t = wave;
    if (len <= FEW_STATES && t < nt) {                                        // (at most one block per wave)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (bits != 0) attend<F16, DT, 1, true>(own, own + TB, qf, acc, m, l, a.c, bias, bits == ~0u, lane);
        if (any_nan(acc)) {
            clear(acc);
            m = NEG_INF;
            l = 0.f;
            attend<F16, DT, 1>(own, own + TB, qf, acc, m, l, a.c, bias, bits == ~0u, lane);
        }
        t = nt;
    }
    for (; t < nt; t += NW) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (bits != 0) attend<F16, DT, 1>(own, own + TB, qf, acc, m, l, a.c, bias, bits == ~0u, lane);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                    // the block is read before its place is requested again
        if (t + NW < nt) request(t + NW);
    }
    const float one = saturate_from_here<F16>();
    l = sum_halves(l);
    // join the waves: (m, l) of all, then every wave scales its sums to the common maximum and each adds up its share of the columns, in wave
    // order
    wait_all_and_meet();
    float* ml = reinterpret_cast<float*>(conv_lds_dyn);
    float* sums = ml + NW * 64;                                               // [NW][32][DT + 4]
    constexpr int SW = DT + 4;
    static_assert((NW * 64 + NW * 32 * SW) * 4 <= NW * (2 * TB + 1024), "the sums fit");
    if (h == 0) { ml[(wave * 32 + r) * 2] = m; ml[(wave * 32 + r) * 2 + 1] = l; }
    __syncthreads();
    float mm = NEG_INF, ll = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) mm = fmaxf(mm, ml[(w * 32 + r) * 2]);
    const float mu = mm == NEG_INF ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < NW; ++w) ll += ml[(w * 32 + r) * 2 + 1] * __builtin_amdgcn_exp2f(ml[(w * 32 + r) * 2] - mu);
    const float al = __builtin_amdgcn_exp2f(m - mu);
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4*>(sums + (wave * 32 + r) * SW + 32 * d + 8 * q + 4 * h) =
                make_float4(acc[d][4 * q] * al, acc[d][4 * q + 1] * al, acc[d][4 * q + 2] * al, acc[d][4 * q + 3] * al);
    __syncthreads();
    // piece (d, q): 8 columns (4 per lane half); wave w takes pieces w, w + NW, ...
#pragma unroll
    for (int i = 0; i < DT / 8 / NW; ++i) {
        const int piece = wave + i * NW, c = 8 * piece + 4 * h;
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float4 u = *reinterpret_cast<const float4*>(sums + (w * 32 + r) * SW + c);
            t.x += u.x; t.y += u.y; t.z += u.z; t.w += u.w;
        }
        store_piece<F16, DT>(a, bk, hk, split, row, c, t, mm, ll, piece == 0 && h == 0, one);
    }
}

// join the splits of a row in their order: DT / 4 lanes per row, four columns each; a lane weighs one split (or two, ...) and hands its
// weight round, so the loads of the partial sums do not wait for each other (512 rows x 4 splits 4.8 us, 15360 x 2 5.9)
template <bool F16, int DT>
__global__ __launch_bounds__(256) void xattn_join_kernel(XattnArgs a) {
    T16<F16>::enter();
    constexpr int L = DT / 4;
    const int64_t rows = (int64_t)a.Bk * a.Hk * a.M, row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    if (row >= rows) return;
    const int lane = threadIdx.x % L;
    float mm = NEG_INF;
    for (int s = lane; s < a.splits; s += L) mm = fmaxf(mm, a.part2[(s * rows + row) * 2]);
#pragma unroll
    for (int o = 1; o < L; o <<= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
    const float mu = mm == NEG_INF ? 0.f : mm;
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < a.splits; s0 += L) {
        float w = 0.f, wl = 0.f;
        if (s0 + lane < a.splits) {
            const float2 ml = *reinterpret_cast<const float2*>(a.part2 + ((s0 + lane) * rows + row) * 2);
            w = __builtin_amdgcn_exp2f(ml.x - mu);
            wl = w * ml.y;
        }
        const int n = min(L, a.splits - s0);
        const float* from = a.part + (s0 * rows + row) * DT + 4 * lane;
        for (int s = 0; s < n; s += 4) {                     // four partial sums on their way at once (past the last: the last again, not added)
            float4 p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(from + min(s + i, n - 1) * rows * DT);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ws = __shfl(w, s + i, L);
                if (s + i < n) {
                    l += __shfl(wl, s + i, L);
                    o.x = __builtin_fmaf(ws, p[i].x, o.x); o.y = __builtin_fmaf(ws, p[i].y, o.y);
                    o.z = __builtin_fmaf(ws, p[i].z, o.z); o.w = __builtin_fmaf(ws, p[i].w, o.w);
                }
            }
        }
    }
    const int grp = (int)(row / a.M);
    const RowAt w = row_at(a, grp / a.Hk, grp % a.Hk, (int)(row % a.M));
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    if (4 * lane < a.D)
        *reinterpret_cast<uint2*>(a.out + off_out(a, w) + 4 * lane) = make_uint2(T16<F16>::pack2(o.x * inv, o.y * inv), T16<F16>::pack2(o.z * inv, o.w * inv));
    if (lane == 0) a.lse[off_lse(a, w)] = l == 0.f ? NEG_INF : (mm + __builtin_amdgcn_logf(l)) * LN2;
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Backward. dQ first (a workgroup keeps 128 rows, forms their delta = rowsum(dout o out) and walks the states), then dK, dV (a workgroup keeps
// 128 states, 32 per wave, and walks the rows); one launch adds up the splits of all three. Every sum has a fixed order: no atomics.
//
// fp16: P is formed as 2^12 P (P_UP), and each column of dS carries a power of two chosen from what it meets: it starts so that the first block's
// largest |dS| lies in [2^10, 2^11) and is lowered, with the sums so far, when a block passes 2^15. bf16 has f32's range and needs neither.
// ------------------------------------------------------------------------------------------------------------------------------------

// Where a thread's row lies, RT rows further with every step. Where G divides RT and a sample holds at least RT rows, a step stays on the same
// head and passes at most one sample's end: two additions instead of two divisions and the products of three strides.
template <int RT>
struct RowWalk {
    int64_t q, d;                  // offsets in q and dout
    int i, r, lse;                 // position, row, index into lse
    __device__ __forceinline__ void at(const XattnArgs& a, int bk, int hk, int row) {
        r = row;
        const RowAt w = row_at(a, bk, hk, min(row, a.M - 1));
        q = off_at(w, a.q_sb, a.q_sl, a.q_sh);
        d = off_at(w, a.d_sb, a.d_sl, a.d_sh);
        lse = (w.b * a.Hq + w.hq) * a.Lq + w.i;
        i = w.i;
    }
    __device__ __forceinline__ void step(const XattnArgs& a, int bk, int hk) {
        if (!a.walk) { at(a, bk, hk, r + RT); return; }
        const int n = RT / a.G;
        r += RT;
        i += n;
        q += n * a.q_sl;
        d += n * a.d_sl;
        lse += n;
        if (i >= a.Lq) {
            i -= a.Lq;
            q += a.q_sb - a.Lq * a.q_sl;
            d += a.d_sb - a.Lq * a.d_sl;
            lse += (a.Hq - 1) * a.Lq;
        }
    }
};

// The power of two on dS (see above). A lane and its other half hold one column of dS -- a row of dQ, a state of dK -- and of what it is added
// to, so each column has a factor of its own: an infinity or a large row leaves its neighbours alone. Returns with ds scaled.
template <bool F16, int NA>
__device__ __forceinline__ void scale_ds(f32x16& ds, f32x16 (&acc)[NA], float& sc) {
    if constexpr (F16) {
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(ds[i]));
        if (__any(mx * sc > 32768.0f || (sc == 0.f && mx > 0.f))) {
            mx = max_halves(mx);
            if (mx * sc > 32768.0f || (sc == 0.f && mx > 0.f)) {
                const int e = min(max(11 - (int)__builtin_amdgcn_frexp_expf(mx), -100), 100);      // mx = f 2^x, f in [1/2, 1): mx 2^e in [2^10, 2^11)
                const float ns = __builtin_ldexpf(1.0f, e);
                const float f = sc == 0.f ? 1.0f : ns / sc;
#pragma unroll
                for (int d = 0; d < NA; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[d][i] *= f;
                sc = ns;
            }
        }
        const float by = sc == 0.f ? 1.0f : sc;
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] *= by;
    }
}
// dK, dV: S = Q K^T with the rows in the accumulator's rows and a state per lane; P and dS are then operands over the rows. 2 x 16 heads, 4096 rows
// and states: 743 us 128 wide (740 TFLOP/s: dK, dV, K and V of a wave's 32 states need more than 256 registers, so a SIMD has one wave, and
// its products wait for LDS), 334 us 64 wide (823, two waves).
constexpr int DKV_ROWS = 64;                                        // rows per barrier
template <bool F16, int DT>
__global__ __launch_bounds__(256, DT == 64 ? 2 : 1) void xattn_dkv_kernel(XattnArgs a) {
    const int item = xcd_item(blockIdx.x, a.n_items);
    if (item >= a.n_items) return;
    const int kt = item % a.tiles, split = item / a.tiles % a.splits, grp = item / a.tiles / a.splits, bk = grp / a.Hk, hk = grp % a.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5, tid = threadIdx.x;
    const int key = kt * 128 + wave * 32 + (lane & 31);
    const int len = states_of(a, bk);
    const bool ok = mask_byte(a, bk, key, len) != 0;
    constexpr int RT = DKV_ROWS, TB = RT * DT * 2, STAGE = 2 * TB + RT * 8, CH = DT / 8;    // RT rows of Q, of dout, their lse, their delta
    constexpr int PC = RT * CH / 256;                                         // 16-byte chunks per thread and tensor
    const int r0 = split * a.chunk, r1 = min(a.M, r0 + a.chunk);
    int nt = __syncthreads_or(ok) ? (r1 - r0 + RT - 1) / RT : 0;

    uint4 kf[DT / 16], vf[DT / 16];
    {
        const int kc = min(key, a.Lk - 1);
        const uint16_t* k = a.k + bk * a.k_sb + hk * a.k_sh + (int64_t)kc * a.k_sl;
        const uint16_t* v = a.v + bk * a.v_sb + hk * a.v_sh + (int64_t)kc * a.v_sl;
#pragma unroll
        for (int ks = 0; ks < DT / 16; ++ks) { kf[ks] = row_frag(k, ks, h, a.D, ok); vf[ks] = row_frag(v, ks, h, a.D, ok); }
    }
    f32x16 dk[DT / 32], dv[DT / 32];
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) { dk[d][i] = 0.f; dv[d][i] = 0.f; }
    float sc = F16 ? 0.f : 1.0f;

    // A tile's rows arrive by LDS-DMA, a 16-byte chunk per lane at a time, from wherever the row lies; absent rows and chunks past D come from a
    // few zeros. (Through registers the 256 + 256 of a wave do not reach: the loads were waited for at once, to be put away.)
    float gs = 0.f;
    RowWalk<RT> walk[PC], stat;
#pragma unroll
    for (int j = 0; j < PC; ++j) walk[j].at(a, bk, hk, r0 + (tid + 256 * j) / CH);
    if (tid < 2 * RT) stat.at(a, bk, hk, r0 + tid % RT);
    const uint32_t lds0 = lds_addr_of(conv_lds_dyn);
    auto fetch = [&](int buf) {                                                // the next tile's share of this thread
#pragma unroll
        for (int j = 0; j < PC; ++j) {
            const int p = tid + 256 * j, c = 8 * ((p % CH) ^ tile_xor<DT>(p / CH));
            const bool in = walk[j].r < r1 && c < a.D;
            const uint32_t to = lds0 + buf * STAGE + (wave * 64 + 256 * j) * 16;
            dma16_lane(in ? a.q + walk[j].q + c : a.zeros, to);
            dma16_lane(in ? a.dout + walk[j].d + c : a.zeros, to + TB);
            walk[j].step(a, bk, hk);
        }
        if (tid < 2 * RT) {                                                    // -lse (base 2), delta; absent rows: P = exp2(-inf) = 0
            if (stat.r >= r1) gs = tid < RT ? NEG_INF : 0.f;
            else if (tid < RT) gs = P_UP<F16> - a.lse[stat.lse] * LOG2E;
            else gs = a.delta[(int64_t)grp * a.M + stat.r];
            stat.step(a, bk, hk);
        }
    };
    auto put = [&](int buf) {
        if (tid < 2 * RT) reinterpret_cast<float*>(conv_lds_dyn + buf * STAGE + 2 * TB)[tid] = gs;
    };
    if (nt > 0) { fetch(0); put(0); }
    wait_all_and_meet();
    if (a.M <= RT && nt > 0) {                                                 // few rows: one tile, P and dS with their rests (rest8)
        bool rests = true;
#pragma unroll 1
        for (int rb = 0; rb < 2; ++rb) {
            const float* st = reinterpret_cast<const float*>(conv_lds_dyn + 2 * TB) + 32 * rb;
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) { s[i] = 0.f; dp[i] = 0.f; }
#pragma unroll
            for (int ks = 0; ks < DT / 16; ++ks) {
                s = T16<F16>::mfma32(frag_rows<DT>(conv_lds_dyn, 32 * rb, ks, lane), kf[ks], s);
                dp = T16<F16>::mfma32(frag_rows<DT>(conv_lds_dyn + TB, 32 * rb, ks, lane), vf[ks], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int row = 8 * (i / 4) + 4 * h + i % 4;
                s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.c, st[row]));
                dp[i] = s[i] * (dp[i] - st[RT + row]);
            }
            scale_ds<F16, DT / 32>(dp, dk, sc);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint4 w = pack8<F16>(s, u), x = pack8<F16>(dp, u), wr = rest8<F16>(s, u, w), xr = rest8<F16>(dp, u, x);
#pragma unroll
                for (int d = 0; d < DT / 32; ++d) {
                    const uint4 o = frag_cols<DT, 4, 8>(conv_lds_dyn + TB, 32 * rb + 16 * u, 32 * d, lane), q = frag_cols<DT, 4, 8>(conv_lds_dyn, 32 * rb + 16 * u, 32 * d, lane);
                    dv[d] = T16<F16>::mfma32(o, w, dv[d]);
                    dk[d] = T16<F16>::mfma32(q, x, dk[d]);
                    if (rests) {
                        dv[d] = T16<F16>::mfma32(o, wr, dv[d]);
                        dk[d] = T16<F16>::mfma32(q, xr, dk[d]);
                    }
                }
            }
            if (rb == 1 && rests && any_nan(dv)) {                             // both blocks again
                clear(dv);
                clear(dk);
                sc = F16 ? 0.f : 1.0f;
                rests = false;
                rb = -1;
            }
        }
        nt = 0;
    }
    for (int t = 0; t < nt; ++t) {
        if (t + 1 < nt) fetch((t + 1) & 1);
        // two blocks of 32 rows, one behind the other: while the matrix cores form the second block's S and dP, the vector ALU makes P and dS of
        // the first; while they add the first block to dV and dK, it makes those of the second
        const unsigned char* qt = conv_lds_dyn + (t & 1) * STAGE;
        const unsigned char* dt = qt + TB;
        const float* st = reinterpret_cast<const float*>(qt + 2 * TB);
        constexpr int N = DT / 8, AHEAD = 4, PER = 16 / N;                     // products of a block's S and dP (and of its share of dV and dK)
        f32x16 s[2], dp[2];
        uint4 f[AHEAD], w[2][2], ds[2][2];
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
            for (int i = 0; i < 16; ++i) { s[rb][i] = 0.f; dp[rb][i] = 0.f; }
        auto rows = [&](int n) {                                               // fragment n of the 2 N of S and dP: Q's rows, dout's rows
            const int rb = n / N, i = n % N;
            return frag_rows<DT>(i < N / 2 ? qt : dt, 32 * rb, i % (N / 2), lane);
        };
        auto cols = [&](int n) {                                               // fragment n of the 2 N of dV and dK: dout's and Q's columns in turn
            const int rb = n / N, i = n % N;
            return frag_cols<DT, 4, 8>(i % 2 == 0 ? dt : qt, 32 * rb + 16 * (i / 2 % 2), 32 * (i / 4), lane);
        };
        auto score = [&](int n) {
            const int rb = n / N, i = n % N;
            if (i < N / 2) s[rb] = T16<F16>::mfma32(f[n % AHEAD], kf[i], s[rb]);
            else dp[rb] = T16<F16>::mfma32(f[n % AHEAD], vf[i - N / 2], dp[rb]);
            f[n % AHEAD] = n + AHEAD < 2 * N ? rows(n + AHEAD) : cols(n + AHEAD - 2 * N);
        };
        auto add = [&](int n) {
            const int rb = n / N, i = n % N, d = i / 4, u = i / 2 % 2;
            if (i % 2 == 0) dv[d] = T16<F16>::mfma32(f[n % AHEAD], w[rb][u], dv[d]);
            else dk[d] = T16<F16>::mfma32(f[n % AHEAD], ds[rb][u], dk[d]);
            if (n + AHEAD < 2 * N) f[n % AHEAD] = cols(n + AHEAD);
        };
        float4 nl, de;
        auto weigh = [&](int rb, int i) {                                      // row i of the block: P = exp2(c S - lse), dS = P (dP - delta)
            if (i % 4 == 0) {
                nl = *reinterpret_cast<const float4*>(st + 32 * rb + 2 * i + 4 * h);
                de = *reinterpret_cast<const float4*>(st + RT + 32 * rb + 2 * i + 4 * h);
            }
            const float n1 = i % 4 == 0 ? nl.x : i % 4 == 1 ? nl.y : i % 4 == 2 ? nl.z : nl.w, d1 = i % 4 == 0 ? de.x : i % 4 == 1 ? de.y : i % 4 == 2 ? de.z : de.w;
            s[rb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rb][i], a.c, n1));
            dp[rb][i] = s[rb][i] * (dp[rb][i] - d1);
        };
        auto round = [&](int rb) {
            scale_ds<F16, DT / 32>(dp[rb], dk, sc);
#pragma unroll
            for (int u = 0; u < 2; ++u) { w[rb][u] = pack8<F16>(s[rb], u); ds[rb][u] = pack8<F16>(dp[rb], u); }
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = rows(i);
#pragma unroll
        for (int i = 0; i < N; ++i) { score(i); reads_stay(); }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            score(N + i);
#pragma unroll
            for (int e = 0; e < PER; ++e) weigh(0, PER * i + e);
            reads_stay();
        }
        round(0);
        // fp16: the first block's dS carries the scale of its round; the second block may lower it only after the first is added
#pragma unroll
        for (int i = 0; i < N; ++i) {
            add(i);
#pragma unroll
            for (int e = 0; e < PER; ++e) weigh(1, PER * i + e);
            reads_stay();
        }
        round(1);
#pragma unroll
        for (int i = 0; i < N; ++i) { add(N + i); reads_stay(); }
        if (t + 1 < nt) put((t + 1) & 1);
        wait_all_and_meet();
    }
    if (key >= a.Lk) return;
    const float fv = saturate_from_here<F16>() * __builtin_amdgcn_exp2f(-P_UP<F16>);
    const float fk = a.scale * fv / (sc == 0.f ? 1.0f : sc);
    const int64_t at = a.splits > 1 ? (((int64_t)split * a.Bk * a.Hk + grp) * a.Lk + key) * DT : (((int64_t)bk * a.Lk + key) * a.Hk + hk) * a.D;
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int e = 32 * d + 8 * q + 4 * h;
            float4 x, y;
            float* xs = &x.x;
            float* ys = &y.x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                xs[i] = ok ? dk[d][4 * q + i] * fk : 0.f;
                ys[i] = ok ? dv[d][4 * q + i] * fv : 0.f;
            }
            if (a.splits > 1) {
                *reinterpret_cast<float4*>(a.part + at + e) = x;
                *reinterpret_cast<float4*>(a.part2 + at + e) = y;
            } else if (e < a.D) {
                *reinterpret_cast<uint2*>(a.dk + at + e) = make_uint2(T16<F16>::pack2(x.x, x.y), T16<F16>::pack2(x.z, x.w));
                *reinterpret_cast<uint2*>(a.dv + at + e) = make_uint2(T16<F16>::pack2(y.x, y.y), T16<F16>::pack2(y.z, y.w));
            }
        }
}

// What a row of dQ (a lane and its other half) holds while it walks the states: Q, dout, P_UP - lse (base 2) and delta = rowsum(dout o out), with out
// as it was rounded. That rounding meets dP = dout v directly and weighs 1 / sqrt(n) of dS's own with n states: up to 32 of them delta is formed
// anew from P and dP.
template <bool F16, int DT>
struct GradRow {
    uint4 q[DT / 16], d[DT / 16];
    float nl, de;
    __device__ __forceinline__ void load(const XattnArgs& a, const RowAt& w, int h, bool in) {
        const uint16_t* qp = a.q + off_at(w, a.q_sb, a.q_sl, a.q_sh);
        const uint16_t* dp = a.dout + off_at(w, a.d_sb, a.d_sl, a.d_sh);
#pragma unroll
        for (int ks = 0; ks < DT / 16; ++ks) { q[ks] = row_frag(qp, ks, h, a.D, in); d[ks] = row_frag(dp, ks, h, a.D, in); }
        nl = in ? P_UP<F16> - a.lse[off_lse(a, w)] * LOG2E : NEG_INF;
        // this lane's half of the row, then the other's
        const uint16_t* o = a.out + off_out(a, w);
        de = 0.f;
#pragma unroll
        for (int ks = 0; ks < DT / 16; ++ks) {
            const uint4 x = row_frag(o, ks, h, a.D, in), y = d[ks];
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) de += T16<F16>::lo(xs[i]) * T16<F16>::lo(ys[i]) + T16<F16>::hi(xs[i]) * T16<F16>::hi(ys[i]);
        }
        de = sum_halves(de);
    }
};
// dQ^T += K^T dS^T of 32 states (tiles in LDS). REST: with the rest of dS (rest8); WHOLE: they are all that the row has, delta = sum P dP
enum { MANY, REST, WHOLE };
template <bool F16, int DT, int FEW = MANY>
__device__ __forceinline__ void add_dq(const unsigned char* ktile, const unsigned char* vtile, GradRow<F16, DT>& g, f32x16 (&acc)[DT / 32],
                                       float& sc, float c, const float* bias, bool all, int lane) {
    const int h = lane >> 5;
    f32x16 s, ds;
    start_scores(s, bias, all, h);
#pragma unroll
    for (int i = 0; i < 16; ++i) ds[i] = 0.f;
    constexpr int N = DT / 8, AHEAD = 4;                           // K's and V's fragments in turn
    auto row = [&](int i) { return frag_rows<DT>(i % 2 == 0 ? ktile : vtile, 0, i / 2, lane); };
    uint4 f[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) f[i] = row(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i % 2 == 0) s = T16<F16>::mfma32(f[i % AHEAD], g.q[i / 2], s);
        else ds = T16<F16>::mfma32(f[i % AHEAD], g.d[i / 2], ds);
        if (i + AHEAD < N) f[i % AHEAD] = row(i + AHEAD);
        reads_stay();
    }
    constexpr int NC = DT / 16;                                    // K's columns for dQ^T += K^T dS^T
    auto column = [&](int i) { return frag_cols<DT, 4, 8>(ktile, 16 * (i % 2), 32 * (i / 2), lane); };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) f[i] = column(i);
    reads_stay();
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, g.nl));
    if constexpr (FEW == WHOLE) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t = __builtin_fmaf(s[i], ds[i], t);
        g.de = sum_halves(t) * __builtin_amdgcn_exp2f(-P_UP<F16>);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) ds[i] = s[i] * (ds[i] - g.de);
    scale_ds<F16, DT / 32>(ds, acc, sc);
    uint4 p[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) p[u] = pack8<F16>(ds, u);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        acc[i / 2] = T16<F16>::mfma32(f[i % AHEAD], p[i % 2], acc[i / 2]);
        if constexpr (FEW != MANY) acc[i / 2] = T16<F16>::mfma32(f[i % AHEAD], rest8<F16>(ds, i % 2, p[i % 2]), acc[i / 2]);
        if (i + AHEAD < NC) f[i % AHEAD] = column(i + AHEAD);
        reads_stay();
    }
}

// dQ: as the forward kernel; dS^T has a row per lane, dQ^T += K^T dS^T reads the K tile a second time, transposed. 2 x 16 heads, 4096 rows and
// states: 386 us 128 wide (1068 TFLOP/s), 259 us 64 wide (797).
// ROWS: REST for up to 32 rows of a group, whose products wait for the states anyway (single rows' dq was up to 1.56 times as far off as with f32
// throughout, and few enough not to average out).
template <bool F16, int DT, int ROWS>
__global__ __launch_bounds__(256, 2) void xattn_dq_kernel(XattnArgs a) {
    const int item = xcd_item(blockIdx.x, a.n_items);
    if (item >= a.n_items) return;
    const int rt = item % a.tiles, split = item / a.tiles % a.splits, grp = item / a.tiles / a.splits, bk = grp / a.Hk, hk = grp % a.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5;
    const int r = rt * 128 + wave * 32 + (lane & 31);
    constexpr int TB = KT * DT * 2, STAGE = 2 * TB + KT * 4;
    const int len = states_of(a, bk), k0 = split * a.chunk, k1 = min(len, k0 + a.chunk);
    int nt = k1 > k0 ? (k1 - k0 + KT - 1) / KT : 0;

    const RowAt w = row_at(a, bk, hk, min(r, a.M - 1));
    GradRow<F16, DT> g;
    g.load(a, w, h, r < a.M);
    if (item == 0 && threadIdx.x < 8) a.zeros[threadIdx.x] = 0;            // (the dK, dV kernel's absent rows)
    if (split == 0 && h == 0 && r < a.M) a.delta[(int64_t)grp * a.M + r] = g.de;
    f32x16 acc[DT / 32];
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    float sc = F16 ? 0.f : 1.0f;

    const uint16_t* kb = a.k + bk * a.k_sb + hk * a.k_sh + (int64_t)k0 * a.k_sl;
    const uint16_t* vb = a.v + bk * a.v_sb + hk * a.v_sh + (int64_t)k0 * a.v_sl;
    const uint32_t lds0 = lds_addr_of(conv_lds_dyn);
    TileLoad<DT, KT, 4> lk, lv;
    lk.init(wave, lane, a.k_sl, a.D);
    lv.init(wave, lane, a.v_sl, a.D);
    uint64_t bits = 0, next = 0;
    uint32_t byte = 0;
    auto request = [&](int t, uint64_t valid, uint32_t at) {
        const bool all = valid == ~0ull;
        lk.request(kb + (int64_t)t * KT * a.k_sl, all, valid, lds0 + at, wave);
        lv.request(vb + (int64_t)t * KT * a.v_sl, all, valid, lds0 + at + TB, wave);
        if (wave == 0) put_bias(reinterpret_cast<float*>(conv_lds_dyn + at + 2 * TB), KT, byte, all, lane);
        byte = mask_byte(a, bk, k0 + (t + 1) * KT + lane, k1);
    };
    if (nt > 0) {
        byte = mask_byte(a, bk, k0 + lane, k1);
        bits = __ballot(byte != 0);
        request(0, bits, 0);
    }
    if (nt == 1 && len <= FEW_STATES) {
        wait_all_and_meet();
        const float* bias = reinterpret_cast<const float*>(conv_lds_dyn + 2 * TB);
        if (len <= 32) {
            if (bits != 0) add_dq<F16, DT, WHOLE>(conv_lds_dyn, conv_lds_dyn + TB, g, acc, sc, a.c, bias, false, lane);
            if (h == 0 && r < a.M) a.delta[(int64_t)grp * a.M + r] = g.de;
        } else {
#pragma unroll 1
            for (int b = 0; b < 2; ++b)
                add_dq<F16, DT, REST>(conv_lds_dyn + 32 * b * DT * 2, conv_lds_dyn + TB + 32 * b * DT * 2, g, acc, sc, a.c, bias + 32 * b, bits == ~0ull, lane);
        }
        nt = 0;
    }
    for (int t = 0; t < nt; ++t) {
        next = __ballot(byte != 0);
        wait_all_and_meet();
        const uint32_t cur = (t & 1) * STAGE, oth = STAGE - cur;
        if (t + 1 < nt) request(t + 1, next, oth);
        const float* bias = reinterpret_cast<const float*>(conv_lds_dyn + cur + 2 * TB);
        const unsigned char* ktile = conv_lds_dyn + cur;
        const unsigned char* vtile = ktile + TB;
        if (bits != 0) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
                add_dq<F16, DT, ROWS>(ktile + 32 * b * DT * 2, vtile + 32 * b * DT * 2, g, acc, sc, a.c, bias + 32 * b, bits == ~0ull, lane);
        }
        bits = next;
    }
    if (r >= a.M) return;
    const float f = saturate_from_here<F16>() * a.scale * __builtin_amdgcn_exp2f(-P_UP<F16>) / (sc == 0.f ? 1.0f : sc);
    const int64_t at = a.splits > 1 ? (((int64_t)split * a.Bk * a.Hk + grp) * a.M + r) * DT : off_out(a, w);
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int e = 32 * d + 8 * q + 4 * h;
            const float4 x = make_float4(acc[d][4 * q] * f, acc[d][4 * q + 1] * f, acc[d][4 * q + 2] * f, acc[d][4 * q + 3] * f);
            if (a.splits > 1) *reinterpret_cast<float4*>(a.part + at + e) = x;
            else if (e < a.D) *reinterpret_cast<uint2*>(a.dq + at + e) = make_uint2(T16<F16>::pack2(x.x, x.y), T16<F16>::pack2(x.z, x.w));
        }
}

// dQ in tiles of 32 rows, as the token kernel: eight waves walk their own blocks of 32 states, their sums meet in LDS and are added in wave order
template <bool F16, int DT, int ROWS>
__global__ __launch_bounds__(TOKEN_WAVES * 64, TOKEN_WAVES / 4) void xattn_dq_few_kernel(XattnArgs a) {
    constexpr int NW = TOKEN_WAVES;
    const int item = xcd_item(blockIdx.x, a.n_items);
    if (item >= a.n_items) return;
    const int rt = item % a.tiles, grp = item / a.tiles, bk = grp / a.Hk, hk = grp % a.Hk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, h = lane >> 5, r = lane & 31, row = rt * 32 + r;
    constexpr int TB = 32 * DT * 2;

    const int len = states_of(a, bk), nt = (len + 31) / 32;
    GradRow<F16, DT> g;
    g.load(a, row_at(a, bk, hk, min(row, a.M - 1)), h, row < a.M);
    if (item == 0 && threadIdx.x < 8) a.zeros[threadIdx.x] = 0;            // (the dK, dV kernel's absent rows)
    if (wave == 0 && h == 0 && row < a.M) a.delta[(int64_t)grp * a.M + row] = g.de;
    f32x16 acc[DT / 32];
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
    float sc = F16 ? 0.f : 1.0f;

    const uint16_t* kb = a.k + bk * a.k_sb + hk * a.k_sh;
    const uint16_t* vb = a.v + bk * a.v_sb + hk * a.v_sh;
    unsigned char* own = conv_lds_dyn + wave * (2 * TB + 128);
    float* bias = reinterpret_cast<float*>(own + 2 * TB);
    const uint32_t lds0 = lds_addr_of(own);
    TileLoad<DT, 32, 1> lk, lv;
    lk.init(0, lane, a.k_sl, a.D);
    lv.init(0, lane, a.v_sl, a.D);
    uint32_t byte = 0, bits = 0;
    auto valid = [&](int t) -> uint32_t { return t < nt ? mask_byte(a, bk, 32 * t + (lane & 31), len) : 0u; };
    auto request = [&](int t) {
        bits = (uint32_t)__ballot(byte != 0);
        const bool all = bits == ~0u;
        lk.request(kb + (int64_t)t * 32 * a.k_sl, all, bits, lds0, 0);
        lv.request(vb + (int64_t)t * 32 * a.v_sl, all, bits, lds0 + TB, 0);
        put_bias(bias, 32, byte, all, lane);
        byte = valid(t + NW);
    };
    byte = valid(wave);
    if (wave < nt) request(wave);
    int t = wave;
    if (len <= FEW_STATES && t < nt) {                                        // (at most one block per wave)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (nt == 1) {
            if (bits != 0) add_dq<F16, DT, WHOLE>(own, own + TB, g, acc, sc, a.c, bias, bits == ~0u, lane);
            if (h == 0 && row < a.M) a.delta[(int64_t)grp * a.M + row] = g.de;
        } else {
            add_dq<F16, DT, REST>(own, own + TB, g, acc, sc, a.c, bias, bits == ~0u, lane);
        }
        t = nt;
    }
    for (; t < nt; t += NW) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        if (bits != 0) add_dq<F16, DT, ROWS>(own, own + TB, g, acc, sc, a.c, bias, bits == ~0u, lane);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                    // the block is read before its place is requested again
        if (t + NW < nt) request(t + NW);
    }
    const float f = saturate_from_here<F16>() * a.scale * __builtin_amdgcn_exp2f(-P_UP<F16>) / (sc == 0.f ? 1.0f : sc);
    wait_all_and_meet();
    float* sums = reinterpret_cast<float*>(conv_lds_dyn);                     // [NW][32][DT + 4]
    constexpr int SW = DT + 4;
    static_assert(NW * 32 * SW * 4 <= NW * (2 * TB + 1024), "the sums fit");
#pragma unroll
    for (int d = 0; d < DT / 32; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4*>(sums + (wave * 32 + r) * SW + 32 * d + 8 * q + 4 * h) =
                make_float4(acc[d][4 * q] * f, acc[d][4 * q + 1] * f, acc[d][4 * q + 2] * f, acc[d][4 * q + 3] * f);
    __syncthreads();
    if (row >= a.M) return;
    const RowAt w = row_at(a, bk, hk, row);
#pragma unroll
    for (int i = 0; i < DT / 8 / NW; ++i) {
        const int c = 8 * (wave + i * NW) + 4 * h;
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < NW; ++u) {
            const float4 x = *reinterpret_cast<const float4*>(sums + (u * 32 + r) * SW + c);
            t.x += x.x; t.y += x.y; t.z += x.z; t.w += x.w;
        }
        if (c < a.D) *reinterpret_cast<uint2*>(a.dq + off_out(a, w) + c) = make_uint2(T16<F16>::pack2(t.x, t.y), T16<F16>::pack2(t.z, t.w));
    }
}

// sums of the splits in their order, 16 lanes per row: the rows of dQ, then the states of dK, then those of dV (whichever were split)
struct SumArgs {
    const float *pq, *pk, *pv;
    int64_t rows, states;                          // rows of dQ, states of dK (and of dV); 0: not split
    int sq, sk;                                    // their splits
};
template <bool F16, int DT>
__global__ __launch_bounds__(256) void xattn_sum_kernel(XattnArgs a, SumArgs p) {
    T16<F16>::enter();
    int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (row >= p.rows + 2 * p.states) return;
    const int l = threadIdx.x & 15;
    const bool query = row < p.rows, value = row >= p.rows + p.states;
    if (!query) row -= value ? p.rows + p.states : p.rows;
    const int n = query ? a.M : a.Lk, splits = query ? p.sq : p.sk, grp = (int)(row / n), i = (int)(row % n);
    const int64_t step = (query ? p.rows : p.states) * DT;
    constexpr int E = DT / 16;
    const float* from = (query ? p.pq : value ? p.pv : p.pk) + row * DT + l * E;
    float o[E] = {};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(from + s * step + e);
            o[e] += v.x; o[e + 1] += v.y; o[e + 2] += v.z; o[e + 3] += v.w;
        }
    }
    const int64_t at = query ? off_out(a, row_at(a, grp / a.Hk, grp % a.Hk, i)) : (((int64_t)(grp / a.Hk) * a.Lk + i) * a.Hk + grp % a.Hk) * a.D;
    uint16_t* to = (query ? a.dq : value ? a.dv : a.dk) + at + l * E;
#pragma unroll
    for (int e = 0; e < E; e += 4)
        if (l * E + e < a.D) *reinterpret_cast<uint2*>(to + e) = make_uint2(T16<F16>::pack2(o[e], o[e + 1]), T16<F16>::pack2(o[e + 2], o[e + 3]));
}

// ------------------------------------------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------------------------------------------
// splits of `len` (in units of `unit`) so that base * splits comes up to, not over, `wanted` workgroups; each at least `least` units long
void choose_splits(int64_t base, int wanted, int len, int unit, int least, int& splits, int& chunk) {
    const int64_t units = cdiv(std::max(len, 1), unit);
    int64_t s = std::min<int64_t>(wanted / base, units / least);
    s = std::min<int64_t>(std::max<int64_t>(s, 1), 64);
    const int64_t per = (units + s - 1) / s;
    splits = (int)((units + per - 1) / per);
    chunk = (int)(per * unit);
}
// One workgroup per CU is where splitting stops to pay (us, forward / dK dV / dQ alone, 1 split .. more; 120 workgroups without a split:
// 46.1, 42.4 (2), 50.8 (5); 30: 37.3, 22.9 (4), 24.3 (8), 31.7 (15); 416: 27.7, 46.1 (2); dK dV with 30: 153 -> 64.3 (8), 75.7 (12); with
// 192: 78.4, 96.5 (2)): the partial results cost more than the idle half of a CU. Single tokens read instead of compute: two workgroups
// per CU, each with at least 1024 states (16 x 8 groups x 16384 x 128: 156, with one per CU 162), and no split at all up to 2048 states.
constexpr int CUS = 256;
int dt_of(const XattnArgs& a) { return a.D <= 64 ? 64 : 128; }
// Tiles of 32 rows, their states shared out over the waves of a workgroup, instead of tiles of 128 rows whose states are shared out over
// workgroups and joined by another launch: for at most 32 rows, and where the 128-row tiles would leave most CUs idle, between 64 states (two
// blocks: the other waves had none; where the CUs take these tiles in two rounds, 192, up to which the 128-row form splits nothing) and 2048. us,
// 128-row tiles and these (tiles of 32 x states x width):
//   120 x 1800 x 128: 23.2, 16.5    240 x 1800 x 128: 27.6, 18.7    480 x 1800 x 128: 36.9, 33.3    768 x 300 x 128: 13.5, 22.8
//   256 x 300 x 64: 11.4, 6.2       512 x 300 x 64: 13.6, 9.1       768 x 300 x 64: 9.2, 11.9       128 x 4000 x 64: 18.2, 19.4
//   128 x 64 x 128: 6.8, 7.2        128 x 65 x 128: 8.1, 7.4        8 x 1800 x 128: 13.8, 15.0      8 x 1800 x 64: 10.7, 10.7
//   256 x 192 x 128: 9.3, 7.9       320 x 100 x 128: 8.3, 12.8      320 x 192 x 128: 9.4, 13.8      320 x 224 x 128: 17.4, 14.0
//   512 x 192 x 128: 9.6, 14.1      512 x 300 x 128: 21.7, 15.4     512 x 1000 x 128: 28.5, 22.4    320 x 192 x 64: 6.8, 7.4
//   320 x 224 x 64: 12.1, 7.5       512 x 600 x 64: 17.0, 10.0      512 x 1800 x 64: 24.6, 16.8     400 x 600 x 128: 22.7, 17.9
bool few_rows(const XattnArgs& a) {
    if (a.M <= 32) return true;
    const int64_t tiles = (int64_t)a.Bk * a.Hk * cdiv(a.M, 32);
    return a.Lk > (tiles > CUS ? 3 * KT : KT) && a.Lk <= 2048 && tiles <= 2 * CUS && (tiles >= 32 || (int64_t)a.Lk * dt_of(a) <= 2048 * 64);
}

// The same for dQ, whose splits share their join with those of dK and dV: from 64 tiles of 32 rows (below, splits spread better) to one per CU
// (a workgroup each). us of the whole backward pass, 128-row tiles and these: 256 x 300 x 64: 22.1, 17.1; 128 x 300 x 128: 31.1, 26.8; 384 x 300
// x 128: 48.7, 50.3; 240 x 1800 x 64: 49.4, 43.4; 32 x 1800 x 64: 25.7, 28.8; 128 x 1000 x 128: 42.7, 37.0; 120 x 1800 x 128: 54.9, 58.3
bool few_dq(const XattnArgs& a) {
    const int64_t tiles = (int64_t)a.Bk * a.Hk * cdiv(a.M, 32);
    return a.Lk > 64 && (int64_t)a.Lk * dt_of(a) <= 2048 * 64 && tiles >= 64 && tiles <= CUS;
}

struct Plan { int tiles, splits, chunk; };
Plan plan_fwd(const XattnArgs& a) {
    Plan p{};
    const int64_t groups = (int64_t)a.Bk * a.Hk;
    if (few_rows(a)) {
        p.tiles = cdiv(a.M, 32);
        choose_splits(groups * p.tiles, a.Lk > 2048 ? 2 * CUS : 1, a.Lk, 256, 4, p.splits, p.chunk);
    } else {
        p.tiles = cdiv(a.M, 128);
        choose_splits(groups * p.tiles, CUS, a.Lk, KT, 2, p.splits, p.chunk);
    }
    return p;
}
Plan plan_dkv(const XattnArgs& a) {
    Plan p{};
    p.tiles = cdiv(a.Lk, 128);
    choose_splits((int64_t)a.Bk * a.Hk * p.tiles, CUS, a.M, 32, 4, p.splits, p.chunk);
    return p;
}
Plan plan_dq(const XattnArgs& a) {
    Plan p{};
    if (few_dq(a)) return {cdiv(a.M, 32), 1, a.Lk};
    p.tiles = cdiv(a.M, 128);
    choose_splits((int64_t)a.Bk * a.Hk * p.tiles, CUS, a.Lk, KT, 2, p.splits, p.chunk);
    return p;
}
unsigned items(XattnArgs& a, const Plan& p) {
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.n_items = a.Bk * a.Hk * p.tiles * p.splits;                // (below 2^23: blocks_api.cpp)
    return 8u * ((a.n_items + 7) / 8);
}
template <auto Kernel>
int launch(const char* name, unsigned grid, unsigned threads, size_t lds, const XattnArgs& a, hipStream_t st) {
    ISB_TRY(allow_lds<Kernel>(lds));
    Kernel<<<grid, threads, lds, st>>>(a);
    ISB_LAUNCHED(name, st);
    return ISB_OK;
}

template <bool F16, int DT>
int fwd(XattnArgs a, float* ws, hipStream_t st) {
    const Plan p = plan_fwd(a);
    const unsigned grid = items(a, p);
    const int64_t rows = (int64_t)a.Bk * a.Hk * a.M;
    a.part = ws;
    a.part2 = ws + (int64_t)p.splits * rows * DT;
    if (few_rows(a)) ISB_TRY((launch<xattn_token_kernel<F16, DT>>("xattn_token", grid, TOKEN_WAVES * 64, TOKEN_WAVES * (2 * 32 * DT * 2 + 1024), a, st)));
    else ISB_TRY((launch<xattn_fwd_kernel<F16, DT>>("xattn_fwd", grid, 256, 2 * (2 * KT * DT * 2 + KT * 4), a, st)));
    if (p.splits > 1) {
        constexpr int per = 1024 / DT;
        xattn_join_kernel<F16, DT><<<(unsigned)((rows + per - 1) / per), 256, 0, st>>>(a);
        ISB_LAUNCHED("xattn_join", st);
    }
    return ISB_OK;
}

template <bool F16, int DT, int ROWS>
int run_dq(const XattnArgs& a, unsigned grid, hipStream_t st) {
    if (few_dq(a)) return launch<xattn_dq_few_kernel<F16, DT, ROWS>>("xattn_dq_few", grid, TOKEN_WAVES * 64, TOKEN_WAVES * (2 * 32 * DT * 2 + 1024), a, st);
    return launch<xattn_dq_kernel<F16, DT, ROWS>>("xattn_dq", grid, 256, 2 * (2 * KT * DT * 2 + KT * 4), a, st);
}
template <bool F16, int DT>
int bwd(XattnArgs a, float* ws, hipStream_t st) {
    const int64_t rows = (int64_t)a.Bk * a.Hk * a.M, states = (int64_t)a.Bk * a.Hk * a.Lk;
    const Plan q = plan_dq(a), k = plan_dkv(a);
    constexpr int RT = DKV_ROWS;
    a.walk = RT % a.G == 0 && (int64_t)a.Lq * a.G >= RT;
    a.zeros = reinterpret_cast<uint16_t*>(ws);
    a.delta = ws + 64;
    float* pq = ws + 64 + (rows + 63) / 64 * 64;
    float* pk = pq + (q.splits > 1 ? q.splits * rows * DT : 0);
    float* pv = pk + (int64_t)k.splits * states * DT;
    unsigned grid = items(a, q);
    a.part = pq;
    ISB_TRY((a.M <= 32 ? run_dq<F16, DT, REST>(a, grid, st) : run_dq<F16, DT, MANY>(a, grid, st)));
    grid = items(a, k);
    a.part = pk;
    a.part2 = pv;
    ISB_TRY((launch<xattn_dkv_kernel<F16, DT>>("xattn_dkv", grid, 256, 2 * DKV_ROWS * (2 * DT * 2 + 8), a, st)));
    const SumArgs p{pq, pk, pv, q.splits > 1 ? rows : 0, k.splits > 1 ? states : 0, q.splits, k.splits};
    const int64_t n = p.rows + 2 * p.states;
    if (n > 0) {
        xattn_sum_kernel<F16, DT><<<(unsigned)((n + 15) / 16), 256, 0, st>>>(a, p);
        ISB_LAUNCHED("xattn_sum", st);
    }
    return ISB_OK;
}
}  // namespace

// bytes of workspace
size_t xattn_workspace(const XattnArgs& a, bool backward) {
    const size_t rows = (size_t)a.Bk * a.Hk * a.M, states = (size_t)a.Bk * a.Hk * a.Lk, dt = dt_of(a);
    if (!backward) {
        const Plan p = plan_fwd(a);
        return p.splits > 1 ? p.splits * rows * (dt + 2) * 4 : 0;
    }
    const Plan k = plan_dkv(a), q = plan_dq(a);
    const size_t pk = k.splits > 1 ? 2 * k.splits * states * dt : 0, pq = q.splits > 1 ? q.splits * rows * dt : 0;
    return (64 + (rows + 63) / 64 * 64 + pk + pq) * 4;
}
int launch_xattn_fwd(XattnArgs a, bool f16, float* ws, hipStream_t st) {
    if (dt_of(a) == 64) return f16 ? fwd<true, 64>(a, ws, st) : fwd<false, 64>(a, ws, st);
    return f16 ? fwd<true, 128>(a, ws, st) : fwd<false, 128>(a, ws, st);
}
int launch_xattn_bwd(XattnArgs a, bool f16, float* ws, hipStream_t st) {
    if (dt_of(a) == 64) return f16 ? bwd<true, 64>(a, ws, st) : bwd<false, 64>(a, ws, st);
    return f16 ? bwd<true, 128>(a, ws, st) : bwd<false, 128>(a, ws, st);
}

}  // namespace isb
