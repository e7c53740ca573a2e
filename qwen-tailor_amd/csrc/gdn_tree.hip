// The GatedDeltaNet step of a tree of drafted tokens, and the commit of the path that is accepted, for gfx950.
//
// The chain form (gdn_step.hip, gdn_verify_kernel) writes a state snapshot of 1 MiB for every drafted token, so that whichever is accepted last
// can be taken up.  A tree has too many tokens for that.  Here the step only forms the outputs: it reads the state once and writes none; and
// the commit takes the tokens of the accepted path through the ordinary recurrence, in place: 3 MiB a sequence and layer whatever M is.
//
// With S the committed state, p(i) the parent of token i, G_ij the product of the decays g on the way down from j (not counting it) to i, gamma_i
// that of all decays from the root to i:
//     S_i = g_i S_p(i) + d_i k_i^T,   d_i = beta_i (v_i - g_i S_p(i) k_i),   y_i = S_i q_i
//     d_i + sum over strict ancestors j of beta_i G_ij (k_i . k_j) d_j = beta_i (v_i - gamma_i S k_i)            (I + L) D = R
//     y_i = gamma_i S q_i + sum over ancestors and itself of G_ij (q_i . k_j) d_j                                Y = gamma Q S^T + A D
// A parent comes before its children, so I + L is lower triangular whatever the tree looks like: a token that is no ancestor leaves a zero.
#include <algorithm>

#include "tree.h"

using namespace qt;

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int HEAD_THREADS = 512;
constexpr int QK_LD = DK + 8;           // row stride (bf16) of q, k and v in LDS: the 16 rows of a fragment start 4 banks apart
constexpr float LOG_DECAY_MIN = -1e4f;  // exp of it is 0 in float; -inf would turn differences of sums into NaN
constexpr unsigned V_MOST = (127u + 100u) << 7;      // |v| from 2^100 on, infinities and NaN, as bf16 bits

// conv4 + SiLU of 8 channels of one token, as bf16 pairs (qt_common.h: conv8_silu_pairs without the table)
__device__ __forceinline__ void conv8_silu(const u32x4 (&x)[4], const u32x4 (&taps)[4], uint32_t (&r)[4]) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        auto in = [&](int i) { return e & 1 ? hi_bf(x[i][e >> 1]) : lo_bf(x[i][e >> 1]); };
        const uint32_t c0 = taps[e >> 1][2 * (e & 1)], c1 = taps[e >> 1][2 * (e & 1) + 1];
        s[e] = in(0) * lo_bf(c0);
        s[e] = s[e] + in(1) * hi_bf(c0);
        s[e] = s[e] + in(2) * lo_bf(c1);
        s[e] = s[e] + in(3) * hi_bf(c1);
    }
    u16x2 most = {0, 0};
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        t[i] = pack2_bf(s[2 * i], s[2 * i + 1]);
        most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, t[i] & 0x7fff7fffu));
        const uint32_t sg = sigmoid_bf16_small2(t[i]);
        r[i] = pack2_bf(lo_bf(t[i]) * lo_bf(sg), hi_bf(t[i]) * hi_bf(sg));
    }
    if (__builtin_expect(max(most.x, most.y) > (__float_as_uint(SIGMOID_FAST_MAX) >> 16), 0)) {
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
            const uint32_t ti = i == 0 ? t[0] : i == 1 ? t[1] : i == 2 ? t[2] : t[3], o = pack2_bf(silu_bf16(lo_bf(ti)), silu_bf16(hi_bf(ti)));
            r[0] = i == 0 ? o : r[0], r[1] = i == 1 ? o : r[1], r[2] = i == 2 ? o : r[2], r[3] = i == 3 ? o : r[3];
        }
    }
}

// One workgroup of eight wavefronts per (sequence, head); MT = 16-token tiles.  Wavefront w takes value columns 16 w .. + 15.
//   rows   : the tokens' q, k and v input rows of this head and the stored window go to LDS directly, each once; a token's conv takes its own row and those of
//            three ancestors from there.  (Read from memory by every token that needs them, a conv waited for its parent's index, then for four rows.)
//   S      : lane (column n, group g) loads S[16 w + n][32 kb + 16 eh + 4 g .. + 3]: the B operand of K S^T and Q S^T when a 32-deep block is enumerated in
//            the order (g, eh, i); k and q are stored in LDS in that order.  S = hi + mid + lo in bf16, exact (two terms leave 2^-17 of an element,
//            which shows where the products with k or q cancel; the third costs 0.2 us, at 64 tokens 0.6); k and q are bf16 already
//   K K^T, Q K^T : bf16 MFMA, exact products; L and A in float
//   (I + L) D = R : blocks of 16: the inverses of the diagonal blocks by forward substitution, the rest as products in float (16x16x4): an
//            accumulator tile, register r of lane group g = row 4 g + r, is the B operand of step r for the k indices 4 g + r
// Measured, us: 1 sequence x 7 tokens 7.0 (a string of dependent phases of 1 - 2 thousand clocks), 16 x 16 9.8, 16 x 64 21.7 (of 40 thousand clocks the conv takes 12,
// whose instructions the bf16 rounding points fix, staging 7, products and solve 15).
template <int MT, bool TABLE>
__global__ __launch_bounds__(HEAD_THREADS, 2) void gdn_tree_kernel(const bf16_t* __restrict__ proj, const bf16_t* __restrict__ conv_pool,
                                                                   const bf16_t* __restrict__ cw, const float* __restrict__ A_log,
                                                                   const float* __restrict__ dt_bias, const float* __restrict__ ssm_pool,
                                                                   const int* __restrict__ slots, const int* __restrict__ pos,
                                                                   const int* __restrict__ parents, const bf16_t* __restrict__ silu_table, bf16_t* __restrict__ y, int M,
                                                                   int n_slots) {
    constexpr int R = 16 * MT, LM_LD = R + 4;
    __shared__ __align__(16) bf16_t k_s[R * QK_LD], q_s[R * QK_LD], v_s[R * QK_LD];
    __shared__ __align__(1024) bf16_t raw_s[((R + 3) * 48 + 63) / 64 * 512];
    __shared__ int up_s[R + 3];
    // L and A, and before them the table of SiLU
    constexpr int LA = 2 * R * LM_LD, TAB = TABLE ? SILU_TAB_SIZE / 2 : 0;
    __shared__ __align__(1024) float la_s[LA > TAB ? LA : TAB];
    float *const L_s = la_s, *const A_s = la_s + R * LM_LD;
    bf16_t* const tab = reinterpret_cast<bf16_t*>(la_s);
    __shared__ __align__(1024) bf16_t taps_s[3 * 128 * 4];
    __shared__ __align__(16) float T_s[MT * 16 * 20];
    __shared__ double lc_s[R];
    __shared__ uint64_t anc_s[R];
    __shared__ float beta_s[R], gamma_s[R];
    __shared__ unsigned bad_s[2];

    const int b = blockIdx.x / HV, h = blockIdx.x % HV;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
    bf16_t* const yb = y + (size_t)b * M * KD + h * DV;
    const bf16_t* const rows = proj + (size_t)b * M * PW;
    const auto lds_of = [](void* x) { return (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(char*)x); };
    const unsigned raw_at = lds_of(raw_s);
    // 16-byte chunks of the rows, 48 a row, 64 a load: rows 0 .. M - 1 are the tokens', M .. M + 2 the window's, the last one first
    auto stage = [&](int first, int end, auto row_at) {
        for (int c0 = first + 64 * w; c0 < end; c0 += HEAD_THREADS) {
            const int c = min(c0 + lane, end - 1), r = c / 48, k = c % 48;
            lds_dma16_from(reinterpret_cast<const char*>(row_at(r) + (k >> 4) * KD + h * DK + 8 * (k & 15)), raw_at + 16 * (unsigned)c0);
        }
    };
    const int parent = tree_parent(parents + (size_t)b * M, lane, M);            // every wavefront holds the tree, a token per lane
    const bf16_t* const gates = rows + (size_t)min(lane, M - 1) * PW + CD + KD + h;
    bf16_t b_raw = 0, a_raw = 0;
    if (w == 7) b_raw = gates[0], a_raw = gates[HV];
    const int slot = slots[b], p0 = pos[b];
    if (w < 3) lds_dma16_from(reinterpret_cast<const char*>(cw + (size_t)(w * KD + h * DK) * 4 + 8 * lane), lds_of(taps_s) + 1024 * w);
    if constexpr (TABLE) {
        static_assert(SILU_TAB_SIZE == 12 * 512 + 8, "twelve whole loads, and where inputs outside the table land");
        for (int i = w; i < 12; i += 8) lds_dma16_from(reinterpret_cast<const char*>(silu_table + 512 * i + 8 * lane), lds_of(tab) + 1024 * i);
        if (tid == 0) *reinterpret_cast<u32x4*>(tab + SILU_TAB_HALF) = u32x4{0, 0, 0, 0};
    }
    // (whole loads: the tokens' rows end in the middle of one, which comes with the window)
    const int whole = M * 48 / 64 * 64;
    stage(0, whole, [&](int r) { return rows + (size_t)r * PW; });
    if (tid < 2) bad_s[tid] = 0;
    if (w == 6) {                                                // the row above each row
        if (lane < M) up_s[lane] = parent < 0 ? M : parent;
        if (lane < 3) up_s[M + lane] = M + min(lane + 1, 2);
    }
    if (w < 3)                                                   // rows past the last token: zeros
        for (int i = 16 * M + lane; i < 16 * R; i += 64) {
            bf16_t* const x = w == 0 ? q_s : w == 1 ? k_s : v_s;
            *reinterpret_cast<u32x4*>(x + (i >> 4) * QK_LD + 8 * (i & 15)) = u32x4{0, 0, 0, 0};
        }
    if ((unsigned)slot >= (unsigned)n_slots) {                   // a skipped sequence
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (int i = tid; i < M * 16; i += HEAD_THREADS) *reinterpret_cast<u32x4*>(yb + (size_t)(i >> 4) * KD + 8 * (i & 15)) = u32x4{0, 0, 0, 0};
        return;
    }
    const bf16_t* const window = conv_pool + (size_t)(slot * 2 + (p0 & 1)) * 3 * CD;
    stage(whole, (M + 3) * 48, [&](int r) { return r < M ? rows + (size_t)r * PW : window + (size_t)(M + 2 - r) * CD; });
    __builtin_amdgcn_sched_barrier(0);
    const int dv = 16 * w + n;
    f4 s[4][2];
    {
        const float* S = ssm_pool + (((size_t)slot * HV + h) * DV + dv) * DK + 4 * g;
#pragma unroll
        for (int kb = 0; kb < 4; kb++)
#pragma unroll
            for (int eh = 0; eh < 2; eh++) s[kb][eh] = __builtin_nontemporal_load(reinterpret_cast<const f4*>(S + 32 * kb + 16 * eh));
    }
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");             // the rows have landed; the state is behind them
    __syncthreads();
    // conv, SiLU and norms: items of 128 channels of one token (q, then k, then v), one per 16 lanes, four at a time per wavefront.  The last wavefront has the tree and the
    // gates to do beside them and leaves the first round to the others: items 0 .. 27 go to wavefronts 0 .. 6, then 32 a round to all.
    if (w == 7) {
        float lg = log_decay(A_log[h], BF(bf2f(a_raw) + dt_bias[h])), beta = sigmoid_bf16(bf2f(b_raw));
        const bool bad = lane < M && !(lg == lg && beta == beta);
        if (bad || lane >= M) lg = 0.f, beta = 0.f;
        double lc = (double)fmaxf(lg, LOG_DECAY_MIN);
        const uint64_t anc = tree_ancestors_sum(parent, lc, lane), all_bad = __ballot(bad);
        if (lane < R) {
            anc_s[lane] = anc;
            lc_s[lane] = lc;
            gamma_s[lane] = __expf((float)lc);
            beta_s[lane] = beta;
        }
        if (lane == 0) {
            atomicOr(&bad_s[0], (unsigned)all_bad);
            atomicOr(&bad_s[1], (unsigned)(all_bad >> 32));
        }
    }
    for (int it = w < 7 ? 4 * w + g : 56 + g; __any(it < 3 * M); it = it < 28 ? 28 + 4 * w + g : it + 32) {
        const int part = it < M ? 0 : it < 2 * M ? 1 : 2, j = min(it - part * M, M - 1);
        const bool real = it < 3 * M;                            // (past the end a group repeats the last item and stores nothing)
        u32x4 x[4];
        int r = j;
#pragma unroll
        for (int t = 3; t >= 0; t--) {
            x[t] = *reinterpret_cast<const u32x4*>(raw_s + r * 384 + part * 128 + 8 * n);
            if (t > 0) r = up_s[r];
        }
        u32x4 taps[4];
#pragma unroll
        for (int e = 0; e < 4; e++) taps[e] = *reinterpret_cast<const u32x4*>(taps_s + (part * 128 + 8 * n) * 4 + 8 * e);
        uint32_t u[4];
        if constexpr (TABLE) {
            auto q4 = [](const u32x4& v) { return make_uint4(v[0], v[1], v[2], v[3]); };
            const uint4 wt[4] = {q4(taps[0]), q4(taps[1]), q4(taps[2]), q4(taps[3])};
            conv8_silu_pairs(tab, q4(x[0]), q4(x[1]), q4(x[2]), q4(x[3]), wt, u);
        } else {
            conv8_silu(x, taps, u);
        }
        if (__any(part < 2)) {
            double sq = 0.0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double lo = (double)lo_bf(u[e]), hi = (double)hi_bf(u[e]);
                sq = fma(hi, hi, fma(lo, lo, sq));
            }
            const float rn = rsqrt_rn((float)row16_sum_d(sq) / (float)DK + qk_eps());
            const uint4 q = scale8_packed(make_uint4(u[0], u[1], u[2], u[3]), rn, part == 0 ? BF(INV_SCALE * INV_SCALE) : BF(INV_SCALE));
            if (part < 2) u[0] = q.x, u[1] = q.y, u[2] = q.z, u[3] = q.w;
        }
        // A value that is not finite would reach every token through a product with zero: the token counts as bad, takes part with zeros, and its own
        // and its descendants' outputs become NaN
        u16x2 most = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; e++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, u[e] & 0x7fff7fffu));
        const uint64_t bad = __ballot(max(most.x, most.y) >= V_MOST);
        if (__builtin_expect(bad != 0, 0) && (bad >> (16 * g) & 0xffff)) {
            u[0] = u[1] = u[2] = u[3] = 0;
            if (n == 0) atomicOr(&bad_s[j >> 5], 1u << (j & 31));
        }
        bf16_t* const dst = (part == 0 ? q_s : part == 1 ? k_s : v_s) + j * QK_LD;
        if (real) {
            if (part < 2) {
                const int at = 32 * (n >> 2) + 16 * (n & 1) + 4 * ((n >> 1) & 1);
                *reinterpret_cast<u32x2*>(dst + at) = u32x2{u[0], u[1]};
                *reinterpret_cast<u32x2*>(dst + at + 8) = u32x2{u[2], u[3]};
            } else {
                *reinterpret_cast<u32x4*>(dst + 8 * n) = u32x4{u[0], u[1], u[2], u[3]};
            }
        }
    }
    __syncthreads();

    auto frag = [&](const bf16_t* x, int tile, int kb) { return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(x + (16 * tile + n) * QK_LD + 32 * kb + 8 * g)); };
    // tiles of K K^T (-> -L) and Q K^T (-> A)
    constexpr int TILES = MT * (MT + 1) / 2;
    for (int t = w; t < 2 * TILES; t += 8) {
        const bool is_a = t >= TILES;
        int I = 0, J = t % TILES;
        while (J > I) J -= ++I;
        f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kb = 0; kb < 4; kb++) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(is_a ? q_s : k_s, I, kb), frag(k_s, J, kb), acc, 0, 0, 0);
        const int j = 16 * J + n;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = 16 * I + 4 * g + r;
            const bool on = (anc_s[i] >> j & 1) && (is_a || i != j);
            const float G = on ? __expf((float)(lc_s[i] - lc_s[j])) : 0.f;
            (is_a ? A_s : L_s)[i * LM_LD + j] = on ? acc[r] * (is_a ? G : -beta_s[i] * G) : 0.f;
        }
    }
    __syncthreads();
    if (tid < 16 * MT) {                                         // column n of the inverse of diagonal block g
        const float* Lb = L_s + 16 * g * LM_LD + 16 * g;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float t = i == n ? 1.f : 0.f;
#pragma unroll
            for (int j = 0; j < i; j++) t = fmaf(Lb[i * LM_LD + j], x[j], t);
            x[i] = t;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) T_s[(16 * g + i) * 20 + n] = x[i];
    }
    f4 ks[MT], qs[MT];
#pragma unroll
    for (int I = 0; I < MT; I++) ks[I] = qs[I] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < 4; kb++) {
        u32x4 hi, mid, lo;
#pragma unroll
        for (int eh = 0; eh < 2; eh++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float a = s[kb][eh][2 * i], c = s[kb][eh][2 * i + 1];
                const uint32_t hw = pack2_bf(a, c);
                const float ra = a - lo_bf(hw), rc = c - hi_bf(hw);
                const uint32_t mw = pack2_bf(ra, rc);
                hi[2 * eh + i] = hw, mid[2 * eh + i] = mw;
                lo[2 * eh + i] = pack2_bf(ra - lo_bf(mw), rc - hi_bf(mw));
            }
        const bf16x8 terms[3] = {__builtin_bit_cast(bf16x8, lo), __builtin_bit_cast(bf16x8, mid), __builtin_bit_cast(bf16x8, hi)};
#pragma unroll
        for (int I = 0; I < MT; I++) {
            const bf16x8 ka = frag(k_s, I, kb), qa = frag(q_s, I, kb);
#pragma unroll
            for (int t = 0; t < 3; t++) {
                ks[I] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, terms[t], ks[I], 0, 0, 0);
                qs[I] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qa, terms[t], qs[I], 0, 0, 0);
            }
        }
    }
    __syncthreads();
    f4 d[MT];
    const uint64_t bad = (uint64_t)bad_s[1] << 32 | bad_s[0];
#pragma unroll
    for (int I = 0; I < MT; I++) {
        f4 rhs;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int i = 16 * I + 4 * g + r;
            rhs[r] = beta_s[i] * (bf2f(v_s[i * QK_LD + dv]) - gamma_s[i] * ks[I][r]);
            qs[I][r] *= gamma_s[i];
        }
#pragma unroll
        for (int J = 0; J < I; J++) {
            const f4 a = *reinterpret_cast<const f4*>(L_s + (16 * I + n) * LM_LD + 16 * J + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r++) rhs = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], d[J][r], rhs, 0, 0, 0);
        }
        const f4 t = *reinterpret_cast<const f4*>(T_s + (16 * I + n) * 20 + 4 * g);
        d[I] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 4; r++) d[I] = __builtin_amdgcn_mfma_f32_16x16x4f32(t[r], rhs[r], d[I], 0, 0, 0);
    }
#pragma unroll
    for (int I = 0; I < MT; I++) {
#pragma unroll
        for (int J = 0; J <= I; J++) {
            const f4 a = *reinterpret_cast<const f4*>(A_s + (16 * I + n) * LM_LD + 16 * J + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r++) qs[I] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], d[J][r], qs[I], 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {                            // (column dv of v is this wavefront's own: it is done with it)
            const int i = 16 * I + 4 * g + r;
            v_s[i * QK_LD + dv] = anc_s[i] & bad ? (bf16_t)0x7fc0 : f2bf(qs[I][r]);
        }
    }
    __syncthreads();
    for (int i = tid; i < M * 16; i += HEAD_THREADS)
        *reinterpret_cast<u32x4*>(yb + (size_t)(i >> 4) * KD + 8 * (i & 15)) = *reinterpret_cast<const u32x4*>(v_s + (i >> 4) * QK_LD + 8 * (i & 15));
}

// ---- the commit --------------------------------------------------------------------------------------------------------------
constexpr int COMMIT_LAYERS = 32;       // layers of either kind in one launch (their pointers travel in the kernel arguments)
struct GdnLayers {
    const bf16_t* proj[COMMIT_LAYERS];
    bf16_t* conv[COMMIT_LAYERS];
    const bf16_t* cw[COMMIT_LAYERS];
    const float* A_log[COMMIT_LAYERS];
    const float* dt_bias[COMMIT_LAYERS];
    float* ssm[COMMIT_LAYERS];
};
struct KvLayers {
    bf16_t* pool[2 * COMMIT_LAYERS];    // K and V
};

// index into the M tokens of entry j of a path; one that is none counts as the first token
__device__ __forceinline__ int path_token(const int* __restrict__ path, int j, int M) {
    const int i = path[j];
    return (unsigned)i < (unsigned)M ? i : 0;
}

// a path has no more entries than there are, and no more than the tree has tokens: rows pos .. pos + M - 1 are what a sequence is known to have room for
__device__ __forceinline__ int path_length(int count, int M, int D) { return min(count, min(D, M)); }

// a sequence whose slot is none or whose M rows do not fit the K / V pools (Lmax = 0: there are none) is skipped
__device__ __forceinline__ bool takes_part(int slot, int p0, int M, int n_slots, int Lmax) {
    return (unsigned)slot < (unsigned)n_slots && (Lmax == 0 || (p0 >= 0 && p0 <= Lmax - M));
}

// The tokens path[0 .. count - 1] of one (layer, sequence, head), through the recurrence of a decode step: the same bits.  The state stays in
// registers from its load to its store.  The conv window of a sequence lies in buffer pos & 1 and goes to buffer (pos + count) & 1, which for an
// even count is the same: all of this head's channels are read before the first is written, and no other workgroup reads them.
// Tokens are prepared four at a time (rows asked for a group ahead, conv, norms and gates of the four side by side, two barriers): the first group while the
// state is on its way.  One at a time, a single sequence waited for memory at every token.
constexpr int GROUP = 4;
__device__ __forceinline__ void gdn_commit(const GdnLayers& layers, int block, const int* __restrict__ slots, const int* __restrict__ pos, const int* __restrict__ path,
                                           const int* __restrict__ count, int B, int M, int D, int n_slots, int Lmax) {
    __shared__ double red[GROUP][2];
    __shared__ __align__(16) float k_s[GROUP][DK];
    __shared__ float v_s[GROUP][DV], gb_s[2 * GROUP];
    const int h = block % HV, b = block / HV % B, layer = block / HV / B;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, grp = lane >> 4, c = lane & 15;
    const int token = lane < D ? path_token(path + (size_t)b * D, lane, M) : 0;           // entry j of the path in lane j
    const int slot = slots[b], p0 = pos[b], cnt = path_length(count[b], M, D);
    if (!takes_part(slot, p0, M, n_slots, Lmax) || cnt <= 0) return;
    const bf16_t* const proj = layers.proj[layer] + (size_t)b * M * PW;
    const bf16_t* const window = layers.conv[layer] + (size_t)(slot * 2 + (p0 & 1)) * 3 * CD;
    bf16_t* const window_out = layers.conv[layer] + (size_t)(slot * 2 + ((p0 + cnt) & 1)) * 3 * CD;
    // threads 0 .. 127 a k channel, 128 .. 255 a v channel; q only moves through the window (threads 0 .. 127)
    const int ch = (tid < 128 ? KD : 2 * KD) + h * DK + (tid & 127), ch_q = h * DK + (tid & 127);
    unsigned now[GROUP], now_q[GROUP];
    bf16_t gate_raw = 0;
    auto fetch = [&](int j0) {                                   // (past the path's end: its last token again)
#pragma unroll
        for (int t = 0; t < GROUP; t++) {
            const bf16_t* const row = proj + (size_t)__builtin_amdgcn_readlane(token, min(j0 + t, cnt - 1)) * PW;
            now[t] = row[ch], now_q[t] = row[ch_q];
        }
        if (w == 3) gate_raw = proj[(size_t)__shfl(token, min(j0 + (lane >> 1 & 3), cnt - 1)) * PW + CD + KD + (lane & 1) * HV + h];
    };
    const uint2 taps = *reinterpret_cast<const uint2*>(layers.cw[layer] + (size_t)ch * 4);
    const float gA = layers.A_log[layer][h], gdt = layers.dt_bias[layer][h];
    unsigned x[3], xq[3];
#pragma unroll
    for (int i = 0; i < 3; i++) x[i] = window[i * CD + ch], xq[i] = window[i * CD + ch_q];
    fetch(0);
    __builtin_amdgcn_sched_barrier(0);
    f4 s[8][2];
    f4* const S = reinterpret_cast<f4*>(layers.ssm[layer] + ((size_t)slot * HV + h) * DV * DK);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int row = i * 16 + w * 4 + grp;
        s[i][0] = __builtin_nontemporal_load(S + row * (DK / 4) + c);
        s[i][1] = __builtin_nontemporal_load(S + row * (DK / 4) + 16 + c);
    }
    __builtin_amdgcn_sched_barrier(0);
    for (int j0 = 0; j0 < cnt; j0 += GROUP) {
        float u[GROUP];
#pragma unroll
        for (int t = 0; t < GROUP; t++) {
            u[t] = conv_silu(bf2f((bf16_t)x[0]), bf2f((bf16_t)x[1]), bf2f((bf16_t)x[2]), bf2f((bf16_t)now[t]), taps);
            if (j0 + t < cnt) {
                x[0] = x[1], x[1] = x[2], x[2] = now[t];
                xq[0] = xq[1], xq[1] = xq[2], xq[2] = now_q[t];
            }
        }
        if (w < 2) {
#pragma unroll
            for (int t = 0; t < GROUP; t++) {
                const double tot = wave_sum_d((double)u[t] * (double)u[t]);
                if (lane == 0) red[t][w] = tot;
            }
        } else {
#pragma unroll
            for (int t = 0; t < GROUP; t++) v_s[t][tid - 128] = u[t];
        }
        if (w == 3) {
            const float gv = bf2f(gate_raw), gate = lane & 1 ? decay_gate(gA, BF(gv + gdt)) : sigmoid_bf16(gv);
            if (lane < 2 * GROUP) gb_s[lane] = gate;             // beta, g of each token
        }
        __syncthreads();
        if (w < 2) {
#pragma unroll
            for (int t = 0; t < GROUP; t++) {
                const float r = rsqrt_rn((float)(red[t][0] + red[t][1]) / (float)DK + qk_eps());
                k_s[t][tid] = BF(BF(u[t] * r) * BF(INV_SCALE));
            }
        }
        __syncthreads();
        if (j0 + GROUP < cnt) fetch(j0 + GROUP);
        const int here = min(GROUP, cnt - j0);
#pragma unroll 1
        for (int t = 0; t < here; t++) {
            float k8[8];
            {
                const float4 a = reinterpret_cast<const float4*>(k_s[t])[c], e = reinterpret_cast<const float4*>(k_s[t])[16 + c];
                k8[0] = a.x, k8[1] = a.y, k8[2] = a.z, k8[3] = a.w, k8[4] = e.x, k8[5] = e.y, k8[6] = e.z, k8[7] = e.w;
            }
            const float beta = gb_s[2 * t], gg = gb_s[2 * t + 1];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float sv[8] = {s[i][0].x, s[i][0].y, s[i][0].z, s[i][0].w, s[i][1].x, s[i][1].y, s[i][1].z, s[i][1].w};
                gdn_row_step(sv, k8, k8, v_s[t][i * 16 + w * 4 + grp], gg, beta, 0.f);
                s[i][0] = f4{sv[0], sv[1], sv[2], sv[3]};
                s[i][1] = f4{sv[4], sv[5], sv[6], sv[7]};
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int row = i * 16 + w * 4 + grp;
        __builtin_nontemporal_store(s[i][0], S + row * (DK / 4) + c);
        __builtin_nontemporal_store(s[i][1], S + row * (DK / 4) + 16 + c);
    }
#pragma unroll
    for (int i = 0; i < 3; i++) {                                // (every thread's window has been read: a barrier lies in between)
        window_out[i * CD + ch] = (bf16_t)x[i];
        if (tid < 128) window_out[i * CD + ch_q] = (bf16_t)xq[i];
    }
}

// K / V rows pos + path[j] -> pos + j of one (pool, sequence, head): eight rows of 512 bytes at a time, all read before the first is written
__device__ __forceinline__ void kv_commit(const KvLayers& layers, int block, const int* __restrict__ slots, const int* __restrict__ pos, const int* __restrict__ path,
                                          const int* __restrict__ count, int B, int M, int D, int n_slots, int Lmax) {
    const int head = block % AKV, b = block / AKV % B, pool = block / AKV / B;
    const int lane = threadIdx.x & 63, j0 = threadIdx.x >> 5, c = threadIdx.x & 31;
    const int token = lane < D ? path_token(path + (size_t)b * D, lane, M) : 0;
    const int slot = slots[b], p0 = pos[b], cnt = path_length(count[b], M, D);
    if (!takes_part(slot, p0, M, n_slots, Lmax)) return;
    u32x4* const base = reinterpret_cast<u32x4*>(layers.pool[pool] + (((size_t)slot * AKV + head) * Lmax + p0) * AD) + c;
    u32x4 v[TREE_MAX / 8];
#pragma unroll
    for (int i = 0; i < TREE_MAX / 8; i++) {
        const int from = __shfl(token, 8 * i + j0);
        v[i] = u32x4{0, 0, 0, 0};
        if (8 * i < cnt && 8 * i + j0 < cnt) v[i] = base[(size_t)from * (AD / 8)];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TREE_MAX / 8; i++)
        if (8 * i + j0 < cnt) base[(size_t)(8 * i + j0) * (AD / 8)] = v[i];
}

// Both kinds in one launch (a second one cost a single sequence 2 us); the short ones of the K / V rows last.  18 recurrent layers: 1 sequence 10.5 us, 16 sequences
// 108 (643 MB, the rate of reading and writing in place).
__global__ __launch_bounds__(256, 2) void commit_kernel(const GdnLayers gdn, const KvLayers kv, int n_gdn, const int* __restrict__ slots, const int* __restrict__ pos,
                                                        const int* __restrict__ path, const int* __restrict__ count, int B, int M, int D, int n_slots, int Lmax) {
    const int gdn_blocks = n_gdn * B * HV, block = blockIdx.x;
    if (block < gdn_blocks)
        gdn_commit(gdn, block, slots, pos, path, count, B, M, D, n_slots, Lmax);
    else
        kv_commit(kv, block - gdn_blocks, slots, pos, path, count, B, M, D, n_slots, Lmax);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

extern "C" {

int qt_gdn_tree_step(const void* proj, const void* conv_pool, const void* conv_w, const float* A_log, const float* dt_bias, const float* ssm_pool,
                     const int32_t* slots, const int32_t* pos, const int32_t* parents, const void* silu_table, void* y, int B, int M, int n_slots,
                     hipStream_t stream) {
    if (B < 0 || n_slots < 1 || B > (1 << 26)) return QT_ERR_DIM;
    if (M < 1 || M > TREE_MAX) return QT_ERR_UNSUPPORTED;
    if (B == 0) return QT_OK;
    if (!proj || !conv_pool || !conv_w || !A_log || !dt_bias || !ssm_pool || !slots || !pos || !parents || !y) return QT_ERR_NULL;
    for (const void* p : {proj, conv_pool, conv_w, (const void*)ssm_pool, silu_table, (const void*)y})
        if (!aligned16(p)) return QT_ERR_ALIGN;
    // SiLU from the table from 17 tokens on: below it is evaluated by fewer wavefronts than the table takes to arrive
#define QT_TREE(MT, TABLE)                                                                                                                            \
    hipLaunchKernelGGL((gdn_tree_kernel<MT, TABLE>), dim3((unsigned)B * HV), dim3(HEAD_THREADS), 0, stream, (const bf16_t*)proj,                       \
                       (const bf16_t*)conv_pool, (const bf16_t*)conv_w, A_log, dt_bias, ssm_pool, slots, pos, parents, (const bf16_t*)silu_table, (bf16_t*)y, \
                       M, n_slots)
    if (M <= 16) QT_TREE(1, false);
    else if (M <= 32 && silu_table) QT_TREE(2, true);
    else if (M <= 32) QT_TREE(2, false);
    else if (M <= 48 && silu_table) QT_TREE(3, true);
    else if (M <= 48) QT_TREE(3, false);
    else if (silu_table) QT_TREE(4, true);
    else QT_TREE(4, false);
#undef QT_TREE
    QT_CHECK_LAUNCH();
    return QT_OK;
}

int qt_tree_commit(const void* const* proj, void* const* conv_pool, const void* const* conv_w, const float* const* A_log, const float* const* dt_bias,
                   float* const* ssm_pool, int n_gdn, void* const* kv_pool, int n_kv, const int32_t* slots, const int32_t* pos, const int32_t* path,
                   const int32_t* count, int B, int M, int D, int n_slots, int Lmax, hipStream_t stream) {
    if (n_gdn < 0 || n_kv < 0 || B < 0 || B > (1 << 20) || n_slots < 1) return QT_ERR_DIM;
    if (M < 1 || M > TREE_MAX || D < 1 || D > TREE_MAX) return QT_ERR_UNSUPPORTED;
    if (n_kv > 0 && Lmax < 1) return QT_ERR_DIM;
    if (B == 0) return QT_OK;
    if (!slots || !pos || !path || !count) return QT_ERR_NULL;
    if (n_gdn > 0 && (!proj || !conv_pool || !conv_w || !A_log || !dt_bias || !ssm_pool)) return QT_ERR_NULL;
    if (n_kv > 0 && !kv_pool) return QT_ERR_NULL;
    for (int i = 0; i < n_gdn; i++) {
        for (const void* p : {proj[i], (const void*)conv_pool[i], conv_w[i], (const void*)A_log[i], (const void*)dt_bias[i], (const void*)ssm_pool[i]})
            if (!p) return QT_ERR_NULL;
        if (!aligned16(ssm_pool[i]) || (reinterpret_cast<uintptr_t>(conv_w[i]) & 7u)) return QT_ERR_ALIGN;
    }
    for (int i = 0; i < n_kv; i++) {
        if (!kv_pool[i]) return QT_ERR_NULL;
        if (!aligned16(kv_pool[i])) return QT_ERR_ALIGN;
    }
    for (int g0 = 0, k0 = 0; g0 < n_gdn || k0 < n_kv; g0 += COMMIT_LAYERS, k0 += 2 * COMMIT_LAYERS) {
        GdnLayers gdn = {};
        KvLayers kv = {};
        const int ng = std::max(0, std::min(n_gdn - g0, COMMIT_LAYERS)), nk = std::max(0, std::min(n_kv - k0, 2 * COMMIT_LAYERS));
        for (int i = 0; i < ng; i++) {
            gdn.proj[i] = (const bf16_t*)proj[g0 + i];
            gdn.conv[i] = (bf16_t*)conv_pool[g0 + i];
            gdn.cw[i] = (const bf16_t*)conv_w[g0 + i];
            gdn.A_log[i] = A_log[g0 + i];
            gdn.dt_bias[i] = dt_bias[g0 + i];
            gdn.ssm[i] = ssm_pool[g0 + i];
        }
        for (int i = 0; i < nk; i++) kv.pool[i] = (bf16_t*)kv_pool[k0 + i];
        hipLaunchKernelGGL(commit_kernel, dim3((unsigned)B * (ng * HV + nk * AKV)), dim3(256), 0, stream, gdn, kv, ng, slots, pos, path, count, B, M, D, n_slots,
                           n_kv > 0 ? Lmax : 0);
        QT_CHECK_LAUNCH();
    }
    return QT_OK;
}

}  // extern "C"
