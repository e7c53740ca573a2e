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

// conv4 + SiLU of 8 channels of one token, as bf16 pairs (qt_common.h: conv8_silu_pairs without the table, which pays from hundreds of tokens on)
__device__ __forceinline__ void conv8_silu(const u32x4 (&x)[4], const u32x4 (&taps)[4], uint32_t (&r)[4]) {
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint32_t c0 = taps[e >> 1][2 * (e & 1)], c1 = taps[e >> 1][2 * (e & 1) + 1];
        auto in = [&](int i) { return e & 1 ? hi_bf(x[i][e >> 1]) : lo_bf(x[i][e >> 1]); };
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
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = pack2_bf(silu_bf16(lo_bf(t[i])), silu_bf16(hi_bf(t[i])));
    }
}

// the row before input row i of a sequence's tokens: i >= 0 a token, -1, -2, -3 the stored window's last, middle and first row
__device__ __forceinline__ int row_before(const int* parent_s, int i) { return i >= 0 ? parent_s[i] : max(i - 1, -3); }
__device__ __forceinline__ const bf16_t* input_row(const bf16_t* __restrict__ proj, const bf16_t* __restrict__ window, int i) {
    return i >= 0 ? proj + (size_t)i * PW : window + (size_t)(3 + i) * CD;
}

// One workgroup of eight wavefronts per (sequence, head); MT = 16-token tiles.  Wavefront w takes value columns 16 w .. + 15.
//   S      : lane (column n, group g) loads S[16 w + n][32 kb + 16 eh + 4 g .. + 3]: the B operand of K S^T and Q S^T when a 32-deep block is enumerated in
//            the order (g, eh, i); k and q are stored in LDS in that order.  S = hi + lo in bf16 (off by 2^-17 of an element); k and q are bf16 already
//   K K^T, Q K^T : bf16 MFMA, exact products; L and A in float
//   (I + L) D = R : blocks of 16: the inverses of the diagonal blocks by forward substitution, the rest as products in float (16x16x4): an
//            accumulator tile, register r of lane group g = row 4 g + r, is the B operand of step r for the k indices 4 g + r
template <int MT>
__global__ __launch_bounds__(HEAD_THREADS, 2) void gdn_tree_kernel(const bf16_t* __restrict__ proj, const bf16_t* __restrict__ conv_pool,
                                                                   const bf16_t* __restrict__ cw, const float* __restrict__ A_log,
                                                                   const float* __restrict__ dt_bias, const float* __restrict__ ssm_pool,
                                                                   const int* __restrict__ slots, const int* __restrict__ pos,
                                                                   const int* __restrict__ parents, bf16_t* __restrict__ y, int M, int n_slots) {
    constexpr int R = 16 * MT, LM_LD = R + 4;
    __shared__ __align__(16) bf16_t k_s[R * QK_LD], q_s[R * QK_LD], v_s[R * QK_LD];
    __shared__ __align__(16) float L_s[R * LM_LD], A_s[R * LM_LD], T_s[MT * 16 * 20];
    __shared__ double lc_s[R];
    __shared__ uint64_t anc_s[R];
    __shared__ float beta_s[R], gamma_s[R];
    __shared__ int parent_s[R];
    __shared__ unsigned bad_s[2];

    const int b = blockIdx.x / HV, h = blockIdx.x % HV;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int slot = slots[b];
    bf16_t* const yb = y + (size_t)b * M * KD + h * DV;
    if ((unsigned)slot >= (unsigned)n_slots) {                   // a skipped sequence
        for (int i = tid; i < M * 16; i += HEAD_THREADS) *reinterpret_cast<u32x4*>(yb + (size_t)(i >> 4) * KD + 8 * (i & 15)) = u32x4{0, 0, 0, 0};
        return;
    }
    const bf16_t* const window = conv_pool + (size_t)(slot * 2 + (pos[b] & 1)) * 3 * CD;
    const bf16_t* const rows = proj + (size_t)b * M * PW;
    if (w == 0) {                                                // the tree and the gates, a token per lane
        const int parent = tree_parent(parents + (size_t)b * M, lane, M);
        const bf16_t* gates = rows + (size_t)min(lane, M - 1) * PW + CD + KD + h;
        const float bv = bf2f(gates[0]), av = bf2f(gates[HV]);
        const uint64_t anc = tree_ancestors(parent, lane);
        float lg = log_decay(A_log[h], BF(av + dt_bias[h])), beta = sigmoid_bf16(bv);
        const bool bad = lane < M && !(lg == lg && beta == beta);
        if (bad || lane >= M) lg = 0.f, beta = 0.f;
        const double lc = tree_path_sum(parent, (double)fmaxf(lg, LOG_DECAY_MIN), lane);
        const uint64_t all_bad = __ballot(bad);
        if (lane < R) {
            parent_s[lane] = parent;
            anc_s[lane] = anc;
            lc_s[lane] = lc;
            gamma_s[lane] = expf((float)lc);
            beta_s[lane] = beta;
        }
        if (lane == 0) bad_s[0] = (unsigned)all_bad, bad_s[1] = (unsigned)(all_bad >> 32);
    }
    __syncthreads();

    // conv, SiLU and norms: a row of 128 channels of one token (q, k or v) per 16 lanes
    for (int it = tid >> 4; it < 3 * R; it += HEAD_THREADS / 16) {
        const int part = it / R, j = it % R, ch = part * KD + h * DK + 8 * n;
        bf16_t* const dst = (part == 0 ? q_s : part == 1 ? k_s : v_s) + j * QK_LD;
        uint32_t u[4] = {0, 0, 0, 0};
        if (j < M) {
            u32x4 x[4], taps[4];
            int i = j;
#pragma unroll
            for (int t = 3; t >= 0; t--) {
                x[t] = *reinterpret_cast<const u32x4*>(input_row(rows, window, i) + ch);
                i = row_before(parent_s, i);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) taps[t] = *reinterpret_cast<const u32x4*>(cw + (size_t)ch * 4 + 8 * t);
            conv8_silu(x, taps, u);
        }
        if (part < 2) {
            double sq = 0.0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double lo = (double)lo_bf(u[e]), hi = (double)hi_bf(u[e]);
                sq = fma(hi, hi, fma(lo, lo, sq));
            }
            const float r = rsqrt_rn((float)row16_sum_d(sq) / (float)DK + qk_eps());
            const uint4 s = scale8_packed(make_uint4(u[0], u[1], u[2], u[3]), r, part == 0 ? BF(INV_SCALE * INV_SCALE) : BF(INV_SCALE));
            u[0] = s.x, u[1] = s.y, u[2] = s.z, u[3] = s.w;
        }
        // A value that is not finite would reach every token through a product with zero: the token counts as bad, takes part with zeros, and its own
        // and its descendants' outputs become NaN
        u16x2 most = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; e++) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, u[e] & 0x7fff7fffu));
        const bool bad = max(most.x, most.y) >= V_MOST;
        const uint64_t any = __ballot(bad) >> (16 * g) & 0xffff;
        if (any) {
            u[0] = u[1] = u[2] = u[3] = 0;
            if (n == 0) atomicOr(&bad_s[j >> 5], 1u << (j & 31));
        }
        if (part < 2) {
            const int at = 32 * (n >> 2) + 16 * (n & 1) + 4 * ((n >> 1) & 1);
            *reinterpret_cast<u32x2*>(dst + at) = u32x2{u[0], u[1]};
            *reinterpret_cast<u32x2*>(dst + at + 8) = u32x2{u[2], u[3]};
        } else {
            *reinterpret_cast<u32x4*>(dst + 8 * n) = u32x4{u[0], u[1], u[2], u[3]};
        }
    }
    const int dv = 16 * w + n;
    f4 s[4][2];
    {
        const float* S = ssm_pool + (((size_t)slot * HV + h) * DV + dv) * DK + 4 * g;
#pragma unroll
        for (int kb = 0; kb < 4; kb++)
#pragma unroll
            for (int eh = 0; eh < 2; eh++) s[kb][eh] = __builtin_nontemporal_load(reinterpret_cast<const f4*>(S + 32 * kb + 16 * eh));
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
            const float G = on ? expf((float)(lc_s[i] - lc_s[j])) : 0.f;
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
        u32x4 hi, lo;
#pragma unroll
        for (int eh = 0; eh < 2; eh++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float a = s[kb][eh][2 * i], c = s[kb][eh][2 * i + 1];
                const uint32_t hw = pack2_bf(a, c);
                hi[2 * eh + i] = hw;
                lo[2 * eh + i] = pack2_bf(a - lo_bf(hw), c - hi_bf(hw));
            }
        const bf16x8 bh = __builtin_bit_cast(bf16x8, hi), bl = __builtin_bit_cast(bf16x8, lo);
#pragma unroll
        for (int I = 0; I < MT; I++) {
            const bf16x8 ka = frag(k_s, I, kb), qa = frag(q_s, I, kb);
            ks[I] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, bl, ks[I], 0, 0, 0);
            qs[I] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qa, bl, qs[I], 0, 0, 0);
            ks[I] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, bh, ks[I], 0, 0, 0);
            qs[I] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qa, bh, qs[I], 0, 0, 0);
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

// a sequence whose slot is none or whose M rows do not fit the K / V pools (Lmax = 0: there are none) is skipped
__device__ __forceinline__ bool takes_part(int slot, int p0, int M, int n_slots, int Lmax) {
    return (unsigned)slot < (unsigned)n_slots && (Lmax == 0 || (p0 >= 0 && p0 <= Lmax - M));
}

// The tokens path[0 .. count - 1] of one (layer, sequence, head), through the recurrence of a decode step: the same bits.  The state stays in
// registers from its load to its store.  The conv window of a sequence lies in buffer pos & 1 and goes to buffer (pos + count) & 1, which for an
// even count is the same: all of this head's channels are read before the first is written, and no other workgroup reads them.
__global__ __launch_bounds__(256, 3) void gdn_commit_kernel(const GdnLayers layers, const int* __restrict__ slots, const int* __restrict__ pos,
                                                            const int* __restrict__ path, const int* __restrict__ count, int B, int M, int D,
                                                            int n_slots, int Lmax) {
    __shared__ double red[2];
    __shared__ __align__(16) float k_s[DK];
    __shared__ float v_s[DV], gb_s[2];
    const int h = blockIdx.x % HV, b = blockIdx.x / HV % B, layer = blockIdx.x / HV / B;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, grp = lane >> 4, c = lane & 15;
    const int slot = slots[b], p0 = pos[b], cnt = min(count[b], D);
    if (!takes_part(slot, p0, M, n_slots, Lmax) || cnt <= 0) return;
    const bf16_t* const proj = layers.proj[layer] + (size_t)b * M * PW;
    const bf16_t* const cw = layers.cw[layer];
    const bf16_t* const window = layers.conv[layer] + (size_t)(slot * 2 + (p0 & 1)) * 3 * CD;
    bf16_t* const window_out = layers.conv[layer] + (size_t)(slot * 2 + ((p0 + cnt) & 1)) * 3 * CD;
    const int* const mine = path + (size_t)b * D;
    // threads 0 .. 127 a k channel, 128 .. 255 a v channel; q only moves through the window (threads 0 .. 127)
    const int ch = (tid < 128 ? KD : 2 * KD) + h * DK + (tid & 127), ch_q = h * DK + (tid & 127);
    const uint2 taps = *reinterpret_cast<const uint2*>(cw + (size_t)ch * 4);
    const float gA = layers.A_log[layer][h], gdt = layers.dt_bias[layer][h];
    unsigned x[3], xq[3];
#pragma unroll
    for (int i = 0; i < 3; i++) x[i] = window[i * CD + ch], xq[i] = window[i * CD + ch_q];
    f4 s[8][2];
    f4* const S = reinterpret_cast<f4*>(layers.ssm[layer] + ((size_t)slot * HV + h) * DV * DK);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int row = i * 16 + w * 4 + grp;
        s[i][0] = __builtin_nontemporal_load(S + row * (DK / 4) + c);
        s[i][1] = __builtin_nontemporal_load(S + row * (DK / 4) + 16 + c);
    }
    for (int j = 0; j < cnt; j++) {
        const bf16_t* row = proj + (size_t)path_token(mine, j, M) * PW;
        const unsigned now = row[ch], now_q = row[ch_q];
        const float u = conv_silu(bf2f((bf16_t)x[0]), bf2f((bf16_t)x[1]), bf2f((bf16_t)x[2]), bf2f((bf16_t)now), taps);
        x[0] = x[1], x[1] = x[2], x[2] = now;
        xq[0] = xq[1], xq[1] = xq[2], xq[2] = now_q;
        if (w < 2) {
            const double tot = wave_sum_d((double)u * (double)u);
            if (lane == 0) red[w] = tot;
        } else {
            v_s[tid - 128] = u;
        }
        if (w == 3) {
            const float gv = bf2f(row[CD + KD + (lane == 1 ? HV : 0) + h]);
            const float gate = lane == 1 ? decay_gate(gA, BF(gv + gdt)) : sigmoid_bf16(gv);
            if (lane < 2) gb_s[lane] = gate;                     // beta, g
        }
        __syncthreads();
        if (w < 2) {
            const float r = rsqrt_rn((float)(red[0] + red[1]) / (float)DK + qk_eps());
            k_s[tid] = BF(BF(u * r) * BF(INV_SCALE));
        }
        __syncthreads();
        float k8[8];
        {
            const float4 a = reinterpret_cast<const float4*>(k_s)[c], e = reinterpret_cast<const float4*>(k_s)[16 + c];
            k8[0] = a.x, k8[1] = a.y, k8[2] = a.z, k8[3] = a.w, k8[4] = e.x, k8[5] = e.y, k8[6] = e.z, k8[7] = e.w;
        }
        const float beta = gb_s[0], gg = gb_s[1];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float sv[8] = {s[i][0].x, s[i][0].y, s[i][0].z, s[i][0].w, s[i][1].x, s[i][1].y, s[i][1].z, s[i][1].w};
            gdn_row_step(sv, k8, k8, v_s[i * 16 + w * 4 + grp], gg, beta, 0.f);
            s[i][0] = f4{sv[0], sv[1], sv[2], sv[3]};
            s[i][1] = f4{sv[4], sv[5], sv[6], sv[7]};
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

// K / V rows pos + path[j] -> pos + j of one (pool, sequence, head), eight rows of 512 bytes at a time.  A path goes down a tree, so path[j] >= j grows with
// j: no row is overwritten before it has been read.
__global__ __launch_bounds__(256) void kv_commit_kernel(const KvLayers layers, const int* __restrict__ slots, const int* __restrict__ pos,
                                                        const int* __restrict__ path, const int* __restrict__ count, int B, int M, int D, int n_slots,
                                                        int Lmax) {
    const int head = blockIdx.x % AKV, b = blockIdx.x / AKV % B, pool = blockIdx.x / AKV / B;
    const int slot = slots[b], p0 = pos[b], cnt = min(count[b], D);
    if (!takes_part(slot, p0, M, n_slots, Lmax)) return;
    u32x4* const base = reinterpret_cast<u32x4*>(layers.pool[pool] + (((size_t)slot * AKV + head) * Lmax + p0) * AD);
    for (int j0 = 0; j0 < cnt; j0 += 8) {
        const int j = j0 + (threadIdx.x >> 5), c = threadIdx.x & 31;
        int from = j;
        u32x4 v = {0, 0, 0, 0};
        if (j < cnt) {
            from = path_token(path + (size_t)b * D, j, M);
            if (from != j) v = base[(size_t)from * (AD / 8) + c];
        }
        __syncthreads();
        if (from != j) base[(size_t)j * (AD / 8) + c] = v;
    }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

extern "C" {

int qt_gdn_tree_step(const void* proj, const void* conv_pool, const void* conv_w, const float* A_log, const float* dt_bias, const float* ssm_pool,
                     const int32_t* slots, const int32_t* pos, const int32_t* parents, void* y, int B, int M, int n_slots, hipStream_t stream) {
    if (B < 0 || n_slots < 1 || B > (1 << 26)) return QT_ERR_DIM;
    if (M < 1 || M > TREE_MAX) return QT_ERR_UNSUPPORTED;
    if (B == 0) return QT_OK;
    if (!proj || !conv_pool || !conv_w || !A_log || !dt_bias || !ssm_pool || !slots || !pos || !parents || !y) return QT_ERR_NULL;
    for (const void* p : {proj, conv_pool, conv_w, (const void*)ssm_pool, (const void*)y})
        if (!aligned16(p)) return QT_ERR_ALIGN;
#define QT_TREE(MT)                                                                                                                              \
    hipLaunchKernelGGL((gdn_tree_kernel<MT>), dim3((unsigned)B * HV), dim3(HEAD_THREADS), 0, stream, (const bf16_t*)proj, (const bf16_t*)conv_pool, \
                       (const bf16_t*)conv_w, A_log, dt_bias, ssm_pool, slots, pos, parents, (bf16_t*)y, M, n_slots)
    switch ((M + 15) / 16) {
        case 1: QT_TREE(1); break;
        case 2: QT_TREE(2); break;
        case 3: QT_TREE(3); break;
        default: QT_TREE(4); break;
    }
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
    for (int l0 = 0; l0 < n_gdn; l0 += COMMIT_LAYERS) {
        GdnLayers t = {};
        const int nl = n_gdn - l0 < COMMIT_LAYERS ? n_gdn - l0 : COMMIT_LAYERS;
        for (int i = 0; i < nl; i++) {
            t.proj[i] = (const bf16_t*)proj[l0 + i];
            t.conv[i] = (bf16_t*)conv_pool[l0 + i];
            t.cw[i] = (const bf16_t*)conv_w[l0 + i];
            t.A_log[i] = A_log[l0 + i];
            t.dt_bias[i] = dt_bias[l0 + i];
            t.ssm[i] = ssm_pool[l0 + i];
        }
        hipLaunchKernelGGL(gdn_commit_kernel, dim3((unsigned)nl * B * HV), dim3(256), 0, stream, t, slots, pos, path, count, B, M, D, n_slots,
                           n_kv > 0 ? Lmax : 0);
        QT_CHECK_LAUNCH();
    }
    for (int l0 = 0; l0 < n_kv; l0 += 2 * COMMIT_LAYERS) {
        KvLayers t = {};
        const int nl = n_kv - l0 < 2 * COMMIT_LAYERS ? n_kv - l0 : 2 * COMMIT_LAYERS;
        for (int i = 0; i < nl; i++) t.pool[i] = (bf16_t*)kv_pool[l0 + i];
        hipLaunchKernelGGL(kv_commit_kernel, dim3((unsigned)nl * B * AKV), dim3(256), 0, stream, t, slots, pos, path, count, B, M, D, n_slots, Lmax);
        QT_CHECK_LAUNCH();
    }
    return QT_OK;
}

}  // extern "C"
