// Attention of a tree of drafted tokens over a sequence's cache, 8 query heads on 2 KV heads, head dim 256, for gfx950.
//
// Row r = b * M + j is token j of sequence b.  It attends the pool keys below pos[b] and, among the M new keys of its sequence, those of its ancestors
// and its own; new key j goes into the pool at pos[b] + j.  Up to 64 tokens share one pass over the cache (the chain form, gqa_decode.hip, takes four).
//
// Split over one flat space of 32-key tiles, as there: a segment (sequence, KV head) owns ceil(pos / 32) tiles of the pool and ceil(M / 32) of new keys, the
// segments lie end to end, every workgroup takes the same number of consecutive tiles and writes an unnormalised partial result per segment that
// it touches; a second kernel joins them.
//   tiles  : HBM -> LDS directly, 4 buffers of K and V (16 KiB each), three tiles in flight.  A row is 32 pieces of 16 bytes; piece c of row r lies at place c ^ (r & 15),
//            which spreads the 16 rows of a fragment over the banks
//   scores : S^T[32 keys x 16 rows] = K . Q^T (16x16x32 bf16 MFMA); a row tile is four tokens x the four heads of the KV head; Q^T stays in registers
//   P . V  : O^T[256 x 16 rows] += V^T . P^T, V^T through the transposing LDS load
// Eight wavefronts: each takes row tiles of its own; where there are fewer than eight, CG of them share a row tile's scores and take 256 / CG columns of O
// each.  (Key halves instead would need half the score products, but a partial result each.)
// A visit to a segment is prepared while the one before is finished: its first tiles are asked for ahead of the stores of the partial result.
//
// Measured, us, this launch and the join at the least (profiled): 1 sequence x 7 tokens on 300 keys 8.1 and 3.4 (launches, then slots, segment, rows and tiles one after the other); the layer
// of 16 x 16 on 1024 - 8192 keys 45.7 and 6.7 (160 MB read: 3.5 TB/s over the launch; the tiles by themselves, without arithmetic, stream at more than 6); 8 x 64 on 8192 - 32768 keys 131
// and 13.3 (350 MB; a tile takes the matrix units 3070 clocks and the LDS 2050, since each of the eight wavefronts reads all of it; matrix units busy 51 % of the time, beside them 180
// vector instructions a tile and wavefront; 72 MB of partial results written and read).
#include "tree.h"

using namespace qt;

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int GQA = AH / AKV, QKV_W = AH * 2 * AD + 2 * AKV * AD;
constexpr int KT = 32, ROW_BYTES = AD * 2, TILE_BYTES = KT * ROW_BYTES;        // keys a tile; bytes of its K (or V)
constexpr int BUFS = 4, AHEAD = BUFS - 1, WAVES = 8, THREADS = 64 * WAVES;
constexpr float SCALE_LOG2E = 0.0625f * 1.44269504088896f;                     // 256^-0.5 log2(e): the softmax works with powers of two
constexpr float NEG = -3.0e38f;
constexpr int LAYER_TOKENS = 16, ROPE_BYTES = 32 * 8;                          // tokens of the layer form; (cos, sin) pairs of a position
constexpr int MAX_SEG = 2048, MAX_GRID = 1024;

// the larger of two floats in one instruction (the compiler makes three of fmaxf behind a lane exchange, to quiet signalling NaN)
__device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
    unsigned r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}
__device__ __forceinline__ float max_over_groups(float x) {      // over the lanes n, n + 16, n + 32, n + 48
    const unsigned xi = __float_as_uint(x);
    const auto a = __builtin_amdgcn_permlane32_swap(xi, xi, false, false);
    const unsigned mi = larger(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(mi, mi, false, false);
    return __uint_as_float(larger(b[0], b[1]));
}
__device__ __forceinline__ float sum_over_groups(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float s = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(s), __float_as_uint(s), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

struct Plan {                           // how a launch cuts the flat tile space
    int B, M, Lmax, n_slots, visit, min_tiles;
};
// tiles of a segment in the flat space: the pool's, the new keys', and `visit` empty positions for what a workgroup pays for a segment besides its tiles
__device__ __forceinline__ int segment_tiles(const Plan& p, int slot, int p0) {
    const bool ok = (unsigned)slot < (unsigned)p.n_slots && p0 >= 0 && p0 <= p.Lmax - p.M;
    return ok ? (p0 + KT - 1) / KT + (p.M + KT - 1) / KT + p.visit : 0;
}
__device__ __forceinline__ int tiles_per_wg(int total, int nwg, int min_tiles) { return max(min_tiles, (total + nwg - 1) / nwg); }

// a copy the compiler cannot see through: what is derived from it is computed again where it is used (with two row tiles a wavefront the lane-dependent
// addresses of the tile loop would live in registers that it does not have)
__device__ __forceinline__ int opaque(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
template <int N>
__device__ __forceinline__ void wait_vmem() {                    // the direct-to-LDS loads are not the compiler's to count
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// inclusive prefix sum over the wavefront's lanes: four shifts within each 16-lane row, then the rows' totals as scalars
__device__ __forceinline__ int wave_prefix_sum(int v, int lane) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);           // row_shr:1, 2, 4, 8 (zeros shifted in)
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31), r2 = __builtin_amdgcn_readlane(v, 47);
    return v + (lane < 16 ? 0 : lane < 32 ? r0 : lane < 48 ? r0 + r1 : r0 + r1 + r2);
}
// A direct-to-LDS load of 16 bytes per lane from a scalar address and a lane's 32-bit offset; the 64 pieces land at lds + 16 l.  Inline assembly: waited for by hand.
// Nontemporal: a tile is read once, and plain loads of it stream at 3.3 TB/s, these at more than 6 (16 sequences of 1024 - 8192 keys, no arithmetic).
__device__ __forceinline__ void lds_dma16_at(const void* base, unsigned off, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(base), "s"(lds)
                 : "memory");
}

// the same with four bytes a lane
__device__ __forceinline__ void lds_dma4_at(const void* base, unsigned off, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(off), "s"(base), "s"(lds)
                 : "memory");
}
// What qkv_prep does with a q or k row (attn_glue.hip), in place on row r of a tile by 16 lanes: RMS norm with the sum of squares in double, weights, and the rotation of features
// 0 .. 63 by the pairs of the row's position.  Lane c has pieces c and 16 + c, and returns them in x.
__device__ __forceinline__ void norm_row(unsigned char* tile, int r, int c, const unsigned char* weights, const unsigned char* pairs, float eps, u32x4 (&x)[2]) {
    u32x4* const row = reinterpret_cast<u32x4*>(tile + r * ROW_BYTES);
    x[0] = row[c ^ (r & 15)], x[1] = row[(16 + c) ^ (r & 15)];
    double ss = 0.0;
#pragma unroll
    for (int hf = 0; hf < 2; hf++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const double lo = (double)lo_bf(x[hf][j]), hi = (double)hi_bf(x[hf][j]);
            ss = fma(hi, hi, fma(lo, lo, ss));
        }
    const float inv = rsqrt_rn((float)row16_sum_d(ss) / (float)AD + eps);
#pragma unroll
    for (int hf = 0; hf < 2; hf++) {
        const u32x4 wt = *reinterpret_cast<const u32x4*>(weights + 256 * hf + 16 * c);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t t = pack2_bf(lo_bf(x[hf][j]) * inv, hi_bf(x[hf][j]) * inv);
            x[hf][j] = pack2_bf(lo_bf(wt[j]) * lo_bf(t), hi_bf(wt[j]) * hi_bf(t));
        }
    }
    u32x4 o;                                                     // the partners' features: lane c ^ 4 = the half row mirrored, then every quad reversed
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int m = __builtin_amdgcn_update_dpp(0, (int)x[0][j], 0x141, 0xF, 0xF, true);
        o[j] = (unsigned)__builtin_amdgcn_update_dpp(0, m, 0x1B, 0xF, 0xF, true);
    }
    if (c < 8) {
#pragma clang fp contract(off)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const f32x4 cs = *reinterpret_cast<const f32x4*>(pairs + 64 * (c & 3) + 16 * j);
            const float a0 = lo_bf(x[0][j]) * cs[0], b0 = lo_bf(o[j]) * cs[1], a1 = hi_bf(x[0][j]) * cs[2], b1 = hi_bf(o[j]) * cs[3];
            x[0][j] = c < 4 ? pack2_bf(a0 - b0, a1 - b1) : pack2_bf(b0 + a0, b1 + a1);
        }
    }
    row[c ^ (r & 15)] = x[0], row[(16 + c) ^ (r & 15)] = x[1];
}

// RT row tiles a wavefront, NRG = 8 / CG groups of wavefronts with rows of their own.  LAYER: q, k_new and v_new point into qkv rows; norms and rotation of the query
// rows in the buffer that they come through, those of the new keys in their tile.  Every workgroup of a segment does the former again, which costs less than a launch ahead
// of this one (layer of 1 x 7 tokens on 300 keys 16.8 -> 14.0 us, 16 x 8 on 2000 31.2 -> 29.4, 16 x 16 38.8 -> 37.7).
template <int RT, int CG, bool LAYER>
__global__ __launch_bounds__(THREADS, 2) void attn_tree_kernel(const bf16_t* __restrict__ q, const bf16_t* __restrict__ k_new,
                                                               const bf16_t* __restrict__ v_new, bf16_t* Kp, bf16_t* Vp,
                                                               const int* __restrict__ slots, const int* __restrict__ pos,
                                                               const int* __restrict__ parents, float* __restrict__ part_o,
                                                               float* __restrict__ part_ml, int* __restrict__ seg_tab, const Plan plan,
                                                               const bf16_t* __restrict__ q_norm, const bf16_t* __restrict__ k_norm,
                                                               const float2* __restrict__ rope, float eps) {
    constexpr int Q_W = LAYER ? QKV_W : AH * AD, Q_HEAD = LAYER ? 2 * AD : AD, NEW_W = LAYER ? QKV_W : AKV * AD;      // row and head strides
    constexpr int NRG = WAVES / CG, ROWS = 16 * RT * NRG, CB = 16 / CG;      // rows; column blocks a wavefront takes
    // P takes part as two bf16 terms (off by 2^-16 of a weight).  One term would be off by 2^-8 of each, so an output by 2^-8 sum w |V - o|, which has no bound in terms of the
    // output: of nearly equal weights on opposite V rows little is left.  The second product costs the launches that the cache's bytes bound nothing, 8 x 64 on
    // 8192 - 32768 keys 20 us (120 -> 140).
    constexpr int DEPTH = RT == 1 ? 6 : 4;                       // fragments on their way from LDS
    __shared__ __align__(1024) unsigned char tile_s[BUFS * 2 * TILE_BYTES];
    __shared__ int seg_start[MAX_SEG + 1];
    __shared__ uint64_t seen_s[TREE_MAX];                        // bit i of entry j: token j sees new key i
    __shared__ unsigned bad_s[2];
    constexpr int LT = LAYER ? LAYER_TOKENS : 4;
    __shared__ __align__(1024) unsigned char rope_s[LT * ROPE_BYTES], norm_s[2 * ROW_BYTES];       // pairs of positions pos .. pos + M - 1; weights of q and k
    __shared__ __align__(256) int parent_s[64], depth_s[64];
    const int M = plan.M, nseg = plan.B * AKV;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int rg = w / CG, cg = w % CG;

    // Ends of the segments in the flat space.  Up to 64 segments: in every wavefront's lanes, with their slots and positions, without a barrier
    int lane_end = 0, lane_slot = 0, lane_pos = 0, total;
    if (nseg <= 64) {
        if (lane < nseg) lane_slot = slots[lane / AKV], lane_pos = pos[lane / AKV];
        lane_end = wave_prefix_sum(segment_tiles(plan, lane < nseg ? lane_slot : -1, lane_pos), lane);
        total = __builtin_amdgcn_readlane(lane_end, 63);
        if (blockIdx.x == 0 && w == 0) {                         // (the merge kernel reads the table)
            if (lane == 0) seg_tab[0] = 0;
            if (lane < nseg) seg_tab[lane + 1] = lane_end;
        }
    } else {
        __shared__ int wave_total[WAVES];
        int carry = 0;
        if (threadIdx.x == 0) seg_start[0] = 0;
        for (int base = 0; base < nseg; base += THREADS) {
            const int sg = base + threadIdx.x;
            const int v = wave_prefix_sum(sg < nseg ? segment_tiles(plan, slots[sg / AKV], pos[sg / AKV]) : 0, lane);
            if (lane == 63) wave_total[w] = v;
            __syncthreads();
            int before = carry;
            for (int i = 0; i < WAVES; i++) {
                before += i < w ? wave_total[i] : 0;
                carry += wave_total[i];
            }
            if (sg < nseg) seg_start[sg + 1] = before + v;
            __syncthreads();
        }
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i <= nseg; i += THREADS) seg_tab[i] = seg_start[i];
        total = __builtin_amdgcn_readfirstlane(seg_start[nseg]);
    }
    auto end_of = [&](int sg) { return sg < 0 ? 0 : nseg <= 64 ? __builtin_amdgcn_readlane(lane_end, sg) : __builtin_amdgcn_readfirstlane(seg_start[sg + 1]); };
    const int per = tiles_per_wg(total, gridDim.x, plan.min_tiles);
    const int wt0 = blockIdx.x * per, wt1 = min(wt0 + per, total);
    if (wt0 >= wt1) return;
    int sg = 0;                                                  // the segment that holds position wt0
    if (nseg <= 64) {
        sg = __popcll(__ballot(lane < nseg && lane_end <= wt0));
    } else {
        for (int hi = nseg; sg < hi;) {
            const int mid = (sg + hi) >> 1;
            if (end_of(mid) <= wt0) sg = mid + 1; else hi = mid;
        }
    }
    const unsigned lds0 = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)tile_s);

    // A visit: the part of one segment's tiles that lies in this workgroup's range.  All of it is scalar.
    struct Visit {
        int sg, slot, p0, t0, t1;                                // sg < 0: there is none
    };
    auto find_visit = [&](int s) {                               // the first one at or after segment s
        Visit v = {-1, 0, 0, 0, 0};
        for (; s < nseg; s++) {
            const int begin = end_of(s - 1), end = end_of(s);
            if (begin + plan.visit >= wt1) break;
            if (end == begin || end <= wt0) continue;            // (a skipped sequence)
            v.sg = s;
            v.slot = nseg <= 64 ? __builtin_amdgcn_readlane(lane_slot, s) : __builtin_amdgcn_readfirstlane(slots[s / AKV]);
            v.p0 = nseg <= 64 ? __builtin_amdgcn_readlane(lane_pos, s) : __builtin_amdgcn_readfirstlane(pos[s / AKV]);
            v.t0 = max(wt0 - begin - plan.visit, 0), v.t1 = min(wt1, end) - begin - plan.visit;
            break;
        }
        return v;
    };
    auto pool_rows = [&](const Visit& v) { return ((size_t)v.slot * AKV + v.sg % AKV) * plan.Lmax * AD; };
    auto new_rows = [&](const Visit& v) { return (size_t)(v.sg / AKV) * M * NEW_W + v.sg % AKV * AD; };
    // Wavefront w brings the row pairs w and w + 8 of a tile: lane l place l & 31 of row 2 i + (l >> 5)
    constexpr int PAIRS = KT / 2 / WAVES, PER_TILE = 2 * PAIRS;  // and issues so many loads for it
    auto issue = [&](const Visit& v, int t) {
        const unsigned buf = lds0 + (unsigned)(t & (BUFS - 1)) * (2 * TILE_BYTES);
        const int pool_tiles = (v.p0 + KT - 1) / KT;
        const bool is_new = t >= pool_tiles;
        const int key0 = (is_new ? t - pool_tiles : t) * KT, left = (is_new ? M : v.p0) - key0;
        const size_t at = is_new ? new_rows(v) + (size_t)key0 * NEW_W : pool_rows(v) + (size_t)key0 * AD;
        const bf16_t *ks = (is_new ? k_new : Kp) + at, *vs = (is_new ? v_new : Vp) + at;
        const int ln = RT > 1 ? opaque(lane) : lane;
#pragma unroll
        for (int i = 0; i < PAIRS; i++) {
            int r = 2 * (w + WAVES * i) + (ln >> 5);
            const unsigned piece = (ln & 31) ^ (r & 15);
            if (left < KT) r = min(r, left - 1);                 // (a key past the end: the last one instead, its weight is 0)
            const unsigned off = (unsigned)r * (is_new ? NEW_W * 2 : ROW_BYTES) + 16 * piece;
            const unsigned to = buf + (unsigned)(w + WAVES * i) * (2 * ROW_BYTES);
            lds_dma16_at(ks, off, __builtin_amdgcn_readfirstlane(to));
            lds_dma16_at(vs, off, __builtin_amdgcn_readfirstlane(to + TILE_BYTES));
        }
    };

    Visit v = find_visit(sg);
    if (v.sg < 0) return;
    // Q^T: lane (row n, group g) holds q[row n][32 kb + 8 g .. + 8] of each row tile (rows past the last token repeat it; they are not stored).
    // Up to 64 rows come by way of the tile buffer that is not in use yet, ahead of the tiles: the wait for them leaves the tiles in flight (a load into registers is
    // the compiler's to wait for, which knows nothing of the tiles behind it and waits for those too).
    constexpr bool STAGE_Q = ROWS <= 64;
    bf16x8 bq[RT][8];
    uint64_t seen = 0;                                           // (LAYER) of the lane's token
    auto ask_q = [&](const Visit& v) {
        if constexpr (STAGE_Q) {
            const unsigned buf = lds0 + (unsigned)((v.t0 + AHEAD) & (BUFS - 1)) * (2 * TILE_BYTES);
            const bf16_t* const qs = q + (size_t)(v.sg / AKV) * M * Q_W + v.sg % AKV * GQA * Q_HEAD;
            if constexpr (LAYER) {
                static_assert(LAYER_TOKENS == 4 * 4, "four positions a wavefront");
                auto at = [&](const void* x) { return __builtin_amdgcn_readfirstlane((unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)(char*)x)); };
                if (w < 4) lds_dma16_at(rope + (size_t)v.p0 * 32, (unsigned)(min(4 * w + (lane >> 4), M - 1) * ROPE_BYTES + 16 * (lane & 15)), at(rope_s) + 1024 * w);
                if (w == 4) lds_dma4_at(parents + (size_t)(v.sg / AKV) * M, 4 * min(lane, M - 1), at(parent_s));
                if (w == 5) lds_dma16_from(reinterpret_cast<const char*>((lane < 32 ? q_norm : k_norm) + 8 * (lane & 31)), at(norm_s));
            }
#pragma unroll
            for (int i = 0; i < ROWS / 2 / WAVES; i++) {
                const int r = 2 * (w + WAVES * i) + (lane >> 5);
                const unsigned off = (unsigned)(min(r / GQA, M - 1) * Q_W + r % GQA * Q_HEAD) * 2 + 16 * ((lane & 31) ^ (r & 15));
                lds_dma16_at(qs, off, __builtin_amdgcn_readfirstlane(buf + (unsigned)(w + WAVES * i) * (2 * ROW_BYTES)));
            }
        }
    };
    auto load_q = [&] {
        const int ln = opaque(lane), n = ln & 15, g = ln >> 4;
        if constexpr (STAGE_Q) {
            const int later = min(v.t1 - v.t0, AHEAD);           // tiles in flight behind the rows
            if (later == 3) wait_vmem<3 * PER_TILE>();
            else if (later == 2) wait_vmem<2 * PER_TILE>();
            else wait_vmem<PER_TILE>();
            barrier();
            unsigned char* const qt = tile_s + ((v.t0 + AHEAD) & (BUFS - 1)) * (2 * TILE_BYTES);
            if constexpr (LAYER) {                               // every row once: 16 lanes each
                const int p = ln < M ? parent_s[ln] : -1;
                seen = tree_ancestors((unsigned)p < (unsigned)ln ? p : -1, ln);
#pragma unroll
                for (int r0 = 0; r0 < ROWS; r0 += THREADS / 16) {
                    const int r = r0 + 4 * w + g, up = __shfl(__popcll(seen), min(r / GQA, M - 1)) - 1;
                    u32x4 x[2];
                    norm_row(qt, r, n, norm_s, rope_s + up * ROPE_BYTES, eps, x);
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                barrier();
            }
#pragma unroll
            for (int kb = 0; kb < 8; kb++)
                bq[0][kb] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(qt + (rg * 16 + n) * ROW_BYTES + ((((4 * kb + g) ^ n)) << 4)));
        } else {
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const int tok = min((rg * RT + t) * 4 + n / GQA, M - 1);
                const u32x4* qr = reinterpret_cast<const u32x4*>(q + ((size_t)(v.sg / AKV * M + tok) * AH + v.sg % AKV * GQA + n % GQA) * AD);
#pragma unroll
                for (int kb = 0; kb < 8; kb++) bq[t][kb] = __builtin_bit_cast(bf16x8, qr[kb * 4 + g]);
            }
        }
    };
    ask_q(v);
    if (!STAGE_Q) load_q();
    __builtin_amdgcn_sched_barrier(0);
    for (int i = 0; i < AHEAD; i++)
        if (v.t0 + i < v.t1) issue(v, v.t0 + i);
    while (true) {
        if (STAGE_Q) load_q();
        const int pool_tiles = (v.p0 + KT - 1) / KT;
        const bool has_new = v.t1 > pool_tiles;
        if (has_new && w == 0) {
            const int ln = opaque(lane);
            if (ln < 2) bad_s[ln] = 0;
            if constexpr (LAYER) seen_s[ln] = seen, depth_s[ln] = __popcll(seen);
            else seen_s[ln] = tree_ancestors(tree_parent(parents + (size_t)(v.sg / AKV) * M, ln, M), ln);
        }
        // q is waited for here: in the tile loop the compiler would wait for its loads in every turn, and for the tiles in flight with them
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int kb = 0; kb < 8; kb++) asm volatile("" : "+v"(bq[t][kb]));
        f32x4 O[RT][CB];
        float m_run[RT], l_run[RT];                              // reference points (in the units of the raw products), sums
#pragma unroll
        for (int t = 0; t < RT; t++) {
            m_run[t] = NEG, l_run[t] = 0.f;
#pragma unroll
            for (int j = 0; j < CB; j++) O[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        for (int tile = v.t0; tile < v.t1; tile++) {
            const int ahead = v.t1 - 1 - tile;                   // tiles that are in flight behind this one
            if (ahead >= 2) wait_vmem<2 * PER_TILE>();
            else if (ahead == 1) wait_vmem<PER_TILE>();
            else wait_vmem<0>();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            barrier();                                           // everyone's part of the tile has landed, and everyone is done with the buffer filled next
            if (tile + AHEAD < v.t1) issue(v, tile + AHEAD);
            const unsigned char* const kt = tile_s + (tile & (BUFS - 1)) * (2 * TILE_BYTES);
            unsigned char* const vt = tile_s + (tile & (BUFS - 1)) * (2 * TILE_BYTES) + TILE_BYTES;
            const bool is_new = tile >= pool_tiles;
            const int key0 = is_new ? (tile - pool_tiles) * KT : tile * KT, keys = is_new ? M : v.p0;
            if (is_new) {
                if constexpr (LAYER) {                           // the keys take their places in the pool
                    const int key = threadIdx.x >> 4, c = threadIdx.x & 15;
                    if (key < M) {
                        u32x4 x[2];
                        norm_row(tile_s + (tile & (BUFS - 1)) * (2 * TILE_BYTES), key, c, norm_s + ROW_BYTES, rope_s + (depth_s[key] - 1) * ROPE_BYTES, eps, x);
                        u32x4* const to = reinterpret_cast<u32x4*>(Kp + pool_rows(v) + (size_t)(v.p0 + key) * AD);
                        to[c] = x[0], to[16 + c] = x[1];
                    }
                }
                // A new value that is not finite must not reach rows that do not see it (0 times NaN): it becomes 0 here, and rows that do
                // see its token become NaN at the end.  Rows past the last token become 0.
#pragma unroll
                for (int i = 0; i < TILE_BYTES / 16 / THREADS; i++) {
                    const int at = 64 * w + opaque(lane) + THREADS * i, key = key0 + at / 32;
                    u32x4 x = reinterpret_cast<u32x4*>(vt)[at];
                    bool bad = false;
#pragma unroll
                    for (int e = 0; e < 4; e++) bad |= (x[e] & 0x7f80) == 0x7f80 || (x[e] & 0x7f800000) == 0x7f800000;
                    if (key >= M || bad) reinterpret_cast<u32x4*>(vt)[at] = u32x4{0, 0, 0, 0};
                    if (key < M && bad) atomicOr(&bad_s[key >> 5], 1u << (key & 31));
                }
                __syncthreads();
            }
            const int ln = RT > 1 ? opaque(lane) : lane, n = ln & 15, g = ln >> 4;
            // The fragments of K, then of V, come out of LDS DEPTH steps ahead of their products: what is asked for only just before stands in the way of all that follows.
            // A operand: lane (key n, group g) holds k[key][32 kb + 8 g .. + 8].  V by the transposing load: lane (n, g) points at key 4 g + n / 4, columns 4 (n % 4) ..
            // + 3 of the block, and receives keys 4 g .. + 3 of column n.  Two of them are the A operand when the 32 keys are enumerated as 16 (e >> 2) + 4 g +
            // (e & 3), in which order the lane holds its probabilities.
            f32x4 s[RT][KT / 16];
#pragma unroll
            for (int t = 0; t < RT; t++)
#pragma unroll
                for (int u = 0; u < KT / 16; u++) s[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
            const unsigned kat = n * ROW_BYTES + ((g ^ n) << 4);
            auto k_frag = [&](int x) {                           // step x: block kb = x / 2 of keys 16 (x % 2) .. + 15
                return *reinterpret_cast<const u32x4*>(kt + (kat ^ ((x >> 1 & 3) << 6)) + (x >> 3 << 8) + (x & 1) * 16 * ROW_BYTES);
            };
            const int vkey = 4 * g + (n >> 2);
            const unsigned vat = (vkey * ROW_BYTES + ((((n >> 1) & 1) ^ vkey) << 4) + (n & 1) * 8) ^ (CB < 16 ? cg * CB << 5 : 0);
            auto v_block = [](int x) { return CB == 16 ? x >> 1 | (x & 1) << 3 : x; };
            auto v_frag = [&](int x) {
                const int j = v_block(x);
                const unsigned char* const at = vt + (vat ^ ((j & 7) << 5)) + (j >> 3 << 8);
                s16x4 a[2];
#pragma unroll
                for (int u = 0; u < 2; u++) a[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + u * 16 * ROW_BYTES));
                const s16x4 a0 = a[0], a1 = a[1];
                return __builtin_bit_cast(u32x4, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
            };
            u32x4 ring[DEPTH];
#pragma unroll
            for (int x = 0; x < DEPTH; x++) ring[x] = k_frag(x);
#pragma unroll
            for (int x = 0; x < 16; x++) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < RT; t++)
                    s[t][x & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ring[x % DEPTH]), bq[t][x >> 1], s[t][x & 1], 0, 0, 0);
                if (x + DEPTH < 16) ring[x % DEPTH] = k_frag(x + DEPTH);
            }
            __builtin_amdgcn_sched_barrier(0);
            auto start_v = [&] {
#pragma unroll
                for (int x = 0; x < DEPTH && x < CB; x++) ring[x] = v_frag(x);
                __builtin_amdgcn_sched_barrier(0);
            };
            if (RT == 1) start_v();                              // (with two row tiles a wavefront the registers are taken until the softmax is done)
            // online softmax on the raw products: lane (row n, group g) holds keys 16 u + 4 g .. + 3
            const bool masked = is_new || key0 + KT > keys;
            u32x2 ph[RT][KT / 16], pl[RT][KT / 16];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                if (masked) {
                    const uint64_t seen = is_new ? seen_s[((rg * RT + t) * 4 + n / GQA) & 63] : 0;
#pragma unroll
                    for (int u = 0; u < KT / 16; u++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int key = key0 + 16 * u + 4 * g + i;
                            const bool on = is_new ? key < M && (seen >> (key & 63) & 1) : key < keys;
                            s[t][u][i] = on ? s[t][u][i] : -INFINITY;
                        }
                }
                float mx = fmaxf(s[t][0][0], s[t][0][1]);
#pragma unroll
                for (int u = 0; u < KT / 16; u++)
#pragma unroll
                    for (int i = u == 0 ? 2 : 0; i < 4; i += 2) mx = fmaxf(fmaxf(mx, s[t][u][i]), s[t][u][i + 1]);
                mx = max_over_groups(mx);
                // (the reference point moves only when the maximum has grown by more than 2^8: O is rarely rescaled)
                const float m_new = mx > m_run[t] + 8.f / SCALE_LOG2E ? mx : m_run[t], mc = m_new * SCALE_LOG2E;
                const float corr = __builtin_amdgcn_exp2f((m_run[t] - m_new) * SCALE_LOG2E);
                float sum = 0.f;
#pragma unroll
                for (int u = 0; u < KT / 16; u++) {
                    float p[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        p[i] = __builtin_amdgcn_exp2f(fmaf(s[t][u][i], SCALE_LOG2E, -mc));
                        sum += p[i];
                    }
                    const u32x2 h = {pack2_bf(p[0], p[1]), pack2_bf(p[2], p[3])};
                    ph[t][u] = h;
                    pl[t][u] = u32x2{pack2_bf(p[0] - lo_bf(h[0]), p[1] - hi_bf(h[0])), pack2_bf(p[2] - lo_bf(h[1]), p[3] - hi_bf(h[1]))};
                }
                l_run[t] = l_run[t] * corr + sum;                // this lane's share; summed over g at the end
                m_run[t] = m_new;
                if (__any(corr != 1.f)) {
#pragma unroll
                    for (int j = 0; j < CB; j++) O[t][j] *= corr;
                }
            }
            if (RT > 1) start_v();
#pragma unroll
            for (int x = 0; x < CB; x++) {
                const int j = v_block(x);
                const bf16x8 av = __builtin_bit_cast(bf16x8, ring[x % DEPTH]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const u32x4 hp = {ph[t][0][0], ph[t][0][1], ph[t][1][0], ph[t][1][1]};
                    O[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, __builtin_bit_cast(bf16x8, hp), O[t][j], 0, 0, 0);
                    const u32x4 lp = {pl[t][0][0], pl[t][0][1], pl[t][1][0], pl[t][1][1]};
                    O[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, __builtin_bit_cast(bf16x8, lp), O[t][j], 0, 0, 0);
                }
                if (x + DEPTH < CB) ring[x % DEPTH] = v_frag(x + DEPTH);
            }
        }
        const Visit next = find_visit(v.sg + 1);
        __syncthreads();                                         // everyone is done with the tiles, and has said what is not finite
        if (next.sg >= 0) ask_q(next);
        if (next.sg >= 0)
            for (int i = 0; i < AHEAD; i++)
                if (next.t0 + i < next.t1) issue(next, next.t0 + i);
        // the partial result of this visit: [ROWS][256], and per row (reference point in powers of two, sum)
        const uint64_t bad = has_new ? (uint64_t)bad_s[1] << 32 | bad_s[0] : 0;
        const size_t at = (size_t)blockIdx.x + v.sg;
        {
            const int ln = opaque(lane), n = ln & 15, g = ln >> 4;
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const int row = (rg * RT + t) * 16 + n, tok = row / GQA;
                const float l = sum_over_groups(l_run[t]);
                if (tok < M) {
                    float* po = part_o + (at * ROWS + row) * AD + cg * CB * 16 + 4 * g;
#pragma unroll
                    for (int j = 0; j < CB; j++) *reinterpret_cast<f32x4*>(po + 16 * j) = O[t][j];
                    if (g == 0 && cg == 0) {
                        part_ml[(at * ROWS + row) * 2] = m_run[t] * SCALE_LOG2E;
                        part_ml[(at * ROWS + row) * 2 + 1] = bad && (seen_s[tok] & bad) ? __builtin_nanf("") : l;
                    }
                }
            }
        }
        // the new rows of this visit's tiles go into the pool (nobody reads it from pos on)
        if (has_new) {
            const bf16_t *kn = k_new + new_rows(v), *vn = v_new + new_rows(v);
            for (int i = 64 * w + opaque(lane) + max(v.t0 - pool_tiles, 0) * KT * 32, e = min((v.t1 - pool_tiles) * KT, M) * 32; i < e; i += THREADS) {
                const int key = i / 32, c = i % 32;
                const size_t to = (pool_rows(v) + (size_t)(v.p0 + key) * AD) / 8 + c, from = (size_t)key * (NEW_W / 8) + c;
                const u32x4 kx = reinterpret_cast<const u32x4*>(kn)[from], vx = reinterpret_cast<const u32x4*>(vn)[from];
                if (!LAYER) reinterpret_cast<u32x4*>(Kp)[to] = kx;
                reinterpret_cast<u32x4*>(Vp)[to] = vx;
            }
        }
        if (next.sg < 0) break;
        __syncthreads();                                         // (the next visit clears what this one has collected)
        v = next;
        if (!STAGE_Q) load_q();
    }
}

// Joins the partial results: a wavefront per (sequence, token, head), a lane four columns.
// GATE: out [R,2048] = BF(o * sigmoid_bf16(gate)), o rounded to bf16 before, as the separate kernels do
template <bool GATE>
__global__ __launch_bounds__(256) void attn_tree_merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                                                              const int* __restrict__ seg_tab, bf16_t* __restrict__ out, const bf16_t* __restrict__ qkv,
                                                              int nwg, int rows, const Plan plan) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int id = blockIdx.x * 4 + w;
    if (id >= plan.B * plan.M * AH) return;
    const int head = id % AH, r = id / AH, b = r / plan.M, j = r % plan.M;
    const int kvh = head / GQA, sg = b * AKV + kvh, row = j * GQA + head % GQA;
    const int total = seg_tab[plan.B * AKV], ss = seg_tab[sg], se = seg_tab[sg + 1];
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float l = 1.f;
    if (se > ss) {
        const int per = tiles_per_wg(total, nwg, plan.min_tiles);
        const int wg0 = (ss + plan.visit) / per, ns = (se - 1) / per - wg0 + 1;
        const size_t at = (size_t)wg0 + sg;
        const float* ml = part_ml + (at * rows + row) * 2;
        const float* po = part_o + (at * rows + row) * AD + 4 * lane;
        float mm = NEG;
        for (int s = lane; s < ns; s += 64) mm = fmaxf(mm, ml[(size_t)s * rows * 2]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
        float lp = 0.f;
        for (int s0 = 0; s0 < ns; s0 += 64) {
            float f = 0.f;
            if (s0 + lane < ns) {
                const float2 x = *reinterpret_cast<const float2*>(ml + (size_t)(s0 + lane) * rows * 2);
                f = __builtin_amdgcn_exp2f(x.x - mm);
                lp += x.y * f;
            }
            const int here = min(64, ns - s0);
            int s = 0;
            for (; s + 4 <= here; s += 4) {
                f32x4 x[4];
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = *reinterpret_cast<const f32x4*>(po + (size_t)(s0 + s + i) * rows * AD);
#pragma unroll
                for (int i = 0; i < 4; i++) acc += x[i] * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s + i));
            }
            for (; s < here; s++) acc += *reinterpret_cast<const f32x4*>(po + (size_t)(s0 + s) * rows * AD) * __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) lp += __shfl_xor(lp, o);
        l = lp;
    }
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = acc[i] / l;
    if constexpr (GATE) {
        const u32x2 gate = *reinterpret_cast<const u32x2*>(qkv + (size_t)r * QKV_W + head * 2 * AD + AD + 4 * lane);
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = se > ss ? BF(o[i]) * sigmoid_bf16(i & 1 ? hi_bf(gate[i >> 1]) : lo_bf(gate[i >> 1])) : 0.f;
    }
    *reinterpret_cast<u32x2*>(out + (size_t)id * AD + 4 * lane) = u32x2{pack2_bf(o[0], o[1]), pack2_bf(o[2], o[3])};
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline int grid_size() {
    const int cus = qt::cu_count();
    return cus < MAX_GRID ? cus : MAX_GRID;
}
inline int partial_rows(int M) { return M <= 8 ? 32 : M <= 16 ? 64 : M <= 32 ? 128 : 256; }
constexpr long SEG_TAB_BYTES = ((MAX_SEG + 1) * 4 + 15) / 16 * 16;

struct Rows {                           // what the attention needs of a layer whose qkv rows it takes as they are (rope: null if it does not)
    const bf16_t *q_norm = nullptr, *k_norm = nullptr;
    const float2* rope = nullptr;
    float eps = 0.f;
};
int launch(const void* q, const void* k, const void* v, void* Kp, void* Vp, const int32_t* slots, const int32_t* pos, const int32_t* parents, void* out,
           const void* gate_rows, void* workspace, int B, int M, int Lmax, int n_slots, hipStream_t stream, const Rows& raw = {}) {
    const int rows = partial_rows(M), nwg = grid_size();
    const size_t cap = (size_t)nwg + (size_t)B * AKV;
    float* const part_o = (float*)workspace;
    float* const part_ml = part_o + cap * rows * AD;
    int* const seg_tab = reinterpret_cast<int*>(part_ml + cap * rows * 2);
    // visit, us with none / as here / twice as many: 1 x 7 on 300 keys 13.4 / 12.0 / 12.2, layer of 16 x 16 on 1024 - 8192 53.6 / 50.6 / 48.0, 32 x 16 on 50 - 400 27.4 / 24.6 / 23.9,
    // 8 x 64 on 8192 - 32768 157 / 146 / 144, 32 x 64 on 100 - 1000 72.6 / 58.3 / 58.6, 200 x 5 on 20 - 200 36.7 / 33.2 / 33.6, 100 x 64 on 20 - 200 98.7 / 82.2 / 72.5.
    // min_tiles 1 / 2 / 4 / 8: 1 x 7 on 300 keys 11.2 / 12.0 / 12.6 / 17.4, on 4000 21.9 / 17.4 / 16.0 / 18.6, 1 x 64 on 1000 30.8 / 28.3 / 31.6 / 39.5; in batches all the same.
    const Plan plan = {B, M, Lmax, n_slots, 2 + rows / 64, 2};
#define QT_TREE_ATTN(RT, CG, LAYER)                                                                                                                  \
    hipLaunchKernelGGL((attn_tree_kernel<RT, CG, LAYER>), dim3((unsigned)nwg), dim3(THREADS), 0, stream, (const bf16_t*)q, (const bf16_t*)k, (const bf16_t*)v, \
                       (bf16_t*)Kp, (bf16_t*)Vp, slots, pos, parents, part_o, part_ml, seg_tab, plan, raw.q_norm, raw.k_norm, raw.rope, raw.eps)
    if (M <= 8 && raw.rope) QT_TREE_ATTN(1, 4, true);
    else if (M <= 8) QT_TREE_ATTN(1, 4, false);
    else if (M <= 16 && raw.rope) QT_TREE_ATTN(1, 2, true);
    else if (M <= 16) QT_TREE_ATTN(1, 2, false);
    else if (M <= 32) QT_TREE_ATTN(1, 1, false);
    else QT_TREE_ATTN(2, 1, false);
#undef QT_TREE_ATTN
    QT_CHECK_LAUNCH();
    const dim3 grid((unsigned)((B * M * AH + 3) / 4));
    if (gate_rows)
        hipLaunchKernelGGL(attn_tree_merge_kernel<true>, grid, dim3(256), 0, stream, part_o, part_ml, seg_tab, (bf16_t*)out, (const bf16_t*)gate_rows, nwg, rows, plan);
    else
        hipLaunchKernelGGL(attn_tree_merge_kernel<false>, grid, dim3(256), 0, stream, part_o, part_ml, seg_tab, (bf16_t*)out, (const bf16_t*)nullptr, nwg, rows, plan);
    QT_CHECK_LAUNCH();
    return QT_OK;
}

int check(int B, int M, int Lmax, int n_slots) {
    if (B < 0 || Lmax < 1 || n_slots < 1) return QT_ERR_DIM;
    if (M < 1 || M > TREE_MAX || B > MAX_SEG / AKV) return QT_ERR_UNSUPPORTED;
    return QT_OK;
}

}  // namespace

extern "C" {

// (attn_glue.hip) the q / k norm, rotary embedding and split of qkv rows whose positions follow from a tree
int qt_internal_qkv_prep_tree(const void* qkv, const void* q_norm, const void* k_norm, const int32_t* pos, const int32_t* parents, const void* rope_table,
                              int table_positions, void* q, void* k, void* v, long R, int M, float eps, hipStream_t stream) __attribute__((visibility("hidden")));

static long partial_bytes(int B, int M) {
    return ((long)grid_size() + (long)B * AKV) * partial_rows(M) * (AD + 2) * 4 + SEG_TAB_BYTES;
}

long qt_gqa_tree_workspace_bytes(int B, int M) {
    if (B < 0 || B > MAX_SEG / AKV || M < 1 || M > TREE_MAX) return -1;
    return partial_bytes(B, M);
}
long qt_gqa_tree_layer_workspace_bytes(int B, int M) {
    const long n = qt_gqa_tree_workspace_bytes(B, M);
    return n < 0 ? n : n + (long)B * M * (AH + 2 * AKV) * AD * 2;
}

int qt_gqa_tree_attn(const void* q, const void* k_new, const void* v_new, void* Kp, void* Vp, const int32_t* slots, const int32_t* pos,
                     const int32_t* parents, void* out, void* workspace, long workspace_bytes, int B, int M, int Lmax, int n_slots, hipStream_t stream) {
    if (const int rc = check(B, M, Lmax, n_slots)) return rc;
    if (B == 0) return QT_OK;
    if (!q || !k_new || !v_new || !Kp || !Vp || !slots || !pos || !parents || !out || !workspace) return QT_ERR_NULL;
    for (const void* p : {q, k_new, v_new, (const void*)Kp, (const void*)Vp, (const void*)out, (const void*)workspace})
        if (!aligned16(p)) return QT_ERR_ALIGN;
    if (workspace_bytes < qt_gqa_tree_workspace_bytes(B, M)) return QT_ERR_WORKSPACE;
    return launch(q, k_new, v_new, Kp, Vp, slots, pos, parents, out, nullptr, workspace, B, M, Lmax, n_slots, stream);
}

int qt_gqa_tree_layer(const void* qkv, const void* q_norm, const void* k_norm, const void* rope_table, int table_positions, void* Kp, void* Vp,
                      const int32_t* slots, const int32_t* pos, const int32_t* parents, void* out, void* workspace, long workspace_bytes, int B, int M,
                      int Lmax, int n_slots, float eps, hipStream_t stream) {
    if (const int rc = check(B, M, Lmax, n_slots)) return rc;
    if (table_positions < 0 || (table_positions > 0 && !rope_table)) return QT_ERR_DIM;
    if (B == 0) return QT_OK;
    if (!qkv || !q_norm || !k_norm || !Kp || !Vp || !slots || !pos || !parents || !out || !workspace) return QT_ERR_NULL;
    for (const void* p : {qkv, q_norm, k_norm, rope_table, (const void*)Kp, (const void*)Vp, (const void*)out, (const void*)workspace})
        if (!aligned16(p)) return QT_ERR_ALIGN;
    if (workspace_bytes < qt_gqa_tree_layer_workspace_bytes(B, M)) return QT_ERR_WORKSPACE;
    // Up to 16 tokens (whose query rows fit a tile buffer) and with a table of every position there can be: no launch ahead of the attention
    if (M <= LAYER_TOKENS && table_positions >= Lmax) {
        const bf16_t* const rows = (const bf16_t*)qkv;
        return launch(rows, rows + AH * 2 * AD, rows + (AH * 2 + AKV) * AD, Kp, Vp, slots, pos, parents, out, qkv, workspace, B, M, Lmax, n_slots, stream,
                      {(const bf16_t*)q_norm, (const bf16_t*)k_norm, (const float2*)rope_table, eps});
    }
    bf16_t* const q = reinterpret_cast<bf16_t*>((char*)workspace + partial_bytes(B, M));
    bf16_t* const k = q + (size_t)B * M * AH * AD;
    bf16_t* const v = k + (size_t)B * M * AKV * AD;
    if (const int rc = qt_internal_qkv_prep_tree(qkv, q_norm, k_norm, pos, parents, rope_table, table_positions, q, k, v, (long)B * M, M, eps, stream)) return rc;
    return launch(q, k, v, Kp, Vp, slots, pos, parents, out, qkv, workspace, B, M, Lmax, n_slots, stream);
}

}  // extern "C"
