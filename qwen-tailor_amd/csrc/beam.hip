// Beam search on the slot pools, for gfx950: the selection over beams and vocabulary, and the reordering of the beams' states.
//
// Selection: with l_w = log sum_t exp(x[w][t]) the score of candidate (w, t) is scores[w] + x[w][t] - l_w; wanted are the n largest of a sequence's
// W V candidates, equal ones by the lower index w V + t.  The logits are read once: a launch over slices of the vocabulary keeps, per slice,
// its n largest logits and its part (reference point, sum) of l_w; a second launch joins the slices of a sequence's beams.
#include "qt_common.h"
#include <algorithm>
#include <type_traits>

using namespace qt;

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16;

constexpr int SELECT_MAX = 64;          // beams of a sequence, and candidates to select
constexpr int WAVE_CAP = 256;           // candidates a wavefront holds before it keeps the best n of them
constexpr int NO_INDEX = 0x7fffffff;
constexpr float LOG2E = 1.44269504088896f;
// The reference point of the exponentials follows a maximum that is higher by more: a few times a row, and the arguments of the largest terms stay small
constexpr float REFERENCE_LAG = 1.f;

__device__ __forceinline__ float as_float(bf16_t v) { return bf2f(v); }
__device__ __forceinline__ float as_float(f16 v) { return (float)v; }
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ void wave_lds_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// order-preserving bits of a float (a NaN is below everything)
__device__ __forceinline__ unsigned order_bits(float f) {
    const unsigned u = __float_as_uint(f);
    return f != f ? 0u : u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_order_bits(unsigned k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }

// over the wavefront, every lane gets it: four steps within a row of 16 lanes, two exchanges of rows (a shuffle goes through the LDS pipeline)
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp_mov<0xB1>(v));
    v = fmaxf(v, dpp_mov<0x4E>(v));
    v = fmaxf(v, dpp_mov<0x141>(v));
    v = fmaxf(v, dpp_mov<0x140>(v));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// A lower bound of the wavefront's n-th largest value, n <= 64: its highest order bits, two at a time, until just n are left or 16 bits are known
__device__ __forceinline__ float wave_nth(float x, int n) {
    const unsigned key = order_bits(x);
    unsigned v = 0;
    int c = 64;
#pragma unroll 1
    for (int bit = 30; bit >= 16 && c > n; bit -= 2) {
        const int c1 = __popcll(__ballot(key >= (v | 1u << bit))), c2 = __popcll(__ballot(key >= (v | 2u << bit))), c3 = __popcll(__ballot(key >= (v | 3u << bit)));
        if (c3 >= n) v |= 3u << bit, c = c3;
        else if (c2 >= n) v |= 2u << bit, c = c2;
        else if (c1 >= n) v |= 1u << bit, c = c1;
    }
    const float f = from_order_bits(v);
    return f == f ? f : -INFINITY;
}

struct Cand {                           // a logit and its place in the vocabulary
    float x;
    int t;
};
struct Part {                           // a part of l_w: log of sum, plus m
    double sum;
    float m;
};
__device__ __forceinline__ bool before(float x, int t, const Cand& o) { return x > o.x || (x == o.x && t < o.t); }

// One wavefront's list in LDS, `count` of at most WAVE_CAP candidates -> its best n in order; returns how many there are
__device__ __forceinline__ int wave_keep_best(Cand* list, int count, int n, int lane) {
    wave_lds_sync();
    Cand mine[WAVE_CAP / 64];
    int rank[WAVE_CAP / 64];
#pragma unroll
    for (int i = 0; i < WAVE_CAP / 64; i++) {
        const int at = lane + 64 * i;
        mine[i] = at < count ? list[at] : Cand{0.f, 0};
        rank[i] = at < count ? 0 : NO_INDEX;
    }
    for (int k = 0; k < count; k++) {
        const Cand o = list[k];
#pragma unroll
        for (int i = 0; i < WAVE_CAP / 64; i++) rank[i] += before(o.x, o.t, mine[i]) ? 1 : 0;
    }
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < WAVE_CAP / 64; i++)
        if ((unsigned)rank[i] < (unsigned)n) list[rank[i]] = mine[i];
    wave_lds_sync();
    return min(count, n);
}

// A lane's pieces of 16 bytes of a row's tile; what lies behind the row reads as -inf.  The pieces count from the row's first logit wherever it lies in memory (the
// hardware loads 16 bytes from any element), so that equal rows have equal sums, bit for bit.
constexpr int PIECES = 4;               // of a lane and tile
template <typename T>
__device__ __forceinline__ void load_tile(const T* row, unsigned tile, unsigned V, int lane, u32x4 (&raw)[PIECES]) {
    constexpr unsigned N = 16 / sizeof(T), TILE = 64 * PIECES;
    typedef unsigned words __attribute__((ext_vector_type(4), aligned(2)));
    const unsigned t0 = (tile * TILE + lane) * N;                // (V < 2^31: no sum passes 2^32)
    if ((tile + 1) * TILE * N <= V) {                            // (the same for the whole wavefront: with a branch a lane each load was waited for before the next)
#pragma unroll
        for (int i = 0; i < PIECES; i++) raw[i] = *reinterpret_cast<const words*>(row + t0 + 64 * i * N);
        return;
    }
    constexpr unsigned NONE = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, f16>::value ? 0xfc00fc00u : 0xff80ff80u;      // -inf
    union {
        T e[PIECES][N];
        u32x4 v[PIECES];
    } u;
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        u.v[i] = u32x4{NONE, NONE, NONE, NONE};
#pragma unroll
        for (unsigned k = 0; k < N; k++) {
            const unsigned t = t0 + 64 * i * N + k;
            const T x = row[min(t, V - 1)];
            if (t < V) u.e[i][k] = x;
        }
        raw[i] = u.v[i];
    }
}
template <typename T>
__device__ __forceinline__ void unpack_piece(u32x4 v, float (&x)[16 / sizeof(T)]) {
    union {
        u32x4 v;
        T e[16 / sizeof(T)];
    } u;
    u.v = v;
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); i++) x[i] = as_float(u.e[i]);
}

// Workgroup (slice p, beam, sequence) of four wavefronts, each on `per_wave` tiles of its own of the beam's row: 64 lanes x 4 pieces of 16 bytes.
// What becomes a candidate has to be at least as large as a threshold.  At first that is the largest of the wavefronts' n-th largest lane maxima of their first
// tiles (n different logits are no smaller): of a random row about n candidates a workgroup are left, and almost every logit costs its
// exponential, a comparison and no more.  A wavefront collects its candidates in LDS; when the list has filled (rising or equal logits), it keeps the best
// n and raises its threshold.
// l_w: exponentials and their sum over a lane's part of a tile in float (each is off by 2^-23 and by the rounding of its argument, the sum of 32 by 6.5 2^-24 at most), all
// sums beyond in double: a wavefront may have a whole row, and added up in float equal logits were 1.7e-6 off over 122 tiles, 1e-5 over 2048.  Of normal rows with deviations
// 1 - 8 l_w is at most 1.4e-7 off.  (16 x 4 rows of 248320, both launches: 16.6 us, with float sums 16.2)
template <typename T>
__global__ __launch_bounds__(256) void select_scan_kernel(const T* __restrict__ logits, long stride_g, long stride_w, unsigned V, int n,
                                                          unsigned tiles, unsigned per_wave, Cand* __restrict__ best, Part* __restrict__ part) {
    constexpr int N = 16 / sizeof(T), TILE = 64 * PIECES;        // pieces a tile
    __shared__ Cand list_s[4][WAVE_CAP], flat_s[256];
    __shared__ int count_s[4];
    __shared__ float thr_s[4];
    __shared__ Part part_s[4];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const unsigned p = blockIdx.x, slices = gridDim.x, r = blockIdx.z * gridDim.y + blockIdx.y;
    const T* const row = logits + (long)blockIdx.z * stride_g + (long)blockIdx.y * stride_w;
    const unsigned first = min((4 * p + w) * per_wave, tiles), last = min(first + per_wave, tiles);
    Cand* const list = list_s[w];
    int count = 0;
    float m = -INFINITY;                                         // the wavefront's reference point
    double l = 0.0;                                              // this lane's sum of exp(x - m)
    float thr = -INFINITY;                                       // candidates are (x, t) at or before (thr, thr_t)
    int thr_t = NO_INDEX;
    if (first == last && lane == 0) thr_s[w] = -INFINITY;
    for (unsigned tile = first; tile < last || tile == first; tile++) {
        const bool real = tile < last;
        float x[PIECES][N], pm[PIECES];                          // and the pieces' maxima
        if (real) {
            u32x4 raw[PIECES];
            load_tile(row, tile, V, lane, raw);
#pragma unroll
            for (int i = 0; i < PIECES; i++) unpack_piece<T>(raw[i], x[i]);
#pragma unroll
            for (int i = 0; i < PIECES; i++) {
                pm[i] = fmaxf(x[i][0], x[i][1]);
#pragma unroll
                for (int e = 2; e < N; e += 2) pm[i] = fmaxf(fmaxf(pm[i], x[i][e]), x[i][e + 1]);
            }
            const float top = fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3]));
            if (tile == first) {
                const float t = wave_nth(top, n);
                if (lane == 0) thr_s[w] = t;
            }
            if (__any(top > m + REFERENCE_LAG)) {
                const float higher = wave_max(top);
                if (m > -INFINITY) l *= exp((double)m - (double)higher);             // (otherwise l is 0, or NaN already)
                m = higher;
            }
            const float ref = m == -INFINITY ? 0.f : m;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < PIECES; i++)
#pragma unroll
                for (int e = 0; e < N; e++) sum[e & 3] += __builtin_amdgcn_exp2f((x[i][e] - ref) * LOG2E);        // (x log2 e - ref log2 e would lose bits, or overflow)
            l += (double)((sum[0] + sum[1]) + (sum[2] + sum[3]));
        }
        if (tile == first) {                                     // (every wavefront comes by once)
            __syncthreads();
            thr = fmaxf(fmaxf(thr_s[0], thr_s[1]), fmaxf(thr_s[2], thr_s[3]));
        }
        if (!real) break;
        unsigned hits = 0;                                       // bit i * N + e
        const float low = fmaxf(thr, -3.402823466e38f);          // (-inf is no candidate)
#pragma unroll
        for (int i = 0; i < PIECES; i++)
            if (__any(pm[i] >= low)) {
#pragma unroll
                for (int e = 0; e < N; e++) hits |= x[i][e] >= low ? 1u << (i * N + e) : 0u;
            }
        while (__any(hits)) {                                    // each lane's next one; read again, which costs less than to find it among the registers
            const unsigned k = __builtin_ctz(hits | 1u << 31);
            const int t = (int)((tile * TILE + 64 * (k / N) + lane) * N + k % N);
            const float v = hits ? as_float(row[t]) : -INFINITY;
            const bool in = hits && (v > thr || (v == thr && t <= thr_t));
            hits &= hits - 1;
            const uint64_t who = __ballot(in);
            if (count + 64 > WAVE_CAP) {
                count = wave_keep_best(list, count, n, lane);
                if (count == n) thr = list[n - 1].x, thr_t = list[n - 1].t;
            }
            if (in) list[count + __popcll(who & ((1ull << lane) - 1))] = Cand{v, t};
            count += __popcll(who);
        }
    }
    // the wavefront's part of l_w
    {
        const double ll = wave_sum_d(l);
        if (lane == 0) part_s[w] = Part{ll, m}, count_s[w] = count;
    }
    __syncthreads();
    if (count_s[0] + count_s[1] + count_s[2] + count_s[3] > 256) {
        count = wave_keep_best(list, count, n, lane);
        __syncthreads();
        if (lane == 0) count_s[w] = count;
        __syncthreads();
    }
    // The four lists joined, and the best n of them: a candidate's place is the number of those that come before it, counted by four threads.  (A thread by itself, which
    // waits for every LDS read in turn, took 2.6 us of the launch's 8.)
    const int start = (w > 0 ? count_s[0] : 0) + (w > 1 ? count_s[1] : 0) + (w > 2 ? count_s[2] : 0);
    const int total = count_s[0] + count_s[1] + count_s[2] + count_s[3];
    for (int i = lane; i < count; i += 64) flat_s[start + i] = list[i];
    __syncthreads();
    const long out = ((long)r * slices + p) * n;
    for (int i0 = 0; i0 < total; i0 += 64) {
        const int i = i0 + (threadIdx.x >> 2);
        const Cand mine = flat_s[min(i, total - 1)];
        float rank = 0.f;
#pragma unroll 4
        for (int k = threadIdx.x & 3; k < total; k += 4) rank += before(flat_s[k].x, flat_s[k].t, mine) ? 1.f : 0.f;
        rank += dpp_mov<0xB1>(rank);
        rank += dpp_mov<0x4E>(rank);
        if (i < total && (threadIdx.x & 3) == 0 && rank < (float)n) best[out + (int)rank] = mine;
    }
    for (int i = total + threadIdx.x; i < n; i += 256) best[out + i] = Cand{-INFINITY, NO_INDEX};
    if (threadIdx.x < 4) {
        const Part own = part_s[threadIdx.x];
        float mm = own.m;
        mm = fmaxf(mm, dpp_mov<0xB1>(mm));
        mm = fmaxf(mm, dpp_mov<0x4E>(mm));
        double ll = own.sum * exp((double)own.m - (double)(mm == -INFINITY ? 0.f : mm));
        ll += dpp_mov_d<0xB1>(ll);
        ll += dpp_mov_d<0x4E>(ll);
        if (threadIdx.x == 0) part[(long)r * slices + p] = Part{ll, mm};
    }
}

struct Scored {
    double s;
    int w, t;
};
__device__ __forceinline__ bool before(const Scored& a, const Scored& b) { return a.s > b.s || (a.s == b.s && (a.w < b.w || (a.w == b.w && a.t < b.t))); }

// One workgroup of 16 wavefronts per sequence on the entries of its beams' slices.  Threshold as above: the largest of the wavefronts' n-th largest lane maxima.  What is
// no smaller goes into one list, a candidate's place is the number of those that come before it; should they not fit (many equal scores), the n
// places are filled one by one with the best candidate behind the one before.  Scores in double: floats of this size are 1e-6 apart, so they would change the order within
// a beam; candidates of two beams keep theirs as far as their l_w is known.
constexpr int JOIN_WAVES = 16, JOIN_THREADS = 64 * JOIN_WAVES, JOIN_CAP = 1024;
__global__ __launch_bounds__(JOIN_THREADS) void select_join_kernel(const Cand* __restrict__ best, const Part* __restrict__ part,
                                                                   const float* __restrict__ scores, int W, int n, int slices,
                                                                   float* __restrict__ out_s, int* __restrict__ out_w, int* __restrict__ out_t) {
    __shared__ double base_s[SELECT_MAX];                        // scores[v] - log of the beam's sum of exp(x - top_s[v])
    __shared__ float top_s[SELECT_MAX], thr_s[JOIN_WAVES];
    __shared__ __align__(16) Scored list_s[JOIN_CAP];
    __shared__ int count_s;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const long g = blockIdx.x;
    const int entries = W * slices * n, per_beam = slices * n;
    const Cand* const mine_in = best + g * entries;
    Cand c0 = {-INFINITY, NO_INDEX};                             // (on its way while the sums are joined)
    if ((int)threadIdx.x < entries) c0 = mine_in[threadIdx.x];
    if (threadIdx.x == 0) count_s = 0;
    for (int v = w; v < W; v += JOIN_WAVES) {
        const Part* pr = part + (g * W + v) * slices;
        Part own = {0.0, -INFINITY};
        if (lane < slices) own = pr[lane];
        float mm = own.m;
        for (int i = lane + 64; i < slices; i += 64) mm = fmaxf(mm, pr[i].m);
        mm = wave_max(mm);
        const float ref = mm == -INFINITY ? 0.f : mm;
        double ll = own.sum * exp((double)own.m - (double)ref);
        for (int i = lane + 64; i < slices; i += 64) ll += pr[i].sum * exp((double)pr[i].m - (double)ref);
        ll = wave_sum_d(ll);
        if (lane == 0) base_s[v] = (double)scores[g * W + v] - log(ll), top_s[v] = ref;
    }
    __syncthreads();
    auto entry = [&](int e) {
        const Cand c = e == (int)threadIdx.x ? c0 : mine_in[e];
        const int v = (unsigned)e / (unsigned)per_beam;
        const double s = base_s[v] + ((double)c.x - (double)top_s[v]);        // (the difference first: both may be the type's lowest value)
        return Scored{(float)s > -INFINITY && c.t != NO_INDEX ? s : -INFINITY, v, c.t};     // (as it is given out: a double may be below every float)
    };
    float top = -INFINITY;
    for (int e = threadIdx.x; e < entries; e += JOIN_THREADS) top = fmaxf(top, (float)entry(e).s);
    top = wave_nth(top, n);
    if (lane == 0) thr_s[w] = top;
    __syncthreads();
    float thr = thr_s[lane % JOIN_WAVES];
#pragma unroll
    for (int o = JOIN_WAVES / 2; o > 0; o >>= 1) thr = fmaxf(thr, __shfl_xor(thr, o));
    for (int e = threadIdx.x; e < entries; e += JOIN_THREADS) {
        const Scored c = entry(e);
        if (c.s > -INFINITY && (float)c.s >= thr) {
            const int at = atomicAdd(&count_s, 1);               // (the order does not matter)
            if (at < JOIN_CAP) list_s[at] = c;
        }
    }
    __syncthreads();
    const int count = count_s;
    auto put = [&](int place, const Scored& c) {
        out_s[g * n + place] = c.w < 0 ? -INFINITY : (float)c.s;
        out_w[g * n + place] = c.w;
        out_t[g * n + place] = c.t;
    };
    if (count <= JOIN_CAP) {
        for (int i0 = 0; i0 < count; i0 += JOIN_THREADS / 16) {  // (16 threads count for a candidate)
            const int i = i0 + (threadIdx.x >> 4);
            const Scored mine = list_s[min(i, count - 1)];
            float rank = 0.f;
            for (int k = threadIdx.x & 15; k < count; k += 16) rank += before(list_s[k], mine) ? 1.f : 0.f;
            rank = row16_sum(rank);
            if (i < count && (threadIdx.x & 15) == 0 && rank < (float)n) put((int)rank, mine);
        }
        for (int i = count + threadIdx.x; i < n; i += JOIN_THREADS) put(i, Scored{0.0, -1, -1});
        return;
    }
    Scored last = {INFINITY, -1, -1};                            // (count > JOIN_CAP > n: there are n)
    for (int place = 0; place < n; place++) {
        __syncthreads();                                         // (the list is read no more, and its first entries hold the wavefronts' best)
        Scored top1 = {-INFINITY, NO_INDEX, NO_INDEX};
        for (int e = threadIdx.x; e < entries; e += JOIN_THREADS) {
            const Scored c = entry(e);
            if (before(last, c) && before(c, top1)) top1 = c;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const Scored c = {__hiloint2double(__shfl_xor(__double2hiint(top1.s), o), __shfl_xor(__double2loint(top1.s), o)), __shfl_xor(top1.w, o), __shfl_xor(top1.t, o)};
            if (before(c, top1)) top1 = c;
        }
        if (lane == 0) list_s[w] = top1;
        __syncthreads();
        last = list_s[0];
        for (int v = 1; v < JOIN_WAVES; v++)
            if (before(list_s[v], last)) last = list_s[v];
        if (threadIdx.x == 0) put(place, last);
    }
}

// ---- reordering of states ----------------------------------------------------------------------------------------------------
constexpr int POOL_LAYERS = 48;         // layers of either kind in one launch (their pointers travel in the kernel arguments)
struct PoolTable {
    u32x4* ssm[POOL_LAYERS];
    u32x4* conv[POOL_LAYERS];
    u32x4* kv[2 * POOL_LAYERS];
};
constexpr int SSM_VEC = HV * DV * DK / 4, CONV_VEC = 3 * CD / 8, KV_VEC = AD / 8;
constexpr int KV_WGS = 8;               // workgroups on the rows of one (pool, sequence, head)

// The state of beam w of sequence g, in slot slots[g][w], becomes that of slot slots[g][parents[g][w]], for all beams of a sequence at once and in place.
// A thread owns one 16-byte place of the state in all of the sequence's slots: it loads what every beam takes over and stores it, so no beam's
// old state is overwritten before whoever needs it has read it, whatever the parents are, and nothing is exchanged.  A beam that is its own parent is
// not touched.  Blocks: ssm (layer, sequence, 4 KiB of a slot), conv (layer, sequence, 4 KiB of the live window), K / V (pool, sequence, head, part of the
// rows start .. pos - 1).
// UN: places a thread loads before it stores the first; stores are nontemporal.  Bound by HBM: 8 x 4 beams of 24 layers, 1200 rows of the caches, move 1.54 GB in 313 us
// (4.9 TB/s, a large copy reaches 5.2).  us at 1 x 4 / 8 x 4 beams: one place with plain stores 19.2 / 324, nontemporal stores 18.4 / 314, two places 17.9 /
// 313, four 19.3 / 317; nontemporal loads lose what two beams take from one parent (22.3 / 312).
// More beams, one / two / four places: 4 x 8 on 1650 rows 456 / 432 / 420, 1 x 8 206 / 178 / 178, 1 x 6 on 50 rows 25 / 25 / 30, 1 x 16 on 50 rows 97 / 121 / 125, 2 x 16 on 1650 742 / 595 / 487,
// 1 x 32 on 50 rows 265 / 457, on 1650 859 / 932: beyond 8 beams one place, which is better on short ranges and with 32 beams; long ranges of 16 beams would
// be faster with more.
template <int WMAX, int UN>
__global__ __launch_bounds__(256) void reorder_kernel(const PoolTable pools, const int* __restrict__ slots, const int* __restrict__ parents,
                                                      const int* __restrict__ start, const int* __restrict__ pos, int G, int W, int n_ssm, int n_slots,
                                                      int Lmax) {
    constexpr unsigned SSM_UNITS = SSM_VEC / (256 * UN), CONV_UNITS = (CONV_VEC + 256 * UN - 1) / (256 * UN);
    const unsigned ssm_blocks = (unsigned)n_ssm * G * SSM_UNITS, conv_blocks = (unsigned)n_ssm * G * CONV_UNITS;
    unsigned id = blockIdx.x;
    u32x4* base;
    size_t slot_stride;                                          // vectors from a slot to the next
    long first, end;                                             // this thread's first place, and the end of the places
    int step = 256, g;                                           // between a thread's places
    if (id < ssm_blocks) {
        const unsigned unit = id % SSM_UNITS, lg = id / SSM_UNITS;
        g = lg % G;
        base = pools.ssm[lg / G];
        slot_stride = SSM_VEC;
        first = unit * (256 * UN) + threadIdx.x, end = (unit + 1) * (256 * UN);
    } else if ((id -= ssm_blocks) < conv_blocks) {
        const unsigned unit = id % CONV_UNITS, lg = id / CONV_UNITS;
        g = lg % G;
        base = pools.conv[lg / G] + (pos[g] & 1) * CONV_VEC;
        slot_stride = 2 * CONV_VEC;
        first = unit * (256 * UN) + threadIdx.x, end = min((unit + 1) * (256 * UN), (unsigned)CONV_VEC);
    } else {
        id -= conv_blocks;
        const unsigned part = id % KV_WGS, head = id / KV_WGS % AKV, pg = id / KV_WGS / AKV;
        g = pg % G;
        base = pools.kv[pg / G] + (size_t)head * Lmax * KV_VEC;
        slot_stride = (size_t)AKV * Lmax * KV_VEC;
        first = (long)max(start[g], 0) * KV_VEC + part * 256 + threadIdx.x, end = (long)min(pos[g], Lmax) * KV_VEC, step = KV_WGS * 256;
    }
    int from[WMAX], to[WMAX];                                    // slots; from < 0: nothing to do
#pragma unroll
    for (int w = 0; w < WMAX; w++) {
        from[w] = to[w] = -1;
        if (w < W) {
            const int p = parents[g * W + w];
            to[w] = slots[g * W + w];
            if ((unsigned)p < (unsigned)W && p != w && (unsigned)to[w] < (unsigned)n_slots) from[w] = slots[g * W + p];
            if ((unsigned)from[w] >= (unsigned)n_slots) from[w] = -1;
        }
    }
    for (long at = first; at < end; at += (long)UN * step) {
        u32x4 v[UN][WMAX];
#pragma unroll
        for (int u = 0; u < UN; u++)
#pragma unroll
            for (int w = 0; w < WMAX; w++)
                if (from[w] >= 0 && at + (long)u * step < end) v[u][w] = base[(size_t)from[w] * slot_stride + at + (long)u * step];
#pragma unroll
        for (int u = 0; u < UN; u++)
#pragma unroll
            for (int w = 0; w < WMAX; w++)
                if (from[w] >= 0 && at + (long)u * step < end) __builtin_nontemporal_store(v[u][w], base + (size_t)to[w] * slot_stride + at + (long)u * step);
    }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// How a launch cuts its rows: tiles of 4 KiB, tiles a wavefront, workgroups (of four) a row.  Sixteen wavefronts a CU, which all fit, but no more than
// there are tiles (16 x 4 rows of 248320, us with 8 / 16 / 32 a CU: 23.1 / 17.3 / 18.8; a tile's loads ahead of the one before's arithmetic: no difference).  Beyond four rows a CU some of a
// workgroup's wavefronts have none, of the last workgroup of a row also below; the CU holds other workgroups then (1024 rows 172 us, 2048, two of whose four wavefronts have tiles, 351).
struct ScanPlan {
    unsigned tiles, per_wave, slices;
};
ScanPlan scan_plan(long rows, int V, int elem) {
    const long tiles = ((long)V * elem + 4095) / 4096, waves = std::max(1l, (long)qt::cu_count() * 16 / rows);
    const long per = (tiles + waves - 1) / waves;
    return {(unsigned)tiles, (unsigned)per, (unsigned)((tiles + 4 * per - 1) / (4 * per))};
}

}  // namespace

extern "C" {

long qt_beam_select_workspace_bytes(long G, int W, int V, int n, int elem_size) {
    if (G < 0 || W < 1 || W > SELECT_MAX || V < 1 || n < 1 || n > SELECT_MAX || (elem_size != 2 && elem_size != 4) || G * W > 65535) return -1;
    return G == 0 ? 0 : G * W * scan_plan(G * W, V, elem_size).slices * ((long)n * (long)sizeof(Cand) + (long)sizeof(Part));
}

int qt_beam_select(const void* logits, int dtype, long stride_g, long stride_w, const float* scores, float* out_scores, int32_t* out_parents,
                   int32_t* out_tokens, void* workspace, long workspace_bytes, int G, int W, int V, int n, hipStream_t stream) {
    if (dtype < 0 || dtype > 2) return QT_ERR_UNSUPPORTED;
    const int elem = dtype == 2 ? 4 : 2;
    const long need = qt_beam_select_workspace_bytes(G, W, V, n, elem);
    if (need < 0 || stride_g < 0 || stride_w < 0) return QT_ERR_DIM;
    if (G == 0) return QT_OK;
    if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !workspace) return QT_ERR_NULL;
    if (!aligned16(workspace) || (reinterpret_cast<uintptr_t>(logits) & (unsigned)(elem - 1))) return QT_ERR_ALIGN;
    if (workspace_bytes < need) return QT_ERR_WORKSPACE;
    const ScanPlan plan = scan_plan((long)G * W, V, elem);
    const int slices = (int)plan.slices;
    Part* const part = (Part*)workspace;
    Cand* const best = (Cand*)(part + (size_t)G * W * slices);
    const dim3 grid(plan.slices, (unsigned)W, (unsigned)G);
#define QT_SCAN(T) hipLaunchKernelGGL((select_scan_kernel<T>), grid, dim3(256), 0, stream, (const T*)logits, stride_g, stride_w, (unsigned)V, n, plan.tiles, \
                                      plan.per_wave, best, part)
    if (dtype == 0) QT_SCAN(bf16_t);
    else if (dtype == 1) QT_SCAN(f16);
    else QT_SCAN(float);
#undef QT_SCAN
    QT_CHECK_LAUNCH();
    hipLaunchKernelGGL(select_join_kernel, dim3((unsigned)G), dim3(64 * JOIN_WAVES), 0, stream, best, part, scores, W, n, slices, out_scores, out_parents,
                       out_tokens);
    QT_CHECK_LAUNCH();
    return QT_OK;
}

int qt_beam_reorder(float* const* ssm_pool, void* const* conv_pool, int n_gdn, void* const* kv_pool, int n_kv, const int32_t* slots,
                    const int32_t* parents, const int32_t* start, const int32_t* pos, int G, int W, int n_slots, int Lmax, hipStream_t stream) {
    if (n_gdn < 0 || n_kv < 0 || G < 0 || G > (1 << 16) || n_slots < 1 || (n_kv > 0 && Lmax < 1)) return QT_ERR_DIM;
    if (W < 1 || W > 32) return QT_ERR_UNSUPPORTED;
    if (G == 0) return QT_OK;
    if (!slots || !parents || !start || !pos) return QT_ERR_NULL;
    if ((n_gdn > 0 && (!ssm_pool || !conv_pool)) || (n_kv > 0 && !kv_pool)) return QT_ERR_NULL;
    for (int i = 0; i < n_gdn; i++) {
        if (!ssm_pool[i] || !conv_pool[i]) return QT_ERR_NULL;
        if (!aligned16(ssm_pool[i]) || !aligned16(conv_pool[i])) return QT_ERR_ALIGN;
    }
    for (int i = 0; i < n_kv; i++) {
        if (!kv_pool[i]) return QT_ERR_NULL;
        if (!aligned16(kv_pool[i])) return QT_ERR_ALIGN;
    }
    for (int a = 0, k = 0; a < n_gdn || k < n_kv;) {
        PoolTable t = {};
        const int na = n_gdn - a < POOL_LAYERS ? n_gdn - a : POOL_LAYERS, nk = n_kv - k < 2 * POOL_LAYERS ? n_kv - k : 2 * POOL_LAYERS;
        for (int i = 0; i < na; i++) t.ssm[i] = (u32x4*)ssm_pool[a + i], t.conv[i] = (u32x4*)conv_pool[a + i];
        for (int i = 0; i < nk; i++) t.kv[i] = (u32x4*)kv_pool[k + i];
        a += na, k += nk;
        const int un = W <= 8 ? 2 : 1, per = 256 * un;
        const long blocks = (long)na * G * (SSM_VEC / per + (CONV_VEC + per - 1) / per) + (long)nk * G * AKV * KV_WGS;
        if (blocks > 0x7fffffffl) return QT_ERR_DIM;
#define QT_REORDER(WM, UN) \
    hipLaunchKernelGGL((reorder_kernel<WM, UN>), dim3((unsigned)blocks), dim3(256), 0, stream, t, slots, parents, start, pos, G, W, na, n_slots, Lmax)
        if (W <= 4) QT_REORDER(4, 2);
        else if (W <= 8) QT_REORDER(8, 2);
        else if (W <= 16) QT_REORDER(16, 1);
        else QT_REORDER(32, 1);
#undef QT_REORDER
        QT_CHECK_LAUNCH();
    }
    return QT_OK;
}

}  // extern "C"
