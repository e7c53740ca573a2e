// Beam search on the slot pools, for gfx950: the selection over beams and vocabulary, and the reordering of the beams' states.
//
// Selection: with l_w = log sum_t exp(x[w][t]) the score of candidate (w, t) is scores[w] + x[w][t] - l_w; wanted are the n largest of a sequence's
// W V candidates, equal ones by the lower index w V + t.  The logits are read once: a launch over slices of the vocabulary keeps, per slice,
// its n largest logits and its part (maximum, sum) of l_w; a second launch joins the slices of a sequence's beams.
#include "qt_common.h"

using namespace qt;

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16;

constexpr int SELECT_MAX = 64;          // beams of a sequence, and candidates to select
constexpr int WAVE_CAP = 256;           // candidates a wavefront holds before it keeps the best n of them
constexpr int NO_INDEX = 0x7fffffff;

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

// the largest value v whose low 16 order bits are zero such that n of the wavefront's lanes hold at least v; n <= 64
__device__ __forceinline__ unsigned wave_nth_bits(unsigned key, int n) {
    unsigned v = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; bit--) {
        const unsigned t = v | 1u << bit;
        if (__popcll(__ballot(key >= t)) >= n) v = t;
    }
    return v;
}

struct Cand {                           // a logit and its place in the vocabulary
    float x;
    int t;
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

// the 16 bytes of logits number `piece` of a row; what lies behind the row reads as -inf.  The pieces count from the row's first logit wherever it lies in memory (the
// hardware loads 16 bytes from any element), so that equal rows have equal sums, bit for bit.
template <typename T>
__device__ __forceinline__ void load_piece(const T* row, long piece, int V, float (&x)[16 / sizeof(T)]) {
    constexpr int N = 16 / sizeof(T);
    typedef unsigned words __attribute__((ext_vector_type(4), aligned(2)));
    const long t0 = piece * N;
    if (t0 + N <= V) {
        union {
            u32x4 v;
            T e[N];
        } u;
        u.v = *reinterpret_cast<const words*>(row + t0);
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = as_float(u.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = t0 + i < V ? as_float(row[t0 + i]) : -INFINITY;
    }
}

// Workgroup (slice p, row r) of four wavefronts, each on a part of its own of the slice, in tiles of 64 lanes x 4 pieces of 16 bytes.
// A wavefront keeps a list of candidates in LDS.  What enters has to be at least as large as a threshold: after the first tile the n-th largest of
// the lanes' maxima (n different logits are no smaller), later the n-th best of the list, taken whenever it has filled.  So almost every
// logit costs a comparison, its exponential, and no more.
template <typename T>
__global__ __launch_bounds__(256) void select_scan_kernel(const T* __restrict__ logits, long stride_g, long stride_w, int W, int V, int n, int slices,
                                                          Cand* __restrict__ best, float2* __restrict__ part) {
    constexpr int N = 16 / sizeof(T), PIECES = 4, TILE = 64 * PIECES;         // pieces a tile
    __shared__ Cand list_s[4][WAVE_CAP];
    __shared__ int count_s[4];
    __shared__ float2 ml_s[4];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int p = blockIdx.x, r = blockIdx.y;
    const T* const row = logits + (long)(r / W) * stride_g + (long)(r % W) * stride_w;
    const long pieces = ((long)V + N - 1) / N, tiles = (pieces + TILE - 1) / TILE;
    // tiles of the row dealt out evenly to 4 * slices wavefronts
    const long parts = 4l * slices, me = 4l * p + w;
    const long first = tiles * me / parts, last = tiles * (me + 1) / parts;
    Cand* const list = list_s[w];
    int count = 0;
    float m = -INFINITY, l = 0.f;
    float thr = -INFINITY;                                       // candidates are (x, t) at or before (thr, thr_t)
    int thr_t = NO_INDEX;
    for (long tile = first; tile < last; tile++) {
        float x[PIECES][N];
#pragma unroll
        for (int i = 0; i < PIECES; i++) load_piece(row, tile * TILE + 64 * i + lane, V, x[i]);
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < PIECES; i++)
#pragma unroll
            for (int e = 0; e < N; e++) top = fmaxf(top, x[i][e]);
        const float m_new = fmaxf(m, top), ref = m_new == -INFINITY ? 0.f : m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < PIECES; i++)
#pragma unroll
            for (int e = 0; e < N; e++) sum += __expf(x[i][e] - ref);
        l = l * __expf(m - ref) + sum;                           // (m = -inf: l is 0, or NaN already)
        m = m_new;
        if (tile == first) thr = from_order_bits(wave_nth_bits(order_bits(top), n));
        if (!(thr == thr)) thr = -INFINITY;
#pragma unroll 1
        for (int i = 0; i < PIECES; i++) {
            bool any = false;
            float xi[N];
#pragma unroll
            for (int e = 0; e < N; e++) {
                xi[e] = i == 0 ? x[0][e] : i == 1 ? x[1][e] : i == 2 ? x[2][e] : x[3][e];
                any |= xi[e] >= thr;
            }
            if (!__any(any)) continue;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const int t = (int)((tile * TILE + 64 * i + lane) * N + e);
                const bool in = xi[e] > -INFINITY && (xi[e] > thr || (xi[e] == thr && t <= thr_t));
                const uint64_t who = __ballot(in);
                if (!who) continue;
                if (count + 64 > WAVE_CAP) {
                    count = wave_keep_best(list, count, n, lane);
                    if (count == n) thr = list[n - 1].x, thr_t = list[n - 1].t;
                }
                if (in) list[count + __popcll(who & ((1ull << lane) - 1))] = Cand{xi[e], t};
                count += __popcll(who);
            }
        }
    }
    count = wave_keep_best(list, count, n, lane);
    // the wavefront's part of l_w
    {
        float mm = m;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
        const float ref = mm == -INFINITY ? 0.f : mm;
        float ll = l * __expf(m - ref);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) ll += __shfl_xor(ll, o);
        if (lane == 0) ml_s[w] = make_float2(mm, ll), count_s[w] = count;
    }
    __syncthreads();
    // the four lists joined: a candidate's place is the number of those that come before it
    const long out = ((long)r * slices + p) * n;
    const int c[4] = {count_s[0], count_s[1], count_s[2], count_s[3]};
    const int total = c[0] + c[1] + c[2] + c[3];
    if (lane < c[w]) {
        const Cand mine = list[lane];
        int rank = 0;
        for (int v = 0; v < 4; v++)
            for (int k = 0; k < c[v]; k++) rank += before(list_s[v][k].x, list_s[v][k].t, mine) ? 1 : 0;
        if (rank < n) best[out + rank] = mine;
    }
    for (int i = total + threadIdx.x; i < n; i += 256) best[out + i] = Cand{-INFINITY, NO_INDEX};
    if (threadIdx.x == 0) {
        float mm = ml_s[0].x;
        for (int v = 1; v < 4; v++) mm = fmaxf(mm, ml_s[v].x);
        const float ref = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f;
        for (int v = 0; v < 4; v++) ll += ml_s[v].y * __expf(ml_s[v].x - ref);
        part[(long)r * slices + p] = make_float2(mm, ll);
    }
}

struct Scored {
    double s;
    int w, t;
};
__device__ __forceinline__ bool before(const Scored& a, const Scored& b) { return a.s > b.s || (a.s == b.s && (a.w < b.w || (a.w == b.w && a.t < b.t))); }

// One workgroup of 16 wavefronts per sequence.  Every slice's list is in order, so of a list whose first entry is not among the n best first entries
// nothing is wanted: each wavefront finds the n-th best first entry of its share of the lists (by value, rounded down), takes what is no smaller from them,
// and keeps its best n; then the 16 n are joined.  Scores in double: two beams' candidates may lie closer than floats tell apart.
constexpr int JOIN_WAVES = 16, JOIN_CAP = 192;
__global__ __launch_bounds__(64 * JOIN_WAVES) void select_join_kernel(const Cand* __restrict__ best, const float2* __restrict__ part,
                                                                      const float* __restrict__ scores, int W, int n, int slices,
                                                                      float* __restrict__ out_s, int* __restrict__ out_w, int* __restrict__ out_t) {
    __shared__ double base_s[SELECT_MAX];                        // scores[v] - log of the beam's sum of exp(x - top_s[v])
    __shared__ float top_s[SELECT_MAX];
    __shared__ __align__(16) Scored list_s[JOIN_WAVES][JOIN_CAP];
    __shared__ int count_s[JOIN_WAVES];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const long g = blockIdx.x;
    for (int v = w; v < W; v += JOIN_WAVES) {
        const float2* pr = part + (g * W + v) * slices;
        float mm = -INFINITY;
        for (int i = lane; i < slices; i += 64) mm = fmaxf(mm, pr[i].x);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
        const float ref = mm == -INFINITY ? 0.f : mm;
        double ll = 0.0;
        for (int i = lane; i < slices; i += 64) ll += (double)pr[i].y * exp((double)pr[i].x - (double)ref);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) ll += __hiloint2double(__shfl_xor(__double2hiint(ll), o), __shfl_xor(__double2loint(ll), o));
        if (lane == 0) base_s[v] = (double)scores[g * W + v] - log(ll), top_s[v] = ref;
    }
    __syncthreads();
    const int lists = W * slices;
    const int l0 = (int)((long)lists * w / JOIN_WAVES), l1 = (int)((long)lists * (w + 1) / JOIN_WAVES);
    Scored* const list = list_s[w];
    int count = 0;
    auto entry = [&](int li, int k) {
        const Cand c = best[(g * lists + li) * n + k];
        const int v = li / slices;
        const double s = base_s[v] + ((double)c.x - (double)top_s[v]);        // (the difference first: both may be the type's lowest value)
        return Scored{s == s && c.t != NO_INDEX ? s : -INFINITY, v, c.t};
    };
    // (several lanes' maxima of first entries: n different entries are no smaller than the n-th of them)
    float top = -INFINITY;
    for (int li = l0 + lane; li < l1; li += 64) top = fmaxf(top, (float)entry(li, 0).s);
    float thr = from_order_bits(wave_nth_bits(order_bits(top), n));
    if (!(thr == thr)) thr = -INFINITY;
    auto keep = [&] {
        wave_lds_sync();
        Scored mine[JOIN_CAP / 64];
        int rank[JOIN_CAP / 64];
#pragma unroll
        for (int i = 0; i < JOIN_CAP / 64; i++) {
            const int at = lane + 64 * i;
            mine[i] = at < count ? list[at] : Scored{0.0, 0, 0};
            rank[i] = at < count ? 0 : NO_INDEX;
        }
        for (int k = 0; k < count; k++) {
            const Scored o = list[k];
#pragma unroll
            for (int i = 0; i < JOIN_CAP / 64; i++) rank[i] += before(o, mine[i]) ? 1 : 0;
        }
        wave_lds_sync();
#pragma unroll
        for (int i = 0; i < JOIN_CAP / 64; i++)
            if ((unsigned)rank[i] < (unsigned)n) list[rank[i]] = mine[i];
        wave_lds_sync();
        count = min(count, n);
    };
    for (int b0 = l0; b0 < l1; b0 += 64) {
        for (int k = 0; k < n; k++) {                            // entry k of 64 lists
            bool in = false;
            Scored e = {-INFINITY, 0, 0};
            if (b0 + lane < l1) {
                e = entry(b0 + lane, k);
                in = e.s > -INFINITY && (float)e.s >= thr;
            }
            const uint64_t who = __ballot(in);
            if (!who) break;                                     // (every list is in order)
            if (count + 64 > JOIN_CAP) {
                keep();
                if (count == n) thr = fmaxf(thr, (float)list[n - 1].s);
            }
            if (in) list[count + __popcll(who & ((1ull << lane) - 1))] = e;
            count += __popcll(who);
        }
    }
    keep();
    if (lane == 0) count_s[w] = count;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int v = 0; v < JOIN_WAVES; v++) total += count_s[v];
    if (lane < count) {
        const Scored mine = list[lane];
        int rank = 0;
        for (int v = 0; v < JOIN_WAVES; v++) {
            const int cv = count_s[v];
            for (int k = 0; k < cv; k++) {
                if (!before(list_s[v][k], mine)) break;          // (in order)
                rank++;
            }
        }
        if (rank < n) {
            out_s[g * n + rank] = (float)mine.s;
            out_w[g * n + rank] = mine.w;
            out_t[g * n + rank] = mine.t;
        }
    }
    for (int i = total + threadIdx.x; i < n; i += 64 * JOIN_WAVES) {
        out_s[g * n + i] = -INFINITY;
        out_w[g * n + i] = -1;
        out_t[g * n + i] = -1;
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
constexpr int SSM_UNITS = SSM_VEC / 256, CONV_UNITS = (CONV_VEC + 255) / 256, KV_WGS = 8;

// The state of beam w of sequence g, in slot slots[g][w], becomes that of slot slots[g][parents[g][w]], for all beams of a sequence at once and in place.
// A thread owns one 16-byte place of the state in all of the sequence's slots: it loads what every beam takes over and stores it, so no beam's
// old state is overwritten before whoever needs it has read it, whatever the parents are, and nothing is exchanged.  A beam that is its own parent is
// not touched.  Blocks: ssm (layer, sequence, 4 KiB of a slot), conv (layer, sequence, 4 KiB of the live window), K / V (pool, sequence, head, part of the
// rows start .. pos - 1).
template <int WMAX>
__global__ __launch_bounds__(256) void reorder_kernel(const PoolTable pools, const int* __restrict__ slots, const int* __restrict__ parents,
                                                      const int* __restrict__ start, const int* __restrict__ pos, int G, int W, int n_ssm, int n_slots,
                                                      int Lmax) {
    const unsigned ssm_blocks = (unsigned)n_ssm * G * SSM_UNITS, conv_blocks = (unsigned)n_ssm * G * CONV_UNITS;
    unsigned id = blockIdx.x;
    u32x4* base;
    size_t slot_stride;                                          // vectors from a slot to the next
    long first, end;                                             // this thread's first place, and the end of the places
    int step, g;
    if (id < ssm_blocks) {
        const unsigned unit = id % SSM_UNITS, lg = id / SSM_UNITS;
        g = lg % G;
        base = pools.ssm[lg / G];
        slot_stride = SSM_VEC;
        first = unit * 256 + threadIdx.x, end = SSM_VEC, step = SSM_VEC;
    } else if ((id -= ssm_blocks) < conv_blocks) {
        const unsigned unit = id % CONV_UNITS, lg = id / CONV_UNITS;
        g = lg % G;
        base = pools.conv[lg / G] + (pos[g] & 1) * CONV_VEC;
        slot_stride = 2 * CONV_VEC;
        first = unit * 256 + threadIdx.x, end = CONV_VEC, step = CONV_VEC;
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
    for (long at = first; at < end; at += step) {
        u32x4 v[WMAX];
#pragma unroll
        for (int w = 0; w < WMAX; w++)
            if (from[w] >= 0) v[w] = base[(size_t)from[w] * slot_stride + at];
#pragma unroll
        for (int w = 0; w < WMAX; w++)
            if (from[w] >= 0) base[(size_t)to[w] * slot_stride + at] = v[w];
    }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// slices of a row: enough wavefronts for every CU to hold eight, but no more than the row has tiles of 4 KiB
int select_slices(long rows, int V, int elem) {
    const long tiles = ((long)V * elem + 4095) / 4096, most = (tiles + 3) / 4;
    const long want = ((long)qt::cu_count() * 2 + rows - 1) / rows;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

}  // namespace

extern "C" {

long qt_beam_select_workspace_bytes(long G, int W, int V, int n, int elem_size) {
    if (G < 0 || W < 1 || W > SELECT_MAX || V < 1 || n < 1 || n > SELECT_MAX || (elem_size != 2 && elem_size != 4) || G * W > 65535) return -1;
    return G == 0 ? 0 : G * W * select_slices(G * W, V, elem_size) * ((long)n * (long)sizeof(Cand) + (long)sizeof(float2));
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
    const int slices = select_slices((long)G * W, V, elem);
    float2* const part = (float2*)workspace;
    Cand* const best = (Cand*)(part + (size_t)G * W * slices);
    const dim3 grid((unsigned)slices, (unsigned)(G * W));
#define QT_SCAN(T) hipLaunchKernelGGL((select_scan_kernel<T>), grid, dim3(256), 0, stream, (const T*)logits, stride_g, stride_w, W, V, n, slices, best, part)
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
        const long blocks = (long)na * G * (SSM_UNITS + CONV_UNITS) + (long)nk * G * AKV * KV_WGS;
        if (blocks > 0x7fffffffl) return QT_ERR_DIM;
#define QT_REORDER(WM) \
    hipLaunchKernelGGL((reorder_kernel<WM>), dim3((unsigned)blocks), dim3(256), 0, stream, t, slots, parents, start, pos, G, W, na, n_slots, Lmax)
        if (W <= 4) QT_REORDER(4);
        else if (W <= 8) QT_REORDER(8);
        else if (W <= 16) QT_REORDER(16);
        else QT_REORDER(32);
#undef QT_REORDER
        QT_CHECK_LAUNCH();
    }
    return QT_OK;
}

}  // extern "C"
