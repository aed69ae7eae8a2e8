// Softmax cross entropy of the rows of a matrix of logits, whole or in pieces of the vocabulary,
// and its gradient.
//
// Bandwidth bound: a loss reads the logits once, a gradient reads them once and writes as many.
//   * Loss and gradient in one call, rows that fit a workgroup's registers: the row is read once, its
//     maximum and sum go over the workgroup, the gradient leaves from the registers; a register that
//     has been stored takes the next row's elements at once, so loads and stores overlap.
//   * Everything else is cut into tiles of a row: a tile leaves its maximum and sum (a record, or the
//     row's result where it has one tile), and the gradient of a tile folds the row's records.
// bf16 [8192, 128000], loss and gradient: 799 us (5.3 TB/s), loss alone 308 (6.8); [8192, 151936], rows too long for a
// workgroup's registers, which are read twice: 1191 us (6.3 TB/s of three crossings), loss alone 363 (6.9).  fp16
// [4096, 8192] pieces: 17.7 us a state (3.8 TB/s), 24.1 a gradient (5.6 TB/s).  Loss of fp32 [64, 32000]: 6.4 us.
// Sums and maxima are fp32; exponentials are the hardware's 2^x of (x - maximum) log2(e), where the
// difference comes first: it is exact for neighbours, whatever the logits' common offset.  An fp32 gradient's own
// exponentials are exact to the function's error (scaled_exp); a sum is not nearer to 64 bits for it.
#include <atomic>
#include <utility>

#include "sequence.hip.h"

namespace dlfx {
namespace {

// The rows' target columns, 32 or 64 bits each.
struct Targets {
    const void* base;
    bool wide;
    __device__ __forceinline__ int64_t operator[](int64_t r) const {
        return wide ? static_cast<const int64_t*>(base)[r] : static_cast<const int32_t*>(base)[r];
    }
};

// Running maximum of a row and the sum of exp(x - maximum).
struct MaxSum {
    float mx, sum;
};
constexpr float kNone = -std::numeric_limits<float>::infinity();
constexpr float kLargest = std::numeric_limits<float>::max();

__device__ __forceinline__ float exp_diff(float x, float mx) { return __builtin_amdgcn_exp2f((x - mx) * kLog2E); }

// factor * exp(x - mx), an element of a gradient.  For fp32 elements what the product with log2(e) loses, d u of the
// result at a distance d below the maximum, is made up for to first order; ln 2 itself, rounded, leaves d u / 22.
// Two-byte elements round far above it.
template <typename S>
__device__ __forceinline__ float scaled_exp(float factor, float x, float mx) {
    if constexpr (sizeof(S) == 4) {
        const float d = x - mx, t = d * kLog2E;
        const float v = factor * __builtin_amdgcn_exp2f(t);
        // (under 2^-16 wherever exp(d) is not 0; far below and of -inf any number will do, and a NaN is in v as well)
        const float left = __builtin_amdgcn_fmed3f(fmaf(-t, 0.693147180559945309417f, d), -0x1p-16f, 0x1p-16f);
        return fmaf(v, left, v);
    } else {
        return factor * exp_diff(x, mx);
    }
}

__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
    const float mx = fmaxf(a.mx, b.mx);
    // an empty side (maximum -inf) adds its sum of 0, or the NaN that the side has met
    const float fa = a.mx == mx ? 1.0f : exp_diff(a.mx, mx);
    const float fb = b.mx == mx ? 1.0f : exp_diff(b.mx, mx);
    return {mx, a.sum * fa + b.sum * fb};
}

// Folds N values in.  Differences are taken to a finite maximum: -inf adds 0 to an empty row, +inf
// makes the sum infinite, a NaN stays.
template <int N>
__device__ __forceinline__ void fold(MaxSum& s, const float (&v)[N]) {
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, v[i]);
    mx = fmaxf(mx, s.mx);
    const float to = fminf(fmaxf(mx, -kLargest), kLargest);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) sum += exp_diff(v[i], to);
    s.sum = (s.mx == mx ? s.sum : s.sum * exp_diff(s.mx, to)) + sum;
    s.mx = mx;
}

// Over a wavefront: the maxima first, so that a lane scales its sum once.
__device__ __forceinline__ MaxSum wave_join(MaxSum s) {
    const float mx = wave_reduce(s.mx, [](float a, float b) { return fmaxf(a, b); });
    if (s.mx != mx) s.sum *= exp_diff(s.mx, fminf(mx, kLargest));
    return {mx, wave_reduce(s.sum, [](float a, float b) { return a + b; })};
}

// Over the T threads of a workgroup; every thread gets the result.  Two uses in a row need different
// `lds` or a barrier between them.
template <int T>
__device__ __forceinline__ MaxSum block_join(MaxSum v, MaxSum* lds) {
    constexpr int WAVES = T / kWave;
    v = wave_join(v);
    if (lane_id() == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = lds[lane_id() % WAVES];
    return group_reduce(v, WAVES, join);
}

// Loss of a finished row.  log(sum) + (maximum - logit) in this order: the difference is exact for
// nearby values, maximum + log(sum) would round at the maximum's size.
__device__ __forceinline__ float loss_of(MaxSum s, float logit, float z) {
    if (s.sum == 0.0f) return std::numeric_limits<float>::infinity();
    const float log_sum = logf(s.sum);
    float loss = log_sum + (s.mx - logit);
    if (z != 0.0f) {
        const float lse = s.mx + log_sum;
        loss += z * lse * lse;
    }
    return loss;
}

// What the elements of a row's gradient have in common: dx = p * exp(x - mx) - [target] * up.
struct RowGrad {
    float mx, p, up;
    bool zero;                // a row without a target, or of nothing but -inf
};
__device__ __forceinline__ RowGrad row_grad(MaxSum s, bool live, float weight, float z) {
    RowGrad g = {fminf(fmaxf(s.mx, -kLargest), kLargest), 0.0f, weight, !live || s.sum == 0.0f};
    float factor = 1.0f / s.sum;
    if (z != 0.0f) factor *= 1.0f + 2.0f * z * (s.mx + logf(s.sum));
    g.p = weight * factor;
    return g;
}

template <typename S> constexpr int vector_width() { return 16 / static_cast<int>(sizeof(S)); }

// A vector while it waits in registers: four words, whatever the type (vectors of 16-bit elements
// carried round a loop would take a register per element).
typedef uint32_t Words4 __attribute__((ext_vector_type(4)));
template <int BYTES> struct WordsAt;                 // in memory, on an element's boundary
template <> struct WordsAt<2> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2), may_alias)); };
template <> struct WordsAt<4> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4), may_alias)); };
template <typename S>
__device__ __forceinline__ Words4 load_words(const S* at) { return __builtin_nontemporal_load(reinterpret_cast<const typename WordsAt<sizeof(S)>::type*>(at)); }
template <typename S>
__device__ __forceinline__ void widen(const Words4& w, float (&v)[vector_width<S>()]) {
    if constexpr (sizeof(S) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = bit_cast<float>(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const Vec<S, 2> pair = bit_cast<Vec<S, 2>>(static_cast<uint32_t>(w[i]));
            v[2 * i] = static_cast<float>(pair.v[0]);
            v[2 * i + 1] = static_cast<float>(pair.v[1]);
        }
    }
}

// V elements from position e0 of a row of n, as they are stored; -inf past the end.
template <typename S>
__device__ __forceinline__ Words4 load_part(const S* row, int64_t e0, int64_t n) {
    constexpr int V = vector_width<S>();
    if (e0 + V <= n) return load_words(row + e0);
    Vec<S, V> v;
#pragma unroll
    for (int i = 0; i < V; ++i) v.v[i] = e0 + i < n ? row[e0 + i] : static_cast<S>(kNone);
    return bit_cast<Words4>(v);
}
template <typename S>
__device__ __forceinline__ Vec<S, vector_width<S>()> grad_vector(int64_t e0, const Words4& x, const RowGrad& g, int64_t target) {
    constexpr int V = vector_width<S>();
    float v[V];
    widen<S>(x, v);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = scaled_exp<S>(g.p, v[i], g.mx);
    const uint64_t at = static_cast<uint64_t>(target - e0);
    if (at < V) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (at == static_cast<uint64_t>(i)) v[i] -= g.up;
    }
    Vec<S, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) out.v[i] = static_cast<S>(g.zero ? 0.0f : v[i]);
    return out;
}
template <typename S>
__device__ __forceinline__ void store_whole(S* at, const Vec<S, vector_width<S>()>& v) {
    const typename WordsAt<sizeof(S)>::type words = bit_cast<Words4>(v);
    __builtin_nontemporal_store(words, reinterpret_cast<typename WordsAt<sizeof(S)>::type*>(at));
}
template <typename S>
__device__ __forceinline__ void store_part(S* row, int64_t e0, int64_t n, const Vec<S, vector_width<S>()>& v) {
    constexpr int V = vector_width<S>();
    if (e0 + V <= n) {
        store_whole(row + e0, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (e0 + i < n) row[e0 + i] = v.v[i];
    }
}

// Loss and gradient of whole rows held in registers: NV vectors to a thread, the last of them at or
// over the row's end for some; a workgroup takes every gridDim-th row.  All other loads and stores
// are unconditional, so the next row's loads are still in flight while its first vectors are summed.
template <typename S, int NV, int T>
__global__ __launch_bounds__(T) void grad_rows_held(const S* x, int64_t m, int64_t n, int64_t stride, Targets targets, const float* weights, float z,
                                                    float* loss, S* dx, int64_t dx_stride) {
    constexpr int V = vector_width<S>();
    __shared__ MaxSum lds[2][T / kWave];
    const uint32_t mine = threadIdx.x * V;
    const int64_t end = (NV - 1) * T * V + static_cast<int64_t>(mine);      // where the thread's last vector begins
    auto load = [&](const S* row, int j) { return load_words(row + j * T * V + mine); };
    Words4 raw[NV];
    int64_t r = blockIdx.x;
    raw[NV - 1] = load_part(x + r * stride, end, n);
#pragma unroll
    for (int j = 0; j < NV - 1; ++j) raw[j] = load(x + r * stride, j);
    for (int parity = 0; r < m; r += gridDim.x, parity ^= 1) {
        const int64_t target = targets[r];
        const float weight = weights ? weights[r] : 1.0f;
        MaxSum s = {kNone, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float v[V];
            widen<S>(raw[j], v);
            fold(s, v);
            __builtin_amdgcn_sched_barrier(0);
        }
        float logit = std::numeric_limits<float>::quiet_NaN();
        if (threadIdx.x == 0 && loss && target >= 0 && target < n) logit = static_cast<float>(x[r * stride + target]);
        asm volatile("" : "+v"(logit));             // (here, not later: dx may be x, and others store after the barrier)
        s = block_join<T>(s, lds[parity]);
        if (threadIdx.x == 0 && loss) loss[r] = target < 0 ? 0.0f : loss_of(s, logit, z);
        const RowGrad g = row_grad(s, target >= 0, weight, z);
        S* dr = dx + r * dx_stride;
        const int64_t next = r + gridDim.x < m ? r + gridDim.x : r;      // (past the last row: values that nobody uses)
        const S* xn = x + next * stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) asm volatile("" : "+v"(raw[j]));      // (the words are kept, not the floats the sum was made of)
#pragma unroll
        for (int j = 0; j < NV - 1; ++j) {
            store_whole(dr + j * T * V + mine, grad_vector<S>(j * T * V + static_cast<int64_t>(mine), raw[j], g, target));
            raw[j] = load(xn, j);
            __builtin_amdgcn_sched_barrier(0);
        }
        store_part(dr, end, n, grad_vector<S>(end, raw[NV - 1], g, target));
        raw[NV - 1] = load_part(xn, end, n);
    }
}

// Rows shorter than a vector: a thread each.
template <typename S>
__global__ __launch_bounds__(256) void grad_rows_tiny(const S* x, int64_t m, int n, int64_t stride, Targets targets, const float* weights, float z,
                                                      float* loss, S* dx, int64_t dx_stride) {
    constexpr int V = vector_width<S>();
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (r >= m) return;
    const int64_t target = targets[r];
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < n ? static_cast<float>(x[r * stride + i]) : kNone;
    MaxSum s = {kNone, 0.0f};
    fold(s, v);
    float logit = std::numeric_limits<float>::quiet_NaN();
#pragma unroll
    for (int i = 0; i < V; ++i) logit = i == target && i < n ? v[i] : logit;
    if (loss) loss[r] = target < 0 ? 0.0f : loss_of(s, logit, z);
    const RowGrad g = row_grad(s, target >= 0, weights ? weights[r] : 1.0f, z);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < n) dx[r * dx_stride + i] = static_cast<S>(g.zero ? 0.0f : scaled_exp<S>(g.p, v[i], g.mx) - (i == target ? g.up : 0.0f));
}

// A row cut into tiles, a workgroup each: workgroup = row * tiles + tile.
constexpr int kTileThreads = 256;
constexpr int kTileBatch = 4;                       // vectors of a thread in flight
template <typename S, int T = kTileThreads> constexpr int64_t tile_unit() { return static_cast<int64_t>(T) * vector_width<S>(); }

struct Tiles {
    int64_t count, length;
};

// Workgroups of a pass over tiles in rows of 2^20: along one axis of the grid there can be 2^24.
constexpr uint32_t kGridRow = 1u << 20;
inline dim3 grid_of(int64_t workgroups) {
    if (workgroups <= kGridRow) return dim3(static_cast<unsigned>(workgroups));
    return dim3(kGridRow, static_cast<unsigned>(ceil_div(workgroups, kGridRow)));
}
__device__ __forceinline__ uint32_t workgroup() { return blockIdx.y * kGridRow + blockIdx.x; }

// What a call on a matrix of logits works on; state or loss is where a finished row goes.
template <typename S>
struct LossCall {
    const S* x;
    int64_t m, n, stride;
    Targets targets;
    int64_t first;               // column of the whole vocabulary that column 0 is
    int resume;
    float* state;
    float z;
    float* loss;
    Tiles tiles;
    MaxSum* records;             // tiles.count per row
};

template <typename S>
__device__ __forceinline__ void finish_row(const LossCall<S>& p, int64_t r, MaxSum v) {
    const int64_t target = p.targets[r];
    float logit = std::numeric_limits<float>::quiet_NaN();
    if (!p.loss && p.resume) {
        v = join({p.state[r], p.state[p.m + r]}, v);
        logit = p.state[2 * p.m + r];
    }
    if (target >= p.first && target - p.first < p.n) logit = static_cast<float>(p.x[r * p.stride + (target - p.first)]);
    if (p.loss) {
        p.loss[r] = target < 0 ? 0.0f : loss_of(v, logit, p.z);
    } else {
        p.state[r] = v.mx;
        p.state[p.m + r] = v.sum;
        p.state[2 * p.m + r] = logit;
    }
}

// A tile's record, or with one tile to a row the row's result.
template <typename S, int T>
__global__ __launch_bounds__(T) void loss_tiles(LossCall<S> p) {
    constexpr int V = vector_width<S>();
    __shared__ MaxSum lds[T / kWave];
    const uint32_t tiles = static_cast<uint32_t>(p.tiles.count);
    const uint32_t here = workgroup();
    const int64_t r = here / tiles, tile = here % tiles;
    if (r >= p.m) return;
    const S* xr = p.x + r * p.stride;
    const int64_t begin = tile * p.tiles.length;
    const int64_t end = begin + p.tiles.length < p.n ? begin + p.tiles.length : p.n;
    MaxSum s = {kNone, 0.0f};
    for (int64_t e0 = begin + static_cast<int64_t>(threadIdx.x) * V; e0 < end; e0 += kTileBatch * tile_unit<S, T>()) {
        Words4 raw[kTileBatch];
        float part[V];
        if (e0 + (kTileBatch - 1) * tile_unit<S, T>() + V <= end) {
            float v[kTileBatch * V];
#pragma unroll
            for (int u = 0; u < kTileBatch; ++u) raw[u] = load_words(xr + e0 + u * tile_unit<S, T>());
#pragma unroll
            for (int u = 0; u < kTileBatch; ++u) {
                widen<S>(raw[u], part);
#pragma unroll
                for (int i = 0; i < V; ++i) v[u * V + i] = part[i];
            }
            fold(s, v);
        } else {
#pragma unroll
            for (int u = 0; u < kTileBatch; ++u) {
                const int64_t e = e0 + u * tile_unit<S, T>();
                if (e < end) raw[u] = load_part(xr, e, end);
            }
#pragma unroll
            for (int u = 0; u < kTileBatch; ++u) {
                if (e0 + u * tile_unit<S, T>() >= end) break;
                widen<S>(raw[u], part);
                fold(s, part);
            }
        }
    }
    s = block_join<T>(s, lds);
    if (threadIdx.x) return;
    if (p.tiles.count > 1 || !(p.loss || p.state)) p.records[here] = s;
    else finish_row(p, r, s);
}

__device__ __forceinline__ MaxSum join_records(const MaxSum* records, int64_t count) {
    MaxSum s = {kNone, 0.0f};
    for (int64_t t = lane_id(); t < count; t += kWave) s = join(s, records[t]);
    return wave_join(s);
}

// One wavefront per row joins its records.
template <typename S>
__global__ __launch_bounds__(256) void loss_join_tiles(LossCall<S> p) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    if (r >= p.m) return;
    const MaxSum s = join_records(p.records + r * p.tiles.count, p.tiles.count);
    if (lane_id() == 0) finish_row(p, r, s);
}

__global__ __launch_bounds__(256) void loss_join(int64_t m, Targets targets, const float* state, float z, float* loss) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (r >= m) return;
    loss[r] = targets[r] < 0 ? 0.0f : loss_of({state[r], state[m + r]}, state[2 * m + r], z);
}

// Gradient of a tile: the row's maximum and sum come from the state or from the records.  The loss, where
// it is asked for, is left by the tile that holds the target's logit (dx may be x: nobody else may read it).
template <typename S>
__global__ __launch_bounds__(kTileThreads) void grad_tiles(LossCall<S> p, int64_t record_count, const float* weights, S* dx, int64_t dx_stride) {
    constexpr int V = vector_width<S>();
    const uint32_t tiles = static_cast<uint32_t>(p.tiles.count);
    const uint32_t here = workgroup();
    const int64_t r = here / tiles, tile = here % tiles;
    if (r >= p.m) return;
    const S* xr = p.x + r * p.stride;
    S* dr = dx + r * dx_stride;
    const int64_t begin = tile * p.tiles.length;
    const int64_t end = begin + p.tiles.length < p.n ? begin + p.tiles.length : p.n;
    const int64_t target = p.targets[r];
    const float weight = weights ? weights[r] : 1.0f;
    MaxSum s;
    if (p.state) s = {p.state[r], p.state[p.m + r]};
    else s = join_records(p.records + r * record_count, record_count);
    const RowGrad g = row_grad(s, target >= 0, weight, p.z);
    const int64_t column = target < 0 ? -1 : target - p.first;
    if (p.loss) {
        const bool inside = column >= 0 && column < p.n;
        const bool mine = inside ? column >= begin && column < end : tile == 0;
        if (threadIdx.x == 0 && mine) {
            const float logit = inside ? static_cast<float>(xr[column]) : std::numeric_limits<float>::quiet_NaN();
            p.loss[r] = target < 0 ? 0.0f : loss_of(s, logit, p.z);
        }
        if (inside && mine) __syncthreads();
    }
    for (int64_t e0 = begin + static_cast<int64_t>(threadIdx.x) * V; e0 < end; e0 += kTileBatch * tile_unit<S>()) {
        Words4 raw[kTileBatch];
#pragma unroll
        for (int u = 0; u < kTileBatch; ++u) {
            const int64_t e = e0 + u * tile_unit<S>();
            if (e < end && !g.zero) raw[u] = load_part(xr, e, end);
        }
#pragma unroll
        for (int u = 0; u < kTileBatch; ++u) {
            const int64_t e = e0 + u * tile_unit<S>();
            if (e < end) store_part(dr, e, end, grad_vector<S>(e, raw[u], g, column));
        }
    }
}

bool index_ok(int index_dtype) { return index_dtype == DLFX_I32 || index_dtype == DLFX_I64; }

int check(int64_t m, int64_t n, const void* x, int64_t row_stride, const void* targets) {
    if (m <= 0 || n <= 0 || !x || !targets || row_stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    if (m > 0x7fffffffLL || n > 0x7fffffffLL) return DLFX_ERR_TOO_LARGE;
    return DLFX_OK;
}

// Tiles of a pass that joins (records of scratch: about 2048 workgroups, none under 8 KB) and of one
// that only writes gradients (16 KB each, whatever their number).
template <typename S>
Tiles joining_tiles(int64_t m, int64_t n) {
    constexpr int64_t unit = tile_unit<S>();
    int64_t count = ceil_div(2048, m);
    const int64_t most = ceil_div(n, 2 * unit);
    if (count > most) count = most;
    if (count < 1) count = 1;
    const int64_t length = ceil_div(ceil_div(n, count), unit) * unit;
    return {ceil_div(n, length), length};
}
template <typename S>
Tiles writing_tiles(int64_t n) {
    const int64_t length = kTileBatch * tile_unit<S>();
    return {ceil_div(n, length), length};
}

// Longest row that a workgroup's registers hold.
template <typename S> constexpr int64_t held_most() { return 16 * 1024 * vector_width<S>(); }

// Few rows of middling length are a workgroup's of sixteen wavefronts each, which spares the launch that joins
// tiles.  Calls in a row, us, tiles and rows: the loss of [64, 32768] fp32 14.1 / 11.2, [512, 32768] 18.1 / 16.4,
// [256, 65536] 18.0 / 14.2, beyond [1023, 32768] 25.9 / 29.4 and [64, 131072] 14.1 / 18.5; the loss with its
// gradient, [1 to 190, 32768] fp32 19.2 / 16.0, beyond [64, 65536] 18.6 / 21.6 (from about 190 rows on both fill
// the device: [190, 65536] 32.0 / 31.2).
constexpr int64_t kFewRows = 512, kLossBytes = 256 * 1024, kGradBytes = 128 * 1024, kHeldRows = 192;

// Records of the tiles; calls that make none ask for nothing.
template <typename S>
size_t scratch_of(int64_t m, int64_t n) {
    if (m <= kFewRows && n * static_cast<int64_t>(sizeof(S)) <= kGradBytes) return 0;
    const int64_t count = joining_tiles<S>(m, n).count;
    return count > 1 || n > held_most<S>() ? static_cast<size_t>(m * count) * sizeof(MaxSum) : 0;
}

template <int... I, typename F>
void for_each_of(std::integer_sequence<int, I...>, F&& f) { (f(std::integral_constant<int, I + 2>()), ...); }

// Workgroups of a kernel that the current device holds at once, asked for once per device.
template <auto KERNEL>
int64_t resident(int threads) {
    static std::atomic<int64_t> known[64];
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess || device < 0 || device >= 64) return resident_workgroups(KERNEL, threads);
    int64_t n = known[device].load(std::memory_order_relaxed);
    if (n == 0) known[device].store(n = resident_workgroups(KERNEL, threads), std::memory_order_relaxed);
    return n;
}

template <typename S>
int launch_loss(LossCall<S> p, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    p.tiles = joining_tiles<S>(p.m, p.n);
    if (p.tiles.count > 1 && (!scratch || scratch_bytes < scratch_of<S>(p.m, p.n))) p.tiles = {1, p.n};
    if (p.m * p.tiles.count > 0x7fffffffLL) return DLFX_ERR_TOO_LARGE;
    p.records = static_cast<MaxSum*>(scratch);
    if (p.m <= kFewRows && p.n * static_cast<int64_t>(sizeof(S)) <= kLossBytes) {
        p.tiles = {1, p.n};
        if (p.n > kTileBatch * tile_unit<S>()) {
            loss_tiles<S, 1024><<<grid_of(p.m), dim3(1024), 0, stream>>>(p);
            DLFX_CHECK_LAUNCH();
            return DLFX_OK;
        }
    }
    loss_tiles<S, kTileThreads><<<grid_of(p.m * p.tiles.count), dim3(kTileThreads), 0, stream>>>(p);
    DLFX_CHECK_LAUNCH();
    if (p.tiles.count > 1) {
        loss_join_tiles<S><<<dim3(static_cast<unsigned>(ceil_div(p.m, 4))), dim3(256), 0, stream>>>(p);
        DLFX_CHECK_LAUNCH();
    }
    return DLFX_OK;
}

template <typename S>
int launch_grad_tiles(LossCall<S> p, int64_t record_count, const float* weights, S* dx, int64_t dx_stride, hipStream_t stream) {
    p.tiles = writing_tiles<S>(p.n);
    if (p.m * p.tiles.count > 0x7fffffffLL) return DLFX_ERR_TOO_LARGE;
    grad_tiles<S><<<grid_of(p.m * p.tiles.count), dim3(kTileThreads), 0, stream>>>(p, record_count, weights, dx, dx_stride);
    DLFX_CHECK_LAUNCH();
    return DLFX_OK;
}

template <typename S>
int launch_grad(LossCall<S> p, const float* weights, S* dx, int64_t dx_stride, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    auto held = [&](auto vectors, auto team) {
        constexpr int NV = decltype(vectors)::value, T = decltype(team)::value;
        // as many workgroups as the device holds: each goes on to its next row while it stores the last
        const int64_t most = resident<grad_rows_held<S, NV, T>>(T);
        const int64_t blocks = most > 0 && most < p.m ? most : p.m;
        grad_rows_held<S, NV, T><<<dim3(static_cast<unsigned>(blocks)), dim3(T), 0, stream>>>(p.x, p.m, p.n, p.stride, p.targets, weights, p.z, p.loss,
                                                                                              dx, dx_stride);
        DLFX_CHECK_LAUNCH();
        return static_cast<int>(DLFX_OK);
    };
    using std::integral_constant;
    constexpr int64_t V = vector_width<S>();
    const size_t need = scratch_of<S>(p.m, p.n);
    const bool has_scratch = need && scratch && scratch_bytes >= need;
    if (p.n < V) {
        grad_rows_tiny<S><<<dim3(static_cast<unsigned>(ceil_div(p.m, 256))), dim3(256), 0, stream>>>(p.x, p.m, static_cast<int>(p.n), p.stride, p.targets,
                                                                                                     weights, p.z, p.loss, dx, dx_stride);
        DLFX_CHECK_LAUNCH();
        return DLFX_OK;
    }
    if (p.n <= 256 * V) return held(integral_constant<int, 1>(), integral_constant<int, 256>());
    if (p.n <= 512 * V) return held(integral_constant<int, 2>(), integral_constant<int, 256>());
    if (p.n <= 768 * V) return held(integral_constant<int, 3>(), integral_constant<int, 256>());
    if (p.n <= 1024 * V) return held(integral_constant<int, 4>(), integral_constant<int, 256>());
    if (p.n <= held_most<S>() && (p.n * static_cast<int64_t>(sizeof(S)) <= kGradBytes || p.m >= kHeldRows || !has_scratch)) {
        int status = DLFX_OK;
        const int64_t vectors = ceil_div(p.n, 1024 * V);
        auto one = [&](auto c) {
            if (vectors == decltype(c)::value) status = held(c, integral_constant<int, 1024>());
        };
        for_each_of(std::make_integer_sequence<int, 15>(), one);      // 2 to 16
        return status;
    }
    if (!has_scratch) return DLFX_ERR_SCRATCH_TOO_SMALL;
    // the records first, then the gradients and the loss tile by tile
    LossCall<S> q = p;
    q.tiles = joining_tiles<S>(p.m, p.n);
    if (p.m * q.tiles.count > 0x7fffffffLL) return DLFX_ERR_TOO_LARGE;
    q.records = static_cast<MaxSum*>(scratch);
    float* loss = q.loss;
    q.loss = nullptr;                       // (records)
    loss_tiles<S, kTileThreads><<<grid_of(p.m * q.tiles.count), dim3(kTileThreads), 0, stream>>>(q);
    DLFX_CHECK_LAUNCH();
    q.loss = loss;
    return launch_grad_tiles(q, q.tiles.count, weights, dx, dx_stride, stream);
}

}  // namespace
}  // namespace dlfx

using namespace dlfx;

extern "C" size_t dlfx_cross_entropy_scratch_bytes(int dtype, int64_t m, int64_t n) {
    if (m <= 0 || n <= 0 || m > 0x7fffffffLL || n > 0x7fffffffLL) return 0;
    switch (dtype) {
    case DLFX_F32: return scratch_of<float>(m, n);
    case DLFX_F16: return scratch_of<half_t>(m, n);
    case DLFX_BF16: return scratch_of<bf16_t>(m, n);
    default: return 0;
    }
}

extern "C" int dlfx_cross_entropy(dlfx_stream_t stream, int dtype, int index_dtype, int64_t m, int64_t n,
                                  const void* x, int64_t x_offset, int64_t row_stride, const void* targets,
                                  float z_loss, float* loss, void* scratch, size_t scratch_bytes) {
    if (int e = check(m, n, x, row_stride, targets)) return e;
    if (!loss) return DLFX_ERR_INVALID_ARGUMENT;
    if (!index_ok(index_dtype)) return DLFX_ERR_UNSUPPORTED_DTYPE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        LossCall<S> p{static_cast<const S*>(x) + x_offset, m, n, row_stride, Targets{targets, index_dtype == DLFX_I64}, 0, 0, nullptr, z_loss, loss, {}, nullptr};
        return launch_loss(p, scratch, scratch_bytes, s);
    });
}

extern "C" int dlfx_cross_entropy_grad(dlfx_stream_t stream, int dtype, int index_dtype, int64_t m, int64_t n,
                                       const void* x, int64_t x_offset, int64_t row_stride, const void* targets,
                                       const float* weights, float z_loss, float* loss,
                                       void* dx, int64_t dx_offset, int64_t dx_row_stride,
                                       void* scratch, size_t scratch_bytes) {
    if (int e = check(m, n, x, row_stride, targets)) return e;
    if (!dx || dx_row_stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    if (!index_ok(index_dtype)) return DLFX_ERR_UNSUPPORTED_DTYPE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        LossCall<S> p{static_cast<const S*>(x) + x_offset, m, n, row_stride, Targets{targets, index_dtype == DLFX_I64}, 0, 0, nullptr, z_loss, loss, {}, nullptr};
        if (overwrites(p.x, row_stride, static_cast<const S*>(dx) + dx_offset, dx_row_stride, m)) return static_cast<int>(DLFX_ERR_INVALID_ARGUMENT);
        return launch_grad(p, weights, static_cast<S*>(dx) + dx_offset, dx_row_stride, scratch, scratch_bytes, s);
    });
}

extern "C" int dlfx_cross_entropy_piece(dlfx_stream_t stream, int dtype, int index_dtype, int64_t m, int64_t n,
                                        const void* x, int64_t x_offset, int64_t row_stride, const void* targets,
                                        int64_t first, int resume, float* state, void* scratch, size_t scratch_bytes) {
    if (int e = check(m, n, x, row_stride, targets)) return e;
    if (!state || first < 0) return DLFX_ERR_INVALID_ARGUMENT;
    if (!index_ok(index_dtype)) return DLFX_ERR_UNSUPPORTED_DTYPE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        LossCall<S> p{static_cast<const S*>(x) + x_offset, m, n, row_stride, Targets{targets, index_dtype == DLFX_I64}, first, resume, state, 0.0f, nullptr, {}, nullptr};
        return launch_loss(p, scratch, scratch_bytes, s);
    });
}

extern "C" int dlfx_cross_entropy_join(dlfx_stream_t stream, int index_dtype, int64_t m, const void* targets,
                                       const float* state, float z_loss, float* loss) {
    if (m <= 0 || !targets || !state || !loss) return DLFX_ERR_INVALID_ARGUMENT;
    if (m > 0x7fffffffLL) return DLFX_ERR_TOO_LARGE;
    if (!index_ok(index_dtype)) return DLFX_ERR_UNSUPPORTED_DTYPE;
    loss_join<<<dim3(static_cast<unsigned>(ceil_div(m, 256))), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
        m, Targets{targets, index_dtype == DLFX_I64}, state, z_loss, loss);
    DLFX_CHECK_LAUNCH();
    return DLFX_OK;
}

extern "C" int dlfx_cross_entropy_piece_grad(dlfx_stream_t stream, int dtype, int index_dtype, int64_t m, int64_t n,
                                             const void* x, int64_t x_offset, int64_t row_stride, const void* targets,
                                             int64_t first, const float* state, const float* weights, float z_loss,
                                             void* dx, int64_t dx_offset, int64_t dx_row_stride) {
    if (int e = check(m, n, x, row_stride, targets)) return e;
    if (!state || first < 0 || !dx || dx_row_stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    if (!index_ok(index_dtype)) return DLFX_ERR_UNSUPPORTED_DTYPE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        LossCall<S> p{static_cast<const S*>(x) + x_offset, m, n, row_stride, Targets{targets, index_dtype == DLFX_I64}, first, 0, const_cast<float*>(state), z_loss,
                         nullptr, {}, nullptr};
        if (overwrites(p.x, row_stride, static_cast<const S*>(dx) + dx_offset, dx_row_stride, m)) return static_cast<int>(DLFX_ERR_INVALID_ARGUMENT);
        return launch_grad_tiles(p, 0, weights, static_cast<S*>(dx) + dx_offset, dx_row_stride, s);
    });
}
