// What the forward and backward gated_scan kernels share: gate functions, the walk over a call's
// tensors, how a call's axis is cut.
#pragma once

#include <cstring>

#include "sequence.hip.h"

namespace dlfx {
namespace {

enum GateKind { kGated = 0, kGatedExp = 1, kGatedSigmoid = 2, kGatedBlend = 3 };

// A tensor of the call: row r starts at base + row.at(r), step t is t * step elements further on.
template <typename S>
struct Track {
    S* base;
    int64_t step;
    DimMap row;
};

// Factor a of the state, and 1 - a (blend: the factor of x; sigmoid and blend: a' = a (1 - a)).
// The logistic function from e = exp(-|g|) <= 1: the larger of a and 1 - a is 1 / (1 + e), the
// smaller e / (1 + e), so neither is a difference of nearby numbers and g = +-inf gives 1 and 0.
template <typename S, int KIND>
__device__ __forceinline__ void gate_of(float g, float& a, float& keep) {
    if constexpr (KIND == kGated) {
        a = g;
    } else if constexpr (KIND == kGatedExp) {
        a = fast_exp<S>(g);
    } else {
        const float e = fast_exp<S>(-fabsf(g));
        const float r = fast_reciprocal<S>(1.0f + e);
        const float small = e * r;
        a = g < 0.0f ? small : r;
        keep = g < 0.0f ? r : small;
    }
}

// The gate that leaves a state as it is when x is 0 (a = 1).
template <typename S, int KIND>
__device__ __forceinline__ S neutral_gate() {
    if constexpr (KIND == kGated) return static_cast<S>(1.0f);
    else if constexpr (KIND == kGatedExp) return static_cast<S>(0.0f);
    else return static_cast<S>(std::numeric_limits<float>::infinity());
}

// What a stretch of steps does to the state that enters it: h -> a h + b.  The product of many
// gates can leave the range of fp32 where the states do not (growth from a tiny state, decay of a
// large one), so it is held in 64 bits; it is finite unless a gate is not (times()).
struct Stretch {
    double a;
    float b;
};
__device__ __forceinline__ float through(const Stretch& s, float h) {
    return static_cast<float>(s.a * static_cast<double>(h) + static_cast<double>(s.b));
}

// Products that pass fp64 as well, from there on the largest number: growth that no state but 0 survives.  A gate of 0
// behind them or before still makes 0, which an infinity would not.
constexpr double kFar = 0x1p1000;
__device__ __forceinline__ bool in_range(double a) { return fabs(a) < kFar; }
__device__ __forceinline__ double times(double a, double b) {
    const double p = a * b;
    if (a == 0.0 || b == 0.0 || !(fabs(a) <= std::numeric_limits<double>::max()) || !(fabs(b) <= std::numeric_limits<double>::max())) return p;
    return in_range(a) && in_range(b) && in_range(p) ? p : copysign(std::numeric_limits<double>::max(), p);
}
__device__ __forceinline__ Stretch join(const Stretch& first, const Stretch& then) { return {times(first.a, then.a), through(then, first.b)}; }

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= std::numeric_limits<float>::max(); }

// The product of a lane's gates, in 64 bits where fp32 did not hold it.
template <int N>
__device__ __forceinline__ double product_of(float in_fp32, const float (&a)[N]) {
    double p = a[0];
#pragma unroll
    for (int i = 1; i < N; ++i) p = times(p, static_cast<double>(a[i]));
    return finite(in_fp32) ? static_cast<double>(in_fp32) : p;
}

// V neighbouring elements at base + off bytes.  The base is the same for the whole wavefront and the
// offset a lane's own: with 32 bits of it an access takes both as they are, without address arithmetic.
// NT: with the non-temporal hint, for tensors whose pieces are whole cache lines (5 to 7 % on bf16
// [8, 4096, 2048]); where neighbouring workgroups share lines it costs a third (bf16 [64, 4096, 500]:
// 225 us without, 310 us with it).
template <bool NT, typename S, int V, typename OFF>
__device__ __forceinline__ Vec<S, V> load_at(const S* base, OFF off) {
    const char* at = reinterpret_cast<const char*>(base) + off;
    if constexpr (!NT) {
        return *reinterpret_cast<const Vec<S, V>*>(at);
    } else if constexpr (sizeof(S) * V == 2) {
        return {{bit_cast<S>(__builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(at)))}};
    } else {
        constexpr int WORDS = sizeof(S) * V / 4;
        return bit_cast<Vec<S, V>>(load_stream(reinterpret_cast<const Vec<uint32_t, WORDS>*>(at)));
    }
}
template <bool NT, typename S, int V, typename OFF>
__device__ __forceinline__ void store_at(S* base, OFF off, const Vec<S, V>& v) {
    char* at = reinterpret_cast<char*>(base) + off;
    if constexpr (!NT) {
        *reinterpret_cast<Vec<S, V>*>(at) = v;
    } else if constexpr (sizeof(S) * V == 2) {
        __builtin_nontemporal_store(bit_cast<uint16_t>(v.v[0]), reinterpret_cast<uint16_t*>(at));
    } else {
        constexpr int WORDS = sizeof(S) * V / 4;
        store_stream(reinterpret_cast<Vec<uint32_t, WORDS>*>(at), bit_cast<Vec<uint32_t, WORDS>>(v));
    }
}

// Keeps the compiler from adding a loop's changing base to the lane's offset beforehand.
template <typename OFF>
__device__ __forceinline__ OFF as_it_is(OFF off) {
    if constexpr (sizeof(OFF) == 4) asm volatile("" : "+v"(off));
    return off;
}

// A wavefront takes 64 groups of V neighbouring rows and S consecutive steps of a pass, W wavefronts
// share a pass of W * S steps, and a segment of the axis is walked pass by pass.
struct Cut {
    int64_t m, n;
    int64_t blocks;              // groups of 64 V rows
    int64_t segments, length;    // of the axis; length steps each, the last one shorter
};

constexpr int kColumnSegments = 64, kRowSegments = 512;      // the most

// How rows side by side are walked.  All times: us, forward / backward.
// A lane per row and nothing else up to four steps (decoding: one).
constexpr int64_t kWalked = 4;
// Pairs of two-byte rows to a lane and a workgroup of one wavefront once there are four wavefronts for
// every CU, against 16 wavefronts over one group of 64 rows: bf16 [1024, 131072] 152 / 251 against 157 / 262,
// [1000, 262144] 303 / 518 against 353 / 564; with fewer, [1024, 65536] 116 against 80.
constexpr int64_t kManyPairs = 131072;
// Wavefronts of a workgroup: more of them put more steps in flight, but a pass (16 or 8 steps each) that is
// longer than the axis leaves some idle.  2, 4, 8 and 16 of them, bf16 rows 262144: n = 48 20 23 42 80 / 33 34 45 77,
// n = 128 41 40 43 86 / 77 74 78 91, n = 200 67 70 76 95 / 118 116 128 146, n = 300 106 104 113 159 / 175 173 171 213;
// 16384 rows: n = 200 13.9 11.0 9.5 8.5, n = 300 17.7 12.7 12.5 12.0 / 27.7 20.3 19.1 19.1, n = 1000 48 31 26 24 / 75 49 41 40.
inline int waves_of(int64_t m, int64_t n) {
    if (n <= 64) return 2;
    if (n <= 128 || m >= 131072) return 4;
    return n <= 256 ? 8 : 16;
}
// Only 16 wavefronts over single rows are cut into segments: shorter axes are a pass or two, pairs are many.
template <int V, int W>
constexpr bool cut_columns() { return V == 1 && W == 16; }

// Workgroups go round the eight XCDs in turn, each with a cache of its own: neighbouring pieces of work
// (groups of rows that share cache lines where a row of columns is no whole number of them) go to one
// XCD side by side.  The grid is rounded up to a multiple of 8.
__device__ __forceinline__ int64_t work_of(uint32_t block, uint32_t grid) { return static_cast<int64_t>(block % 8) * (grid / 8) + block / 8; }
inline int64_t grid_of(int64_t work) { return ceil_div(work, 8) * 8; }

// ---- rows along memory: a lane takes kRun consecutive positions of its row in two 128-bit accesses
template <typename S>
constexpr int run_length() { return 32 / static_cast<int>(sizeof(S)); }

// Positions i0 .. i0 + N - 1 of a row that goes up (DIR 1) or down (DIR -1) in memory from `row`; what
// lies at or past `end` is left as it is.  WHOLE: nothing does, for any lane.
template <bool WHOLE, int DIR, typename S, int N>
__device__ __forceinline__ void load_run(const S* row, int64_t i0, int64_t end, S (&out)[N]) {
    constexpr int V = 16 / static_cast<int>(sizeof(S));
    using VecT = typename AnyVec<S, V>::type;
    if (WHOLE || i0 + N <= end) {
        const S* at = DIR > 0 ? row + i0 : row - i0 - (N - 1);
#pragma unroll
        for (int k = 0; k < N; k += V) {
            const VecT v = *reinterpret_cast<const VecT*>(at + k);
#pragma unroll
            for (int e = 0; e < V; ++e) out[DIR > 0 ? k + e : N - 1 - k - e] = v[e];
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (i0 + k < end) out[k] = row[DIR * (i0 + k)];
    }
}
template <bool WHOLE, int DIR, typename S, int N>
__device__ __forceinline__ void store_run(S* row, int64_t i0, int64_t end, const S (&in)[N]) {
    constexpr int V = 16 / static_cast<int>(sizeof(S));
    using VecT = typename AnyVec<S, V>::type;
    if (WHOLE || i0 + N <= end) {
        S* at = DIR > 0 ? row + i0 : row - i0 - (N - 1);
#pragma unroll
        for (int k = 0; k < N; k += V) {
            VecT v;
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = in[DIR > 0 ? k + e : N - 1 - k - e];
            *reinterpret_cast<VecT*>(at + k) = v;
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (i0 + k < end) row[DIR * (i0 + k)] = in[k];
    }
}

// The stretches of a group of G lanes (4, 16, 32 or 64, in order) joined from the group's first lane up
// to each; `before` is what lies before the lane, `all` the whole group's.  again(): the lane's product in 64 bits,
// where fp32 did not hold it.
template <int G, typename Again>
__device__ __forceinline__ void join_lanes(const Stretch& own, Stretch& before, Stretch& all, Again&& again) {
    const int lane = lane_id();
    Stretch s = own;
    auto step = [&](double pa, float pb, bool mine) {
        if (!mine) pa = 1.0, pb = 0.0f;
        s.b = through(s, pb);
        s.a *= pa;
    };
    // (a row shift reaches over a group of four: what comes from the group before is dropped)
    step(dpp_fetch<kRowShr1>(s.a, 1.0), dpp_fetch<kRowShr1>(s.b, 0.0f), G >= 16 || lane % G >= 1);
    step(dpp_fetch<kRowShr2>(s.a, 1.0), dpp_fetch<kRowShr2>(s.b, 0.0f), G >= 16 || lane % G >= 2);
    if constexpr (G >= 16) {
        step(dpp_fetch<kRowShr4>(s.a, 1.0), dpp_fetch<kRowShr4>(s.b, 0.0f), true);
        step(dpp_fetch<kRowShr8>(s.a, 1.0), dpp_fetch<kRowShr8>(s.b, 0.0f), true);
    }
    if constexpr (G >= 32) step(dpp_fetch<kRowBcast15, 0xa>(s.a, 1.0), dpp_fetch<kRowBcast15, 0xa>(s.b, 0.0f), true);
    if constexpr (G >= 64) step(dpp_fetch<kRowBcast31, 0xc>(s.a, 1.0), dpp_fetch<kRowBcast31, 0xc>(s.b, 0.0f), true);
    // a product that passed the range left its mark on all lanes behind it: an infinity, or the NaN that it and a 0
    // make; one that passed fp32 in a lane's own steps is marked so already.  Groups of lanes with such a mark once
    // more, by products that stay in range.
    if (const uint64_t far = __ballot(!in_range(s.a))) {
        Stretch f = {again(), own.b};
#pragma unroll 1
        for (int d = 1; d < G; d <<= 1) {
            const Stretch first = {lane_get(f.a, (lane - d) & (kWave - 1)), lane_get(f.b, (lane - d) & (kWave - 1))};
            if (lane % G >= d) f = join(first, f);
        }
        if (G == kWave || (far >> (lane & ~(G - 1)) & ((1ull << (G & (kWave - 1))) - 1))) s = f;
    }
    before.a = lane_get(s.a, (lane + kWave - 1) % kWave);
    before.b = lane_get(s.b, (lane + kWave - 1) % kWave);
    if (lane % G == 0) before = {1.0, 0.0f};
    if constexpr (G == kWave) all = {lane_read(s.a, kWave - 1), lane_read(s.b, kWave - 1)};
    else all = {lane_get(s.a, lane | (G - 1)), lane_get(s.b, lane | (G - 1))};
}

// The state that enters segment `count` of row r, by a whole wavefront: a lane joins neighbouring records.
__device__ __forceinline__ float enter_segment(const Stretch* records, int64_t m, int64_t r, int64_t count, float state) {
    const int per = static_cast<int>((count + kWave - 1) / kWave);
    Stretch mine = {1.0, 0.0f};
    for (int i = 0; i < per; ++i) {
        const int64_t s = static_cast<int64_t>(lane_id()) * per + i;
        if (s < count) mine = join(mine, records[s * m + r]);
    }
    Stretch before, all;
    join_lanes<kWave>(mine, before, all, [&] { return mine.a; });
    return through(all, state);
}

// The same for columns, by a workgroup of W wavefronts: each reads its share of the column's records at
// once and joins them, the shares meet in LDS.  (One record after the other, by every wavefront:
// 158.7 us against 149.1 for the second launch of fp32 [1, 65536, 1000].)
template <int W>
__device__ __forceinline__ float enter_column(const Stretch* records, int64_t m, int64_t r, int64_t count, float state, Stretch (*lds)[kWave]) {
    constexpr int PER = kColumnSegments / W;
    const int wave = threadIdx.x / kWave, lane = lane_id();
    Stretch got[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        got[i] = {1.0, 0.0f};
        if (wave * PER + i < count) got[i] = records[(wave * PER + i) * m + r];
    }
#pragma unroll
    for (int i = 1; i < PER; ++i) got[0] = join(got[0], got[i]);
    lds[wave][lane] = got[0];
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) state = through(lds[w][lane], state);
    return state;
}

// Every wavefront of the workgroup goes on from the same bits, those of the first one, even if a caller's error lets
// something write to them meanwhile: whether repair_pass waits at barriers must never differ between wavefronts.
template <int V, int W>
__device__ __forceinline__ void share_carry(float (&carry)[V], int wave, int lane) {
    if constexpr (W > 1) {
        __shared__ float start[kWave][V];
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (wave == 0) start[lane][v] = carry[v];
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) carry[v] = start[lane][v];
    }
}

// After a pass of rows side by side that turned a finite state into an infinite one or NaN: in truth, or because a
// wavefront's gates multiplied past fp32 before they met the state.  Such rows go through the pass again, wavefront
// after wavefront and step after step.  All wavefronts hold the same `entering` and `state` (share_carry, then the
// records in LDS), so all of them come here or none.  first: the state that entered the wavefront's steps; again(h)
// walks them from h and stores what they give.  `lds` is the half that the next pass is going to use.  (Here, behind
// the pass's stores: between them and the join it cost the gradient 4 % of its time.)
template <int V, int W, typename Again>
__device__ __forceinline__ void repair_pass(float (*lds)[kWave][2 * V], int wave, int lane, const float (&entering)[V], float (&state)[V],
                                            const float (&first)[V], Again&& again) {
    bool lost = false;
#pragma unroll
    for (int v = 0; v < V; ++v) lost = lost || !finite(state[v]);
    if (__builtin_expect(!__any(lost), 1)) return;
    lost = false;
#pragma unroll
    for (int v = 0; v < V; ++v) lost = lost || (finite(entering[v]) && !finite(state[v]));
    if (!__any(lost)) return;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = entering[v];
#pragma unroll 1
    for (int w = 0; w < W; ++w) {
        if (w == wave) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (!finite(entering[v]) || finite(state[v])) h[v] = first[v];          // (a neighbour's results stay what they are)
            if (lost) again(h);
#pragma unroll
            for (int v = 0; v < V; ++v) lds[w][lane][2 * v] = h[v];
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = lds[w][lane][2 * v];
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (finite(entering[v]) && !finite(state[v])) state[v] = h[v];
}

// +1 or -1 when a track's steps lie one element apart in memory, 0 otherwise.
template <typename S>
int direction(const Track<S>& t) { return t.step == 1 ? 1 : t.step == -1 ? -1 : 0; }

// How many segments: one while the groups of rows alone are enough, otherwise about `wanted` workgroups in
// all, none shorter than `shortest` steps.  A cut axis is read nearly twice.
inline int64_t segments_of(int64_t groups, int64_t n, int64_t shortest, int64_t enough, int64_t wanted, int64_t limit) {
    if (groups >= enough) return 1;
    int64_t s = ceil_div(wanted, groups);
    if (s > limit) s = limit;
    const int64_t most = n / shortest;
    return s < most ? s : (most < 1 ? 1 : most);
}
// us, whole and cut: columns bf16 [8192, 4096] 119 / 76, [8192, 8192] 128 / 139, fp32 [8192, 8192] 182 / 238.  256, 512
// and 1024 workgroups wanted: bf16 [8192, 4096] 71 76 85, [65536, 1024] 133 142 149, fp32 [65536, 1000] 278 268 274.
template <typename S>
int64_t column_segments(int64_t groups, int64_t n, int64_t shortest) {
    return segments_of(groups, n, shortest, 128, sizeof(S) == 2 ? 256 : 512, kColumnSegments);
}
// Rows of 131072 bf16, whole and cut: 64 of them 30 / 28, 128 of them 32 / 46.
inline int64_t row_segments(int64_t groups, int64_t n, int64_t shortest) { return segments_of(groups, n, shortest, 64, 512, kRowSegments); }

// Scratch of a cut call: what every segment but the last does to the state, and a copy of the
// states that enter the axis (the tensor they come from may be the one that `last` is written to).
inline size_t records_bytes(int64_t m, int64_t segments) {
    return segments > 1 ? align_up(static_cast<size_t>(m * (segments - 1)) * sizeof(Stretch), 256) + static_cast<size_t>(m) * sizeof(float) : 0;
}

// Byte offsets of the rows fit 32 bits and none is negative: a row's offset rides in one register
// beside a scalar base.
template <typename S>
bool short_offsets(const Track<S>& t) {
    if (!t.base) return true;
    unsigned __int128 span = 0;
    for (int i = 0; i < t.row.rank; ++i) {
        if (t.row.strides[i] < 0) return false;
        span += static_cast<unsigned __int128>(t.row.dims[i] - 1) * static_cast<uint64_t>(t.row.strides[i]);
    }
    return span * sizeof(S) < (static_cast<unsigned __int128>(1) << 32) - 64;
}
// Rows 2 i and 2 i + 1 lie side by side on a boundary of their own size at every step.
template <typename S>
bool pairs_of_rows(const Track<S>& t) {
    if (!t.base) return true;
    const int r = t.row.rank;
    if (r == 0 || t.row.strides[r - 1] != 1 || t.row.dims[r - 1] % 2 || t.step % 2) return false;
    for (int i = 0; i + 1 < r; ++i)
        if (t.row.strides[i] % 2) return false;
    return reinterpret_cast<uintptr_t>(t.base) % (2 * sizeof(S)) == 0;
}
// Every 64 neighbouring rows are whole 128-byte cache lines at every step.
template <typename S>
bool whole_lines(const Track<S>& t) {
    if (!t.base) return true;
    const int64_t line = 128 / static_cast<int64_t>(sizeof(S));
    const int r = t.row.rank;
    if (r == 0 || t.row.strides[r - 1] != 1 || t.row.dims[r - 1] % line || t.step % line) return false;
    for (int i = 0; i + 1 < r; ++i)
        if (t.row.strides[i] % line) return false;
    return reinterpret_cast<uintptr_t>(t.base) % 128 == 0;
}

template <typename S>
bool make_track(int rank, const int64_t* dims, const void* base, int64_t offset, const int64_t* strides, bool per_row, Track<S>* out) {
    using E = typename std::remove_const<S>::type;
    out->base = nullptr;
    out->step = 0;
    out->row = DimMap{};
    if (!base) return true;
    out->base = const_cast<E*>(static_cast<const E*>(base)) + offset;
    if (!per_row) out->step = strides[rank - 1];
    return make_dim_map(dims, strides, 0, rank - 1, &out->row);
}

inline int kind_of(const char* name) {
    if (!std::strcmp(name, "gated")) return kGated;
    if (!std::strcmp(name, "gated_exp")) return kGatedExp;
    if (!std::strcmp(name, "gated_sigmoid")) return kGatedSigmoid;
    if (!std::strcmp(name, "gated_blend")) return kGatedBlend;
    return -1;
}

template <typename F>
int dispatch_kind(int kind, F&& f) {
    switch (kind) {
    case kGated: return f(std::integral_constant<int, kGated>());
    case kGatedExp: return f(std::integral_constant<int, kGatedExp>());
    case kGatedSigmoid: return f(std::integral_constant<int, kGatedSigmoid>());
    default: return f(std::integral_constant<int, kGatedBlend>());
    }
}

inline bool shape_ok(int64_t m, int64_t n, int rank, const int64_t* dims, const int64_t* some_strides) {
    if (m <= 0 || n <= 0 || rank < 1) return false;
    if (!view_ok(rank, dims, some_strides)) return false;
    return dims[rank - 1] == n && view_size(rank - 1, dims) == m;
}

}  // namespace
}  // namespace dlfx
