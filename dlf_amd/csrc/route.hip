// Routing to experts: scores of a row of router logits, the k largest choices among the kept
// groups, their weights; and the gradient of the logits.
//
// A row belongs to a team of L lanes (16 up to 256 experts, else a wavefront): expert i * L + lane is
// the lane's item i, so that any run of neighbouring experts spreads over all lanes.  Nothing leaves
// the wavefront: no barrier, no scratch.  The work per row is a few hundred vector instructions on a
// kilobyte of logits, so arithmetic bounds it, and the choice is what the time goes to:
//   * choices in fp32.  A bound from the lanes' largest items (the (k+1)-th largest of them) leaves
//     little more than k candidates; those are gathered through LDS, one or two to a lane, and
//     ordered by a bitonic network of (choice, index) words.
//   * where fp32 cannot tell two neighbours of the result apart (a gap under their errors, one row in
//     hundreds with random scores), the row is marked and a second launch does it over in 64 bits,
//     picking one expert after the other.
// Without a bias the logits order the experts exactly, and only sums of two scores can need 64 bits:
// other calls are one launch.
// fp32 [32768, 256] sigmoid, bias, the best 4 of 8 groups, k = 8: 30.6 us (VALU 86 % busy) + 10.3 (the latency of a
// few rows in 64 bits); bf16 [65537, 128] softmax, k = 8: 22.2 us (VALU 90 %); [24, 64]: 3.7 us.
// k = 64 with a bias marks every row: [32768, 256] takes 695 us a call, 394 with k = 63.
#include <cmath>
#include <cstring>

#include "sequence.hip.h"

namespace dlfx {
namespace {

enum ScoreKind { kSoftmaxScore = 0, kSigmoidScore = 1 };

template <typename S> __device__ __forceinline__ float lowest_of();
template <> __device__ __forceinline__ float lowest_of<float>() { return -3.40282346638528859812e38f; }
template <> __device__ __forceinline__ float lowest_of<half_t>() { return -65504.0f; }
template <> __device__ __forceinline__ float lowest_of<bf16_t>() { return -3.38953138925153547590e38f; }

constexpr float kMinusInfinity = -std::numeric_limits<float>::infinity();

// Choices are compared as unsigned images that keep the order of the numbers: an expert outside the
// kept groups is 0, an absent one (or a NaN) 1, every number above that.
__device__ __forceinline__ uint32_t image_of(float v) {
    if (v != v) return 1;
    const uint32_t u = bit_cast<uint32_t>(v + 0.0f);          // -0.0 and +0.0 are one value
    return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t image_of(double v) {
    if (v != v) return 1;
    const uint64_t u = bit_cast<uint64_t>(v + 0.0);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ float value_of(uint32_t image) { return bit_cast<float>((image >> 31) ? image & 0x7fffffffu : ~image); }

template <typename C> struct ImageOf;
template <> struct ImageOf<float> { using type = uint32_t; };
template <> struct ImageOf<double> { using type = uint64_t; };

template <int L, typename T, typename Join>
__device__ __forceinline__ T team_reduce(T v, Join join) {
    return group_reduce(v, L, join);
}

// Orders the LDS accesses of a wavefront: what its lanes have written is there for all of them.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

struct RouteCall {
    int64_t m, stride;
    int n, groups, kept_groups, group_best, size, size_magic, k, renormalise;      // e / size == (e * size_magic) >> 20
    float scale;
    const float* bias;
    float* weights;
    int32_t* indices;
    int32_t* loads;
};

// How far apart two fp32 choices a and b have to be to be told apart: both errors together, with
// u = 2^-24.  `scores` is the scores' part: the logistic function is off by under 1 u from its
// exponential (1.5 |x| + 2 u of it, times s (1 - s)) and a rounding each in its sum, quotient and
// product, 4 u in all, 16 u is taken; a softmax score by under 28 u of itself (terms (1.5 d + 2) u at a
// distance d below the maximum, up to 22 roundings of the sum, two more), and no score is larger than
// the row's 1 / sum: 64 u of that is taken.  The sum with the bias rounds once: 2 u, 4 u taken.
__device__ __forceinline__ float border(float scores, float a, float b) { return scores + 0x1p-22f * fmaxf(fabsf(a), fabsf(b)); }

// LDS of a team: the items' values and the groups', or the candidates, then a byte per group.  (8 of 32
// doubles left over: the teams of a wavefront start 16 banks apart.)
template <int L, int ITEMS>
constexpr int team_doubles() { return L * ITEMS + L * ITEMS / 8 + (40 - (L * ITEMS + L * ITEMS / 8) % 32) % 32; }

// The two largest of a group's values and how many there are.
template <typename C>
struct Best {
    C first, second;
    int count;
    __device__ __forceinline__ void add(C v) {
        if (v != v) return;
        ++count;
        second = v > first ? first : (v > second ? v : second);
        first = v > first ? v : first;
    }
    __device__ __forceinline__ void add(const Best& o) {
        count += o.count;
        const C low = o.first > first ? first : o.first;
        second = o.second > second ? o.second : second;
        second = low > second ? low : second;
        first = o.first > first ? o.first : first;
    }
    __device__ __forceinline__ C value(int best) const {
        if (count == 0) return std::numeric_limits<C>::quiet_NaN();
        return best == 2 && count > 1 ? first + second : first;
    }
};

// Values of the groups in sums[] from their experts' in items[] (NaN: absent), by a team of L lanes.  Returns the
// largest magnitude among the lane's experts.
template <int L, typename C>
__device__ __forceinline__ C group_values(const RouteCall& p, const C* items, C* sums, int lane) {
    const C none = -std::numeric_limits<C>::infinity();
    // lanes_per lanes (a power of two) to a group; a lane walks its part of the group's experts from a
    // place of its own, so that the lanes read different LDS banks
    int lanes_per = L;
    while (lanes_per > 1 && lanes_per * p.groups > L) lanes_per >>= 1;
    const int part = lane & (lanes_per - 1), side_by_side = L / lanes_per;
    C largest = 0;
    for (int g0 = 0; g0 < p.groups; g0 += side_by_side) {
        const int g = g0 + lane / lanes_per;
        Best<C> best = {none, none, 0};
        if (g < p.groups) {
            const int from = g - p.size * ((g * p.size_magic) >> 20);
            for (int i = part; i < p.size; i += lanes_per) {
                int e = i + from;
                e -= e >= p.size ? p.size : 0;
                const C v = items[g * p.size + e];
                best.add(v);
                largest = std::fmax(largest, std::fabs(v));          // (of a NaN and a number: the number)
            }
        }
        for (int j = 1; j < lanes_per; j <<= 1) best.add({lane_xor(best.first, j), lane_xor(best.second, j), lane_xor(best.count, j)});
        if (g < p.groups && part == 0) sums[g] = best.value(p.group_best);
    }
    wave_sync();
    return largest;
}

// Which groups are kept, a byte each.  `unsure` when the values are not exact and a kept group's lies too
// close to one that was left; `largest`: of the |choices| that the lane has seen.
template <int L, typename C>
__device__ __forceinline__ void keep_groups(const RouteCall& p, const C* sums, uint8_t* kept, bool exact, float scores, float largest, int lane,
                                            bool& unsure) {
    const C none = -std::numeric_limits<C>::infinity();
    C worst_kept = -none, best_left = none;
    for (int g = lane; g < p.groups; g += L) {
        // a group's rank: how many come before it (larger value, or equal and lower)
        const C v = sums[g];
        const auto mine = image_of(v);
        int rank = 0;
        for (int o = 0; o < p.groups; ++o) {
            const auto other = image_of(sums[o]);
            rank += other > mine || (other == mine && o < g);
        }
        const bool keep = rank < p.kept_groups;
        kept[g] = keep;
        if (v == v) {
            if (keep) worst_kept = v < worst_kept ? v : worst_kept;
            else best_left = v > best_left ? v : best_left;
        }
    }
    wave_sync();
    if (!exact) {
        worst_kept = team_reduce<L>(worst_kept, [](C a, C b) { return b < a ? b : a; });
        best_left = team_reduce<L>(best_left, [](C a, C b) { return b > a ? b : a; });
        // Two sums of two choices carry four scores' errors, a rounding of each sum (2 u of the larger one in all, at
        // most 4 u of the largest choice) and of each choice with its bias: 4 u of the largest choice, however
        // small the sums are where biases cancel.
        largest = team_reduce<L>(largest, [](float a, float b) { return fmaxf(a, b); });
        const float a = static_cast<float>(worst_kept), b = static_cast<float>(best_left);
        if (best_left != none && !(a - b > 2.0f * scores + 0x1p-20f * largest)) unsure = true;
    }
}

// A row's logits, the absent ones -inf.
template <typename S, int KIND, int L, int ITEMS>
struct RouteRow {
    float x[ITEMS];
    float mx, inverse;        // softmax: the largest logit (a finite number), 1 / sum of exp(x - mx)

    // NEIGHBOURS: a lane's items lie side by side (lane * ITEMS + i), in one or two accesses.
    template <bool NEIGHBOURS = false>
    __device__ __forceinline__ void load(const S* row, int n, int lane) {
        if (NEIGHBOURS && (lane + 1) * ITEMS <= n) {
            const auto v = *reinterpret_cast<const typename AnyVec<S, ITEMS>::type*>(row + lane * ITEMS);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) x[i] = static_cast<float>(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int e = NEIGHBOURS ? lane * ITEMS + i : i * L + lane;
                x[i] = e < n ? static_cast<float>(row[e]) : kMinusInfinity;
            }
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) x[i] = x[i] <= lowest_of<S>() ? kMinusInfinity : x[i];
        mx = -std::numeric_limits<float>::max();
        inverse = 0.0f;
        if constexpr (KIND == kSoftmaxScore) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) mx = fmaxf(mx, x[i]);
            mx = team_reduce<L>(mx, [](float a, float b) { return fmaxf(a, b); });
        }
    }
    __device__ __forceinline__ void normalise() {
        if constexpr (KIND == kSoftmaxScore) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) sum += power(x[i]);
            sum = team_reduce<L>(sum, [](float a, float b) { return a + b; });
            inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        }
    }
    __device__ __forceinline__ float error() const { return KIND == kSoftmaxScore ? 0x1p-18f * inverse : 0x1p-20f; }      // see border()
    __device__ __forceinline__ float power(float v) const { return __builtin_amdgcn_exp2f((v - mx) * kLog2E); }
    __device__ __forceinline__ float score(float v) const {
        if constexpr (KIND == kSoftmaxScore) {
            return power(v) * inverse;
        } else {
            const float e = __builtin_amdgcn_exp2f(-fabsf(v) * kLog2E), r = __builtin_amdgcn_rcpf(1.0f + e);
            return v < 0.0f ? e * r : r;
        }
    }
};

// The k choices of one row in 64 bits by a wavefront, one after the other: place t ends in lane t.
template <typename S, int KIND>
__device__ __forceinline__ int choose_exactly(const RouteCall& p, const S* x, double* items, int lane) {
    double mx = -std::numeric_limits<float>::max(), sum = 0.0;
    auto logit = [&](int e) {
        const float v = static_cast<float>(x[e]);
        return v <= lowest_of<S>() ? kMinusInfinity : v;
    };
    if constexpr (KIND == kSoftmaxScore) {
#pragma unroll 1
        for (int e = lane; e < p.n; e += kWave) mx = fmax(mx, static_cast<double>(logit(e)));
        mx = wave_reduce(mx, [](double a, double b) { return b > a ? b : a; });
    }
    wave_sync();
#pragma unroll 1
    for (int e = lane; e < p.n; e += kWave) {
        const double v = logit(e);
        const double s = KIND == kSoftmaxScore ? exp(v - mx) : 1.0 / (1.0 + exp(-v));
        sum += s;
        items[e] = s;
    }
    double by = 1.0;
    if constexpr (KIND == kSoftmaxScore) {
        sum = wave_reduce(sum, [](double a, double b) { return a + b; });
        by = sum == 0.0 ? 0.0 : 1.0 / sum;
    }
    // (a lane reads back what it wrote)
#pragma unroll 1
    for (int e = lane; e < p.n; e += kWave) {
        const float v = logit(e);
        double c = items[e] * by + (p.bias ? static_cast<double>(p.bias[e]) : 0.0);
        if (!p.bias && (p.kept_groups == p.groups || p.group_best == 1)) c = v;
        items[e] = v == kMinusInfinity ? std::numeric_limits<double>::quiet_NaN() : c;
    }
    wave_sync();
    const bool grouped = p.kept_groups < p.groups;
    uint8_t* flags = reinterpret_cast<uint8_t*>(items + p.n + p.n / 2);
    if (grouped) {
        double* sums = items;                                // (groups of one expert are their experts)
        bool settled = false;
        if (p.size > 1) group_values<kWave>(p, items, sums = items + p.n, lane);
        keep_groups<kWave>(p, sums, flags, true, 0.0f, 0.0f, lane, settled);
    }
    uint64_t* images = reinterpret_cast<uint64_t*>(items);
#pragma unroll 1
    for (int e = lane; e < p.n; e += kWave) {
        double c = items[e];
        if (!p.bias && c == c) c = logit(e);
        images[e] = grouped && !flags[(e * p.size_magic) >> 20] ? 0 : image_of(c);
    }
    int mine = 0;
#pragma unroll 1
    for (int t = 0; t < p.k; ++t) {
        uint64_t best = 0;
        int at = 0x7fffffff;
#pragma unroll 1
        for (int e = lane; e < p.n; e += kWave) {
            const uint64_t v = images[e];
            if (v > best) best = v, at = e;
        }
        const uint64_t top = wave_reduce(best, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        at = wave_reduce(best == top ? at : 0x7fffffff, [](int a, int b) { return a < b ? a : b; });
        if (at % kWave == lane) images[at] = 0;              // (its own lane's)
        if (lane == t) mine = at;
    }
    return mine;
}

// The k choices in fp32: place t ends in lane t.  `unsure` when they may not be the exact ones.
template <typename S, int KIND, int L, int ITEMS>
__device__ __forceinline__ int choose(const RouteCall& p, const RouteRow<S, KIND, L, ITEMS>& row, const S* x, float* lds, int lane, bool& unsure) {
    uint32_t image[ITEMS];
    {
        float c[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            c[i] = row.x[i];
            if (p.bias) c[i] = row.score(c[i]) + (i * L + lane < p.n ? p.bias[i * L + lane] : 0.0f);
        }
        const bool grouped = p.kept_groups < p.groups;
        uint8_t* flags = reinterpret_cast<uint8_t*>(lds + 2 * L * ITEMS);
        if (grouped) {
            // (without a bias: by the scores where two are added, else by the logits themselves)
            const bool exact = !p.bias && p.group_best == 1;
            wave_sync();
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const float v = p.bias || exact ? c[i] : row.score(row.x[i]);
                if (i * L + lane < p.n) lds[i * L + lane] = row.x[i] == kMinusInfinity ? std::numeric_limits<float>::quiet_NaN() : v;
            }
            wave_sync();
            const float largest = group_values<L>(p, lds, lds + L * ITEMS, lane);
            keep_groups<L>(p, lds + L * ITEMS, flags, exact, row.error(), largest, lane, unsure);
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t there = row.x[i] == kMinusInfinity ? 1 : image_of(c[i]);
            image[i] = i * L + lane < p.n ? there : 0;
        }
        if (grouped) {
            // (every item reads a flag, those past the last expert one that nobody set)
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const uint32_t open = flags[((i * L + lane) * p.size_magic) >> 20];
                image[i] = open ? image[i] : 0;
            }
        }
    }
    // candidates: everything from the (k+1)-th largest of the lanes' largest items on
    uint32_t most = image[0];
#pragma unroll
    for (int i = 1; i < ITEMS; ++i) most = image[i] > most ? image[i] : most;
    wave_bitonic<L, true>([&](auto jc, bool keep_better) {
        const uint32_t other = lane_xor_const<decltype(jc)::value>(most);
        most = keep_better == (other > most) ? other : most;
    });
    const int base = lane_id() & ~(L - 1);
    uint32_t bound = p.k < L ? lane_get(most, base + p.k) : 0;
    if (bound == 0) bound = 1;
    int count = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) count += image[i] >= bound;
    int upto = count;
    {
        int o = dpp_fetch<kRowShr1>(upto, 0);
        upto += o;
        o = dpp_fetch<kRowShr2>(upto, 0);
        upto += o;
        o = dpp_fetch<kRowShr4>(upto, 0);
        upto += o;
        o = dpp_fetch<kRowShr8>(upto, 0);
        upto += o;
        if constexpr (L == kWave) {
            o = dpp_fetch<kRowBcast15, 0xa>(upto, 0);
            upto += o;
            o = dpp_fetch<kRowBcast31, 0xc>(upto, 0);
            upto += o;
        }
    }
    const int total = lane_get(upto, base + L - 1);
    uint64_t* slots = reinterpret_cast<uint64_t*>(lds);
    constexpr int SLOTS = 2 * L;
    wave_sync();
    int place = upto - count;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if (image[i] >= bound) {
            if (place < SLOTS) slots[place] = static_cast<uint64_t>(image[i]) << 32 | (0xffffffffu - static_cast<uint32_t>(i * L + lane));
            ++place;
        }
    }
    wave_sync();
    uint64_t mine = lane < total ? slots[lane] : 0;
    auto sort = [&](uint64_t& v) {
        wave_bitonic<L, true>([&](auto jc, bool keep_better) {
            const uint64_t other = lane_xor_const<decltype(jc)::value>(v);
            v = keep_better == (other > v) ? other : v;
        });
    };
    sort(mine);
    if (__any(total > L)) {
        // a second word for some lanes: ordered by itself, its largest against the first words' smallest
        uint64_t more = L + lane < total ? slots[L + lane] : 0;
        sort(more);
        const uint64_t other = lane_get(more, base + (L - 1) - (lane_id() & (L - 1)));
        mine = other > mine ? other : mine;
        sort(mine);
    }
    if (__any(total > SLOTS)) {
        // (equal logits in masses) one after the other
        uint64_t word = 0;
        for (int t = 0; t <= p.k; ++t) {
            uint64_t best = 0;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const uint64_t w = static_cast<uint64_t>(image[i]) << 32 | (0xffffffffu - static_cast<uint32_t>(i * L + lane));
                if (image[i] && w > best) best = w;
            }
            best = team_reduce<L>(best, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
            const int e = static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
                if (i * L + lane == e) image[i] = 0;
            if (lane == t) word = best;
        }
        if (total > SLOTS) mine = word;
    }
    if (p.bias) {
        // neighbours too close for fp32; equal logits with equal biases are equal, whatever the precision
        const uint64_t next = lane_get(mine, base + ((lane + 1) & (L - 1)));
        const uint32_t a = static_cast<uint32_t>(mine >> 32), b = static_cast<uint32_t>(next >> 32);
        if (p.k == L && lane == p.k - 1) unsure = true;           // (no lane for the place behind the last)
        else if (lane < p.k && a > 1 && b > 1) {
            const float va = value_of(a), vb = value_of(b);
            if (!(va - vb > border(row.error(), va, vb))) {
                const int ea = static_cast<int>(0xffffffffu - static_cast<uint32_t>(mine)), eb = static_cast<int>(0xffffffffu - static_cast<uint32_t>(next));
                const bool equal = static_cast<float>(x[ea]) == static_cast<float>(x[eb]) && p.bias[ea] == p.bias[eb];
                // (the last place against the first one left out: others of that value may follow unseen)
                if (!equal || lane == p.k - 1) unsure = true;
            }
        }
    }
    return static_cast<int>(0xffffffffu - static_cast<uint32_t>(mine));
}

// A chosen logit's score over exp(top) (logistic: over exp(min(top, 0))), top the largest chosen one: where only ratios
// count, as after a renormalisation, scores below fp32's range keep theirs.
template <int KIND>
__device__ __forceinline__ float score_to(float v, float top) {
    if constexpr (KIND == kSoftmaxScore) return __builtin_amdgcn_exp2f((v - top) * kLog2E);
    else return __builtin_amdgcn_exp2f((fminf(v, 0.0f) - fminf(top, 0.0f)) * kLog2E) / (1.0f + __builtin_amdgcn_exp2f(-fabsf(v) * kLog2E));
}

// What place `lane` < k of row r gets once its expert e is settled.
constexpr int32_t kUnsettled = -1;
template <typename S, int KIND, int L, int ITEMS>
__device__ __forceinline__ void settle(const RouteCall& p, const RouteRow<S, KIND, L, ITEMS>& row, const S* xr, int e, int64_t r, bool live, int lane,
                                       int32_t* histogram) {
    float s = 0.0f, total = 1.0f;
    const bool place = lane < p.k;
    const float v = place ? static_cast<float>(xr[e]) : kMinusInfinity;
    const bool there = place && !(v <= lowest_of<S>());
    if (p.renormalise) {
        const float top = team_reduce<L>(there ? v : kMinusInfinity, [](float a, float b) { return fmaxf(a, b); });
        if (there) s = score_to<KIND>(v, top);
    } else if (there) {
        s = row.score(v);
    }
    if (p.renormalise) {
        total = team_reduce<L>(s, [](float a, float b) { return a + b; });
        if (total == 0.0f) total = 1.0f;
    }
    if (live && place) {
        p.weights[r * p.k + lane] = p.renormalise ? s / total * p.scale : s * p.scale;
        p.indices[r * p.k + lane] = e;
        if (p.loads) atomicAdd(&histogram[e], 1);
    }
}

__device__ __forceinline__ void clear_loads(const RouteCall& p, int32_t* histogram) {
    if (!p.loads) return;
    for (int e = threadIdx.x; e < p.n; e += 256) histogram[e] = 0;
    __syncthreads();
}
__device__ __forceinline__ void flush_loads(const RouteCall& p, int32_t* histogram) {
    if (!p.loads) return;
    __syncthreads();
    for (int e = threadIdx.x; e < p.n; e += 256)
        if (histogram[e]) atomicAdd(&p.loads[e], histogram[e]);
}

// (four wavefronts to a SIMD, which the LDS of 256 experts has room for: left alone, the compiler takes 130 registers,
// two too many, and fp32 [32768, 256] with groups takes 44.1 us a call instead of 38.6)
template <typename S, int KIND, int L, int ITEMS>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4))) void route_rows(const S* x, RouteCall p) {
    constexpr int TEAMS = 256 / L;
    __shared__ double lds[TEAMS][team_doubles<L, ITEMS>()];
    __shared__ int32_t histogram[L * ITEMS];
    const int lane = threadIdx.x % L, team = threadIdx.x / L;
    clear_loads(p, histogram);
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * TEAMS; r0 < p.m; r0 += static_cast<int64_t>(gridDim.x) * TEAMS) {
        const int64_t r = r0 + team;
        const bool live = r < p.m;
        const S* xr = x + (live ? r : 0) * p.stride;
        RouteRow<S, KIND, L, ITEMS> row;
        row.load(xr, p.n, lane);
        if (p.bias || p.kept_groups < p.groups || !p.renormalise) row.normalise();
        bool unsure = false;
        const int e = choose<S, KIND, L, ITEMS>(p, row, xr, reinterpret_cast<float*>(lds[team]), lane, unsure);
        if (team_reduce<L>(static_cast<int>(unsure), [](int a, int b) { return a | b; })) {
            if (live && lane == 0) p.indices[r * p.k] = kUnsettled;
            continue;
        }
        settle<S, KIND, L, ITEMS>(p, row, xr, e, r, live, lane, histogram);
    }
    flush_loads(p, histogram);
}

// Rows that route_rows left marked: kRowsPerWave neighbouring rows to a wavefront.
constexpr int kRowsPerWave = 4;
template <typename S, int KIND, int ITEMS>
__global__ __launch_bounds__(256) void route_unsettled(const S* x, RouteCall p) {
    __shared__ double lds[4][kWave * ITEMS * 13 / 8];          // the experts' values, the groups' (half as many), a byte per group
    __shared__ int32_t histogram[kWave * ITEMS];
    const int lane = lane_id(), wave = threadIdx.x / kWave;
    clear_loads(p, histogram);
    const int64_t r0 = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * kRowsPerWave;
    const bool marked = lane < kRowsPerWave && r0 + lane < p.m && p.indices[(r0 + lane) * p.k] == kUnsettled;
    for (uint64_t rows = __ballot(marked); rows; rows &= rows - 1) {
        const int64_t r = r0 + __builtin_ctzll(rows);
        const S* xr = x + r * p.stride;
        RouteRow<S, KIND, kWave, ITEMS> row;
        row.load(xr, p.n, lane);
        row.normalise();
        const int e = choose_exactly<S, KIND>(p, xr, lds[wave], lane);
        settle<S, KIND, kWave, ITEMS>(p, row, xr, e, r, true, lane, histogram);
    }
    flush_loads(p, histogram);
}

struct RouteGradCall {
    int64_t m, stride, dx_stride;
    int n, k, renormalise;
    float scale;
    const int32_t* indices;
    const float* dweights;
};

// With c the chosen experts, d the weights' gradients times scale:
//   sigmoid:                 dx[c] = d s (1 - s);  renormalised: q (d - sum d q) (1 - s), q = s / S, S the chosen scores' sum
//   softmax:                 dx = s (ds - sum ds s), over every expert
//   softmax, renormalised:   the weights are the chosen logits' own softmax q: dx[c] = q (d - sum d q), 0 elsewhere -
//                            only the k chosen logits are read.
// The places' gradients meet the row in LDS; a lane writes ITEMS neighbouring experts.  (The same by
// handing every place to every lane and comparing: 14.6 us for bf16 [65537, 128], k = 8, against this one's
// 8.2, at 4.6 TB/s.)  An index that stands in the row twice is added up in the order of the places.
template <typename S, int KIND, int L, int ITEMS>
__global__ __launch_bounds__(256) void route_grad_rows(const S* x, S* dx, RouteGradCall p) {
    constexpr int TEAMS = 256 / L;
    const int lane = threadIdx.x % L, team = threadIdx.x / L;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * TEAMS + team;
    __shared__ float lds[TEAMS][L * (ITEMS + 1)];          // (one left over per lane: 64 lanes, 64 banks, also over four teams)
    __shared__ uint8_t owners[TEAMS][L * ITEMS];
    auto slot = [&](int e) -> float& { return lds[team][e + e / ITEMS]; };
    float* const own = &lds[team][lane * (ITEMS + 1)];
    const bool live = r < p.m;
    const int64_t rr = live ? r : p.m - 1;
    const S* xr = x + rr * p.stride;
    const int32_t* index = p.indices + rr * p.k;
    const float* dw = p.dweights + rr * p.k;
    auto add = [](float a, float b) { return a + b; };

    RouteRow<S, KIND, L, ITEMS> row;
    if (!(KIND == kSoftmaxScore && p.renormalise)) {
        row.template load<true>(xr, p.n, lane);
        row.normalise();
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) own[i] = 0.0f;
    // the places of the row, L at a time: place t in lane t % L
    float top = kMinusInfinity, total = 0.0f, dot = 0.0f;
    auto fetch = [&](int t, int& e, float& v, float& d) {
        e = t < p.k ? index[t] : -1;
        const bool ok = e >= 0 && e < p.n;
        v = ok ? static_cast<float>(xr[e]) : kMinusInfinity;
        d = ok ? dw[t] * p.scale : 0.0f;
        if (v <= lowest_of<S>()) e = -1;                 // absent: no weight, no gradient
    };
    int first_e;
    float first_v, first_d;
    fetch(lane, first_e, first_v, first_d);
    auto place = [&](int t0, int& e, float& v, float& d) {
        if (t0) fetch(t0 + lane, e, v, d);
        else e = first_e, v = first_v, d = first_d;
    };
    if (p.renormalise) {
        for (int t0 = 0; t0 < p.k; t0 += L) {
            int e;
            float v, d;
            place(t0, e, v, d);
            if (e >= 0) top = fmaxf(top, v);
        }
        top = team_reduce<L>(top, [](float a, float b) { return fmaxf(a, b); });
    }
    auto score = [&](float v) { return p.renormalise ? score_to<KIND>(v, top) : row.score(v); };
    for (int t0 = 0; t0 < p.k; t0 += L) {
        int e;
        float v, d;
        place(t0, e, v, d);
        const float s = e >= 0 ? score(v) : 0.0f;
        total += s;
        dot += d * s;
    }
    total = team_reduce<L>(total, add);
    dot = team_reduce<L>(dot, add);
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    wave_sync();
    for (int t0 = 0; t0 < p.k; t0 += L) {
        int e;
        float v, d;
        place(t0, e, v, d);
        float g = 0.0f;
        if (e >= 0) {
            float s = score(v);
            if (p.renormalise) s *= by, d -= dot * by;
            if constexpr (KIND == kSoftmaxScore) g = s * d;
            else g = s * d * row.score(-v);
        }
        if (e >= 0) owners[team][e] = static_cast<uint8_t>(lane);
        wave_sync();
        if (__any(e >= 0 && owners[team][e] != lane)) {
            for (int t = 0; t < L && t0 + t < p.k; ++t) {
                if (lane == t && e >= 0) slot(e) += g;
                wave_sync();
            }
        } else if (e >= 0) {
            slot(e) += g;
        }
        wave_sync();
    }
    if (!live) return;
    float grad[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        grad[i] = own[i];
        if (KIND == kSoftmaxScore && !p.renormalise) grad[i] -= dot * row.score(row.x[i]);
    }
    S* out = dx + r * p.dx_stride + lane * ITEMS;
    if ((lane + 1) * ITEMS <= p.n) {
        typename AnyVec<S, ITEMS>::type v;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) v[i] = static_cast<S>(grad[i]);
        *reinterpret_cast<typename AnyVec<S, ITEMS>::type*>(out) = v;
    } else {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (lane * ITEMS + i < p.n) out[i] = static_cast<S>(grad[i]);
    }
}

// f(lanes of a team, items of a lane): sixteen lanes while their items fit and the places leave the
// border's one to spare, otherwise a wavefront.
template <typename F>
int dispatch_team(int64_t n, int64_t k, F&& f) {
    using std::integral_constant;
    if (k < 16) {
        if (n <= 64) return f(integral_constant<int, 16>(), integral_constant<int, 4>());
        if (n <= 128) return f(integral_constant<int, 16>(), integral_constant<int, 8>());
        if (n <= 256) return f(integral_constant<int, 16>(), integral_constant<int, 16>());
    }
    if (n <= 256) return f(integral_constant<int, kWave>(), integral_constant<int, 4>());
    return f(integral_constant<int, kWave>(), integral_constant<int, 16>());
}

int check(const char* name, int64_t m, int64_t n, int64_t k, const void* x, int64_t stride, int* kind) {
    if (!name || !x || m <= 0 || n <= 0 || k <= 0 || k > n || stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    if (!std::strcmp(name, "softmax")) *kind = kSoftmaxScore;
    else if (!std::strcmp(name, "sigmoid")) *kind = kSigmoidScore;
    else return DLFX_ERR_UNKNOWN_OP;
    if (n > DLFX_ROUTE_MAX_N || k > DLFX_ROUTE_MAX_K || ceil_div(m, 4) > kMostThreads / 256) return DLFX_ERR_TOO_LARGE;
    return DLFX_OK;
}

}  // namespace
}  // namespace dlfx

using namespace dlfx;

extern "C" int dlfx_route(dlfx_stream_t stream, const char* name, int dtype, int64_t m, int64_t n,
                          const void* x, int64_t x_offset, int64_t row_stride, const float* bias,
                          int64_t groups, int64_t kept_groups, int group_best, int64_t k, int renormalise, float scale,
                          float* weights, int32_t* indices, int32_t* loads) {
    int kind;
    if (int e = check(name, m, n, k, x, row_stride, &kind)) return e;
    if (!weights || !indices) return DLFX_ERR_INVALID_ARGUMENT;
    if (groups <= 0 || n % groups || kept_groups <= 0 || kept_groups > groups || (group_best != 1 && group_best != 2)) return DLFX_ERR_INVALID_ARGUMENT;
    const int64_t size = n / groups;
    if (kept_groups * size < k) return DLFX_ERR_INVALID_ARGUMENT;
    RouteCall p{m, row_stride, static_cast<int>(n), static_cast<int>(groups), static_cast<int>(kept_groups), group_best, static_cast<int>(size),
                static_cast<int>(ceil_div(1 << 20, size)), static_cast<int>(k), renormalise, scale, bias, weights, indices, loads};
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        return dispatch_team(n, k, [&](auto lanes, auto items) {
            constexpr int L = decltype(lanes)::value, ITEMS = decltype(items)::value;
            auto run = [&](auto kernel) {
                // counting: a workgroup takes many rows, or adding up its counters costs more than the rows
                const int64_t blocks = ceil_div(m, 256 / L), most = loads ? 512 : 0x7fffffffLL;
                kernel<<<dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                    static_cast<const S*>(x) + x_offset, p);
                DLFX_CHECK_LAUNCH();
                return static_cast<int>(DLFX_OK);
            };
            auto again = [&](auto kernel) {
                kernel<<<dim3(static_cast<unsigned>(ceil_div(m, 4 * kRowsPerWave))), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                    static_cast<const S*>(x) + x_offset, p);
                DLFX_CHECK_LAUNCH();
                return static_cast<int>(DLFX_OK);
            };
            const bool exact = !bias && (kept_groups == groups || group_best == 1);
            int status = kind == kSoftmaxScore ? run(route_rows<S, kSoftmaxScore, L, ITEMS>) : run(route_rows<S, kSigmoidScore, L, ITEMS>);
            if (status != DLFX_OK || exact) return status;
            // (a team of 16 lanes has up to 256 experts: four to a lane of a wavefront)
            constexpr int MANY = L == 16 ? 4 : ITEMS;
            return kind == kSoftmaxScore ? again(route_unsettled<S, kSoftmaxScore, MANY>) : again(route_unsettled<S, kSigmoidScore, MANY>);
        });
    });
}

extern "C" int dlfx_route_grad(dlfx_stream_t stream, const char* name, int dtype, int64_t m, int64_t n,
                               const void* x, int64_t x_offset, int64_t row_stride,
                               int64_t k, const int32_t* indices, const float* dweights, int renormalise, float scale,
                               void* dx, int64_t dx_offset, int64_t dx_row_stride) {
    int kind;
    if (int e = check(name, m, n, k, x, row_stride, &kind)) return e;
    if (!indices || !dweights || !dx || dx_row_stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    RouteGradCall p{m, row_stride, dx_row_stride, static_cast<int>(n), static_cast<int>(k), renormalise, scale, indices, dweights};
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        if (overwrites(static_cast<const S*>(x) + x_offset, row_stride, static_cast<const S*>(dx) + dx_offset, dx_row_stride, m))
            return static_cast<int>(DLFX_ERR_INVALID_ARGUMENT);
        return dispatch_team(n, 1, [&](auto lanes, auto items) {
            constexpr int L = decltype(lanes)::value, ITEMS = decltype(items)::value;
            auto run = [&](auto kernel) {
                kernel<<<dim3(static_cast<unsigned>(ceil_div(m, 256 / L))), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                    static_cast<const S*>(x) + x_offset, static_cast<S*>(dx) + dx_offset, p);
                DLFX_CHECK_LAUNCH();
                return static_cast<int>(DLFX_OK);
            };
            return kind == kSoftmaxScore ? run(route_grad_rows<S, kSoftmaxScore, L, ITEMS>) : run(route_grad_rows<S, kSigmoidScore, L, ITEMS>);
        });
    });
}
