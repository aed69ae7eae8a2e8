// Gated linear recurrence h[t] = a[t] h[t-1] + b[t] along one axis of strided views.
#include <algorithm>

#include "gated_common.hip.h"

namespace dlfx {
namespace {

template <typename S>
struct ScanCall {
    Cut cut;
    Track<const S> g, x;
    Track<S> y;
    Track<const float> initial;
    Track<float> last;
    Stretch* records;       // cut.segments - 1 per row, segment-major
    float* entering;        // m states (cut calls)
};

// A short axis: one lane per row, step after step.  A decoding step, bf16 [48, 1, 2560]: 5.1 us, a launch's latency.
template <typename S, int KIND>
__global__ __launch_bounds__(256) void gated_walk(ScanCall<S> p) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (r >= p.cut.m) return;
    const S* gp = p.g.base + p.g.row.at(r);
    const S* xp = p.x.base + p.x.row.at(r);
    S* yp = p.y.base + p.y.row.at(r);
    float h = p.initial.base ? p.initial.base[p.initial.row.at(r)] : 0.0f;
    for (int64_t t = 0; t < p.cut.n; ++t) {
        float a, keep = 1.0f, b = static_cast<float>(xp[t * p.x.step]);
        gate_of<S, KIND>(static_cast<float>(gp[t * p.g.step]), a, keep);
        if constexpr (KIND == kGatedBlend) b *= keep;
        h = fmaf(a, h, b);
        yp[t * p.y.step] = static_cast<S>(h);
    }
    if (p.last.base) p.last.base[p.last.row.at(r)] = h;
}

constexpr int kSteps = 16;       // of a wavefront in a pass

// Rows side by side: lanes run along the rows, wavefronts along the axis.  Every wavefront holds its
// steps of a pass in registers, leaves what they do to the state in LDS, and walks them again from
// the state that the wavefronts before it make of the pass's; the next pass is loaded meanwhile.
// The loop over whole passes has no branch beside its loads and stores: behind one, the wait for the
// next pass's loads would be a wait for this pass's stores.  Lanes past the last row do the last row's
// work over, value for value.
// PARTIAL: only what the segment does to the state, for the segments behind it.
// Bound by HBM, short of it by passes that join at a barrier while the VALU is half busy: bf16 [8, 4096, 2048] blend
// 91 us (4.4 TB/s; a workgroup per CU), [64, 4096, 512] 156 us (5.2 TB/s), fp32 [8, 4096, 2048] 154 us (5.2 TB/s);
// cut, fp32 [1, 65536, 1000] 121 + 148 us (4.4 and 5.4 TB/s of what the two launches move).
template <typename S, int KIND, int V, int W, typename OFF, bool NT, bool PARTIAL>
__global__ __launch_bounds__(W * kWave) void gated_cols(ScanCall<S> p) {
    constexpr int N = kSteps;
    __shared__ float lds[2][W][kWave][2 * V];
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t work = work_of(blockIdx.x, gridDim.x);
    if (work >= p.cut.blocks * (PARTIAL ? p.cut.segments - 1 : p.cut.segments)) return;
    // (segments from the last one on after PARTIAL went from the first: what it read last may still be cached)
    const int64_t segment = PARTIAL ? work / p.cut.blocks : p.cut.segments - 1 - work / p.cut.blocks;
    const int64_t block = work % p.cut.blocks;
    const int64_t wanted = (block * kWave + lane) * V;
    const int64_t r = wanted < p.cut.m ? wanted : p.cut.m - V;
    const OFF go = static_cast<OFF>(p.g.row.at(r) * static_cast<int64_t>(sizeof(S)));
    const OFF xo = static_cast<OFF>(p.x.row.at(r) * static_cast<int64_t>(sizeof(S)));
    const OFF yo = static_cast<OFF>(p.y.row.at(r) * static_cast<int64_t>(sizeof(S)));
    const int64_t begin = segment * p.cut.length;
    const int64_t end = begin + p.cut.length < p.cut.n ? begin + p.cut.length : p.cut.n;

    float carry[V];
    double product[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        product[v] = 1.0;
        carry[v] = 0.0f;
        if (p.cut.segments == 1 || (PARTIAL && segment == 0)) {
            const float h = p.initial.base ? p.initial.base[p.initial.row.at(r + v)] : 0.0f;
            if constexpr (PARTIAL) {
                if (wave == 0) p.entering[r + v] = h;
            } else {
                carry[v] = h;
            }
        } else if (!PARTIAL) {
            if constexpr (cut_columns<V, W>()) {
                __shared__ Stretch shares[W][kWave];
                carry[v] = enter_column<W>(p.records, p.cut.m, r, segment, p.entering[r], shares);
            }
        }
    }

    if constexpr (!PARTIAL) share_carry<V, W>(carry, wave, lane);

    Vec<S, V> graw[N], xraw[N];
    float a[N][V], b[N][V];
    auto fetch = [&](int64_t t0) {
        const S* gp = p.g.base + t0 * p.g.step;
        const S* xp = p.x.base + t0 * p.x.step;
        const OFF gi = as_it_is(go), xi = as_it_is(xo);
#pragma unroll
        for (int i = 0; i < N; ++i, gp += p.g.step, xp += p.x.step) {
            graw[i] = load_at<NT, S, V>(gp, gi);
            xraw[i] = load_at<NT, S, V>(xp, xi);
        }
    };
    auto widen = [&] {
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float keep = 1.0f;
                b[i][v] = static_cast<float>(xraw[i].v[v]);
                gate_of<S, KIND>(static_cast<float>(graw[i].v[v]), a[i][v], keep);
                if constexpr (KIND == kGatedBlend) b[i][v] *= keep;
            }
        }
    };
    // The pass's states from the stretches of all wavefronts; h: the state that enters this one's steps.
    int parity = 0;
    float entering[V], first[V];
    auto enter = [&](float (&h)[V]) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float pa = a[0][v], pb = b[0][v];
#pragma unroll
            for (int i = 1; i < N; ++i) {
                pa *= a[i][v];
                pb = fmaf(a[i][v], pb, b[i][v]);
            }
            lds[parity][wave][lane][2 * v] = pa;
            lds[parity][wave][lane][2 * v + 1] = pb;
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float c = entering[v] = carry[v], mine = carry[v];
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (w == wave) mine = c;
                const float wa = lds[parity][w][lane][2 * v];
                c = fmaf(wa, c, lds[parity][w][lane][2 * v + 1]);
                if constexpr (PARTIAL) product[v] *= static_cast<double>(wa);
            }
            carry[v] = c;
            h[v] = first[v] = mine;
        }
        parity ^= 1;
    };
    auto state = [&](int i, float (&h)[V]) {
        Vec<S, V> out;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            h[v] = fmaf(a[i][v], h[v], b[i][v]);
            out.v[v] = static_cast<S>(h[v]);
        }
        return out;
    };

    const int64_t passes = (end - begin) / (W * N);
    int64_t t0 = begin + wave * N;
    // (after enter has turned to the other half of lds)
    auto repair = [&](int64_t past) {
        repair_pass<V, W>(lds[parity], wave, lane, entering, carry, first, [&](float (&h)[V]) {
            S* yp = p.y.base + t0 * p.y.step;
#pragma unroll
            for (int i = 0; i < N; ++i, yp += p.y.step) {
                const Vec<S, V> out = state(i, h);
                if (t0 + i < past) store_at<false, S, V>(yp, yo, out);
            }
        });
    };
    auto walk = [&] {
        float h[V];
        enter(h);
        if constexpr (!PARTIAL) {
            S* yp = p.y.base + t0 * p.y.step;
            const OFF yi = as_it_is(yo);
#pragma unroll
            for (int i = 0; i < N; ++i, yp += p.y.step) store_at<NT, S, V>(yp, yi, state(i, h));
            repair(t0 + N);
        }
        t0 += W * N;
    };
    if (passes > 0) {
        fetch(t0);
        for (int64_t pass = 1; pass < passes; ++pass) {
            widen();
            fetch(t0 + W * N);
            walk();
        }
        widen();
        walk();
    }
    if (begin + passes * (W * N) < end) {
        // the last, shorter pass: steps past the end read the last one and become neutral, without a branch
        const OFF gi = as_it_is(go), xi = as_it_is(xo);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t t = t0 + i < end ? t0 + i : end - 1;
            graw[i] = load_at<NT, S, V>(p.g.base + t * p.g.step, gi);
            xraw[i] = load_at<NT, S, V>(p.x.base + t * p.x.step, xi);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                graw[i].v[v] = t0 + i < end ? graw[i].v[v] : neutral_gate<S, KIND>();
                xraw[i].v[v] = t0 + i < end ? xraw[i].v[v] : static_cast<S>(0.0f);
            }
        }
        widen();
        float h[V];
        enter(h);
        if constexpr (!PARTIAL) {
            S* yp = p.y.base + t0 * p.y.step;
#pragma unroll
            for (int i = 0; i < N; ++i, yp += p.y.step) {
                const Vec<S, V> out = state(i, h);
                if (t0 + i < end) store_at<NT, S, V>(yp, yo, out);
            }
            repair(end);
        }
    }
    if constexpr (PARTIAL) {
        // a segment whose state got lost (as in repair_pass) or whose product passed the range once more, step after step
        if (wave == 0 && !(finite(carry[0]) && in_range(product[0]))) {
            float h = 0.0f;
            double far = 1.0;
            for (int64_t t = begin; t < end; ++t) {
                float factor, keep = 1.0f, x = static_cast<float>(load_at<false, S, 1>(p.x.base + t * p.x.step, xo).v[0]);
                gate_of<S, KIND>(static_cast<float>(load_at<false, S, 1>(p.g.base + t * p.g.step, go).v[0]), factor, keep);
                if constexpr (KIND == kGatedBlend) x *= keep;
                h = fmaf(factor, h, x);
                far = times(far, static_cast<double>(factor));
            }
            carry[0] = h;
            product[0] = far;
        }
    }
    if (wave == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (PARTIAL) p.records[segment * p.cut.m + r + v] = {product[v], carry[v]};
            else if (p.last.base && segment == p.cut.segments - 1) p.last.base[p.last.row.at(r + v)] = carry[v];
        }
    }
}

template <typename S, int KIND, int V, int W, typename OFF, bool NT>
int launch_cols(ScanCall<S> p, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    p.cut.blocks = ceil_div(p.cut.m, kWave * V);
    int64_t segments = cut_columns<V, W>() ? column_segments<S>(p.cut.blocks, p.cut.n, W * kSteps) : 1;
    if (segments > 1 && (!scratch || scratch_bytes < records_bytes(p.cut.m, segments))) return DLFX_ERR_SCRATCH_TOO_SMALL;
    p.cut.length = align_up(ceil_div(p.cut.n, segments), W * kSteps);
    segments = p.cut.segments = ceil_div(p.cut.n, p.cut.length);
    if (grid_of(p.cut.blocks * segments) > kMostThreads / (W * kWave)) return DLFX_ERR_TOO_LARGE;
    if constexpr (cut_columns<V, W>()) {
        if (segments > 1) {
            p.records = static_cast<Stretch*>(scratch);
            p.entering = reinterpret_cast<float*>(static_cast<char*>(scratch) + align_up(static_cast<size_t>(p.cut.m * (segments - 1)) * sizeof(Stretch), 256));
            gated_cols<S, KIND, V, W, OFF, NT, true><<<dim3(static_cast<unsigned>(grid_of(p.cut.blocks * (segments - 1)))), dim3(W * kWave), 0, stream>>>(p);
            DLFX_CHECK_LAUNCH();
        }
    }
    gated_cols<S, KIND, V, W, OFF, NT, false><<<dim3(static_cast<unsigned>(grid_of(p.cut.blocks * segments))), dim3(W * kWave), 0, stream>>>(p);
    DLFX_CHECK_LAUNCH();
    return DLFX_OK;
}

// Rows along memory: G lanes (4, 16, 32 or 64) or W wavefronts per row, a run of consecutive steps to a
// lane; the lanes' stretches are joined by DPP, the wavefronts' through LDS, pass after pass.  Bound by HBM:
// bf16 [16384, 4096] 77 us (5.2 TB/s), [1000000, 64] 72 us (5.3 TB/s), fp16 [6144, 5001] 43 us (4.3 TB/s: the loads of
// the last, shorter pass wait behind the stores of the one before; calls of [6144, 5120] 42.4 us, five whole passes, of
// [6144, 5000] 45.6, on even elements or odd).
template <typename S, int KIND, int G, int W, int DIR, bool PARTIAL>
__global__ __launch_bounds__(W > 4 ? W * kWave : 256) void gated_rows(ScanCall<S> p) {
    static_assert(W == 1 || G == kWave, "whole wavefronts share a row");
    constexpr int N = run_length<S>();
    constexpr int BLOCK = W > 4 ? W * kWave : 256, TEAM = W * G, TEAMS = BLOCK / TEAM;
    constexpr int PASS = TEAM * N;
    __shared__ Stretch lds[W > 1 ? 2 : 1][W > 1 ? TEAMS : 1][W];
    const int team = threadIdx.x / TEAM, place = threadIdx.x % TEAM, wave = place / kWave;
    const int64_t segment = PARTIAL ? blockIdx.x / p.cut.blocks : p.cut.segments - 1 - blockIdx.x / p.cut.blocks;
    const int64_t wanted = (blockIdx.x % p.cut.blocks) * TEAMS + team;
    // a wavefront past the last row has nothing to do; groups past it beside others do the last row's work
    // over, value for value and in step with the wavefront's group that owns it
    if (wanted - (W == 1 ? threadIdx.x % kWave / G : 0) >= p.cut.m) return;
    const int64_t r = wanted < p.cut.m ? wanted : p.cut.m - 1;
    const S* gp = p.g.base + p.g.row.at(r);
    const S* xp = p.x.base + p.x.row.at(r);
    S* yp = p.y.base + p.y.row.at(r);
    const int64_t begin = segment * p.cut.length;
    const int64_t end = begin + p.cut.length < p.cut.n ? begin + p.cut.length : p.cut.n;

    float carry = 0.0f;
    double product = 1.0;
    if (p.cut.segments == 1 || (PARTIAL && segment == 0)) {
        const float h = p.initial.base ? p.initial.base[p.initial.row.at(r)] : 0.0f;
        if constexpr (PARTIAL) {
            if (place == 0) p.entering[r] = h;
        } else {
            carry = h;
        }
    } else if (!PARTIAL) {
        carry = p.entering[r];
        if constexpr (W > 4) carry = enter_segment(p.records, p.cut.m, r, segment, carry);
    }

    S graw[N], xraw[N];
    float a[N], b[N];
    auto widen = [&] {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float keep = 1.0f;
            b[i] = static_cast<float>(xraw[i]);
            gate_of<S, KIND>(static_cast<float>(graw[i]), a[i], keep);
            if constexpr (KIND == kGatedBlend) b[i] *= keep;
        }
    };
    int parity = 0;
    auto enter = [&]() -> float {
        float pa = a[0], pb = b[0];
#pragma unroll
        for (int i = 1; i < N; ++i) {
            pa *= a[i];
            pb = fmaf(a[i], pb, b[i]);
        }
        Stretch before, all;
        join_lanes<G>({pa, pb}, before, all, [&] { return product_of(pa, a); });
        float h = carry;
        if constexpr (W > 1) {
            if (lane_id() == 0) lds[parity][team][wave] = all;
            __syncthreads();
            float c = carry;
            double far = product;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (w == wave) h = c;
                const Stretch s = lds[parity][team][w];
                c = through(s, c);
                if constexpr (PARTIAL) far *= s.a;
            }
            if constexpr (PARTIAL) {
                if (!in_range(far)) {
                    far = product;
#pragma unroll 1
                    for (int w = 0; w < W; ++w) far = times(far, lds[parity][team][w].a);
                }
                product = far;
            }
            carry = c;
            parity ^= 1;
        } else {
            carry = through(all, carry);
        }
        return through(before, h);
    };
    auto states = [&](float h, S (&out)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            h = fmaf(a[i], h, b[i]);
            out[i] = static_cast<S>(h);
        }
    };

    const int64_t passes = (end - begin) / PASS;
    int64_t i0 = begin + place * N;
    auto fetch = [&](int64_t i) {
        load_run<true, DIR>(gp, i, end, graw);
        load_run<true, DIR>(xp, i, end, xraw);
    };
    auto walk = [&] {
        const float h = enter();
        if constexpr (!PARTIAL) {
            S out[N];
            states(h, out);
            store_run<true, DIR>(yp, i0, end, out);
        }
        i0 += PASS;
    };
    if (passes > 0) {
        fetch(i0);
        for (int64_t pass = 1; pass < passes; ++pass) {
            widen();
            fetch(i0 + PASS);
            walk();
        }
        widen();
        walk();
    }
    if (begin + passes * PASS < end) {
#pragma unroll
        for (int i = 0; i < N; ++i) graw[i] = neutral_gate<S, KIND>(), xraw[i] = static_cast<S>(0.0f);
        load_run<false, DIR>(gp, i0, end, graw);
        load_run<false, DIR>(xp, i0, end, xraw);
        widen();
        const float h = enter();
        if constexpr (!PARTIAL) {
            S out[N];
            states(h, out);
            store_run<false, DIR>(yp, i0, end, out);
        }
    }
    if (place == 0) {
        if constexpr (PARTIAL) p.records[segment * p.cut.m + r] = {product, carry};
        else if (p.last.base && segment == p.cut.segments - 1) p.last.base[p.last.row.at(r)] = carry;
    }
}

template <typename S, int KIND, int G, int W, int DIR>
int launch_rows(ScanCall<S> p, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    constexpr int BLOCK = W > 4 ? W * kWave : 256, PASS = W * G * run_length<S>();
    p.cut.blocks = ceil_div(p.cut.m, BLOCK / (W * G));
    int64_t segments = W > 4 ? row_segments(p.cut.blocks, p.cut.n, PASS) : 1;
    if (segments > 1 && (!scratch || scratch_bytes < records_bytes(p.cut.m, segments))) return DLFX_ERR_SCRATCH_TOO_SMALL;
    p.cut.length = align_up(ceil_div(p.cut.n, segments), PASS);
    segments = p.cut.segments = ceil_div(p.cut.n, p.cut.length);
    if (p.cut.blocks * segments > kMostThreads / BLOCK) return DLFX_ERR_TOO_LARGE;
    if constexpr (W > 4) {
        if (segments > 1) {
            p.records = static_cast<Stretch*>(scratch);
            p.entering = reinterpret_cast<float*>(static_cast<char*>(scratch) + align_up(static_cast<size_t>(p.cut.m * (segments - 1)) * sizeof(Stretch), 256));
            gated_rows<S, KIND, G, W, DIR, true><<<dim3(static_cast<unsigned>(p.cut.blocks * (segments - 1))), dim3(BLOCK), 0, stream>>>(p);
            DLFX_CHECK_LAUNCH();
        }
    }
    gated_rows<S, KIND, G, W, DIR, false><<<dim3(static_cast<unsigned>(p.cut.blocks * segments)), dim3(BLOCK), 0, stream>>>(p);
    DLFX_CHECK_LAUNCH();
    return DLFX_OK;
}

// How rows along memory are walked: no pass is longer than the row (a run is 32 bytes), which would leave lanes
// idle.  us, 4, 16, 32, 64 lanes: bf16 [262144, 64] 22 71 - -, [65536, 256] 22 23 42 -, [32768, 512] - 23 23 42,
// [16384, 1024] - - 22 23.  One, four, sixteen wavefronts: [512, 32768] 45 21 26, [2048, 32768] 86 80 89,
// [256, 131072] - 44 39, [512, 131072] - 82 85; [64, 4096] 10.6 9.8 10.2.
template <typename S, int KIND, int DIR>
int launch_direction(const ScanCall<S>& p, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    const int64_t runs = p.cut.n / run_length<S>();
    if (runs < 16) return launch_rows<S, KIND, 4, 1, DIR>(p, scratch, scratch_bytes, stream);
    if (runs < 32) return launch_rows<S, KIND, 16, 1, DIR>(p, scratch, scratch_bytes, stream);
    if (runs < kWave) return launch_rows<S, KIND, 32, 1, DIR>(p, scratch, scratch_bytes, stream);
    if (p.cut.m >= 2048 && runs < 32 * kWave) return launch_rows<S, KIND, kWave, 1, DIR>(p, scratch, scratch_bytes, stream);
    if (p.cut.m >= 512 || runs <= 4 * kWave) return launch_rows<S, KIND, kWave, 4, DIR>(p, scratch, scratch_bytes, stream);
    return launch_rows<S, KIND, kWave, 16, DIR>(p, scratch, scratch_bytes, stream);
}

template <typename S, int KIND>
int launch_scan(const ScanCall<S>& p, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    const int64_t m = p.cut.m, n = p.cut.n;
    if (n <= kWalked) {
        if (ceil_div(m, 256) > kMostThreads / 256) return DLFX_ERR_TOO_LARGE;
        gated_walk<S, KIND><<<dim3(static_cast<unsigned>(ceil_div(m, 256))), dim3(256), 0, stream>>>(p);
        DLFX_CHECK_LAUNCH();
        return DLFX_OK;
    }
    const int d = direction(p.y);
    if (d != 0 && d == direction(p.g) && d == direction(p.x))
        return d > 0 ? launch_direction<S, KIND, 1>(p, scratch, scratch_bytes, stream) : launch_direction<S, KIND, -1>(p, scratch, scratch_bytes, stream);
    if (!(short_offsets(p.g) && short_offsets(p.x) && short_offsets(p.y)))
        return launch_cols<S, KIND, 1, 16, int64_t, false>(p, scratch, scratch_bytes, stream);
    const bool lines = whole_lines(p.g) && whole_lines(p.x) && whole_lines(p.y);
    if constexpr (sizeof(S) == 2) {
        if (m >= kManyPairs && pairs_of_rows(p.g) && pairs_of_rows(p.x) && pairs_of_rows(p.y))
            return lines ? launch_cols<S, KIND, 2, 1, uint32_t, true>(p, scratch, scratch_bytes, stream)
                         : launch_cols<S, KIND, 2, 1, uint32_t, false>(p, scratch, scratch_bytes, stream);
    }
    const int waves = waves_of(m, n);
    if (waves == 2) return launch_cols<S, KIND, 1, 2, uint32_t, false>(p, scratch, scratch_bytes, stream);
    if (waves == 4) return launch_cols<S, KIND, 1, 4, uint32_t, false>(p, scratch, scratch_bytes, stream);
    if (waves == 8) return launch_cols<S, KIND, 1, 8, uint32_t, false>(p, scratch, scratch_bytes, stream);
    return lines ? launch_cols<S, KIND, 1, 16, uint32_t, true>(p, scratch, scratch_bytes, stream)
                 : launch_cols<S, KIND, 1, 16, uint32_t, false>(p, scratch, scratch_bytes, stream);
}

}  // namespace
}  // namespace dlfx

using namespace dlfx;

// (an upper bound over every layout of m rows of n steps, forward and backward: the query does not see the strides)
extern "C" size_t dlfx_gated_scan_scratch_bytes(int dtype, int64_t m, int64_t n) {
    if (m <= 0 || n <= 0 || (dtype != DLFX_F32 && dtype != DLFX_F16 && dtype != DLFX_BF16)) return 0;
    return records_bytes(m, std::max(column_segments<float>(ceil_div(m, kWave), n, 128), row_segments(m, n, 8192)));
}

extern "C" int dlfx_gated_scan(dlfx_stream_t stream, const char* name, int dtype, int64_t m, int64_t n,
                               int rank, const int64_t* dims,
                               const void* gate, int64_t gate_offset, const int64_t* gate_strides,
                               const void* x, int64_t x_offset, const int64_t* x_strides,
                               const float* initial, int64_t initial_offset, const int64_t* initial_strides,
                               void* y, int64_t y_offset, const int64_t* y_strides,
                               float* last, int64_t last_offset, const int64_t* last_strides,
                               void* scratch, size_t scratch_bytes) {
    if (!name || !gate || !x || !y || !gate_strides || !x_strides || !y_strides) return DLFX_ERR_INVALID_ARGUMENT;
    const int kind = kind_of(name);
    if (kind < 0) return DLFX_ERR_UNKNOWN_OP;
    if (!shape_ok(m, n, rank, dims, y_strides) || !strides_distinct(rank, dims, y_strides)) return DLFX_ERR_INVALID_ARGUMENT;
    if (rank > 1 && ((initial && !initial_strides) || (last && !last_strides))) return DLFX_ERR_INVALID_ARGUMENT;
    if (last && !strides_distinct(rank - 1, dims, last_strides)) return DLFX_ERR_INVALID_ARGUMENT;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        ScanCall<S> p{};
        p.cut.m = m;
        p.cut.n = n;
        if (!make_track(rank, dims, gate, gate_offset, gate_strides, false, &p.g) || !make_track(rank, dims, x, x_offset, x_strides, false, &p.x) ||
            !make_track(rank, dims, y, y_offset, y_strides, false, &p.y) ||
            !make_track(rank, dims, initial, initial_offset, initial_strides, true, &p.initial) ||
            !make_track(rank, dims, last, last_offset, last_strides, true, &p.last))
            return static_cast<int>(DLFX_ERR_RANK);
        return dispatch_kind(kind, [&](auto k) { return launch_scan<S, decltype(k)::value>(p, scratch, scratch_bytes, s); });
    });
}

