// Backward pass of the gated linear recurrence.
#include "gated_common.hip.h"

namespace dlfx {
namespace {

template <typename S>
struct GradCall {
    Cut cut;
    Track<const S> g, x, y, dy;
    Track<S> dg, dx;
    Track<const float> initial, dlast;
    Track<float> dinitial;
    Stretch* records;
    float* entering;
};

// Everything of one step that does not depend on what comes from the steps after it: the factor a,
// the gradient dy, side = (state before the step) * a' and, for "gated_blend", 1 - a.
template <typename S, int KIND>
__device__ __forceinline__ void step_of(float g, float x, float before, float& a, float& keep, float& side) {
    keep = 1.0f;
    gate_of<S, KIND>(g, a, keep);
    if constexpr (KIND == kGatedBlend) before -= x;
    if constexpr (KIND == kGated) side = before;
    else if constexpr (KIND == kGatedExp) side = before * a;
    else side = before * (a * keep);
}

// A short axis: one lane per row, step after step.
template <typename S, int KIND>
__global__ __launch_bounds__(256) void gated_grad_walk(GradCall<S> p) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (r >= p.cut.m) return;
    const S* gp = p.g.base + p.g.row.at(r);
    const S* xp = KIND == kGatedBlend ? p.x.base + p.x.row.at(r) : nullptr;
    const S* yp = p.y.base + p.y.row.at(r);
    const S* dyp = p.dy.base + p.dy.row.at(r);
    S* dgp = p.dg.base + p.dg.row.at(r);
    S* dxp = p.dx.base + p.dx.row.at(r);
    float mu = p.dlast.base ? p.dlast.base[p.dlast.row.at(r)] : 0.0f;
    const float h0 = p.initial.base ? p.initial.base[p.initial.row.at(r)] : 0.0f;
    for (int64_t t = p.cut.n - 1; t >= 0; --t) {
        float a, keep, side;
        step_of<S, KIND>(static_cast<float>(gp[t * p.g.step]), KIND == kGatedBlend ? static_cast<float>(xp[t * p.x.step]) : 0.0f,
                         t > 0 ? static_cast<float>(yp[(t - 1) * p.y.step]) : h0, a, keep, side);
        const float lam = static_cast<float>(dyp[t * p.dy.step]) + mu;
        mu = a * lam;
        dgp[t * p.dg.step] = static_cast<S>(lam * side);
        dxp[t * p.dx.step] = static_cast<S>(KIND == kGatedBlend ? lam * keep : lam);
    }
    if (p.dinitial.base) p.dinitial.base[p.dinitial.row.at(r)] = mu;
}

constexpr int kGradSteps = 8;       // of a wavefront in a pass

// Rows side by side, as in the forward kernel, from the last step to the first: position i of the
// walk is step n - 1 - i.  Eight steps a pass: four inputs of them and two outputs fill the registers.
// Bound by HBM as the forward kernel: bf16 [8, 4096, 2048] sigmoid 147 us (4.6 TB/s), blend 173 us (4.7), [64, 4096, 512]
// 316 us (5.1); fp32 [3, 1777, 515], cut, 11.3 + 21.8 us (latency: a pass or two by 176 workgroups).
template <typename S, int KIND, int V, int W, typename OFF, bool NT, bool PARTIAL>
__global__ __launch_bounds__(W * kWave) void gated_grad_cols(GradCall<S> p) {
    constexpr int N = kGradSteps;
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
    auto offset = [&](const auto& track) { return static_cast<OFF>(track.row.at(r) * static_cast<int64_t>(sizeof(S))); };
    const OFF go = offset(p.g), dyo = offset(p.dy);
    const OFF xo = KIND == kGatedBlend ? offset(p.x) : OFF(0);
    const OFF yo = offset(p.y), dgo = offset(p.dg), dxo = offset(p.dx);
    const int64_t begin = segment * p.cut.length;
    const int64_t end = begin + p.cut.length < p.cut.n ? begin + p.cut.length : p.cut.n;
    const int64_t top = p.cut.n - 1;

    float carry[V], h0[V];
    double product[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        product[v] = 1.0;
        carry[v] = h0[v] = 0.0f;
        if constexpr (!PARTIAL) {
            if (segment == p.cut.segments - 1 && p.initial.base) h0[v] = p.initial.base[p.initial.row.at(r + v)];
        }
        if (p.cut.segments == 1 || (PARTIAL && segment == 0)) {
            const float d = p.dlast.base ? p.dlast.base[p.dlast.row.at(r + v)] : 0.0f;
            if constexpr (PARTIAL) {
                if (wave == 0) p.entering[r + v] = d;
            } else {
                carry[v] = d;
            }
        } else if (!PARTIAL) {
            if constexpr (cut_columns<V, W>()) {
                __shared__ Stretch shares[W][kWave];
                carry[v] = enter_column<W>(p.records, p.cut.m, r, segment, p.entering[r], shares);
            }
        }
    }

    if constexpr (!PARTIAL) share_carry<V, W>(carry, wave, lane);

    Vec<S, V> graw[N], dyraw[N], yraw[N], xraw[N];
    float a[N][V], d[N][V], keep[N][V], side[N][V];
    // Position i0 + i: the state before it is the next position's, for the axis's last one `initial`.
    auto fetch_one = [&](int i, const S* gp, const S* dyp, const S* yp, const S* xp, OFF gi, OFF dyi, OFF yi, OFF xi) {
        graw[i] = load_at<NT, S, V>(gp, gi);
        dyraw[i] = load_at<NT, S, V>(dyp, dyi);
        if constexpr (!PARTIAL) {
            yraw[i] = load_at<NT, S, V>(yp, yi);
            if constexpr (KIND == kGatedBlend) xraw[i] = load_at<NT, S, V>(xp, xi);
        }
    };
    auto fetch = [&](int64_t i0) {
        const int64_t t0 = top - i0;
        const S* gp = p.g.base + t0 * p.g.step;
        const S* dyp = p.dy.base + t0 * p.dy.step;
        const S* yp = p.y.base + (t0 - 1) * p.y.step;
        const S* xp = KIND == kGatedBlend ? p.x.base + t0 * p.x.step : nullptr;
        const OFF gi = as_it_is(go), dyi = as_it_is(dyo), yi = as_it_is(yo), xi = as_it_is(xo);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            fetch_one(i, gp, dyp, yp, xp, gi, dyi, yi, xi);
            gp -= p.g.step;
            dyp -= p.dy.step;
            yp -= p.y.step;
            if constexpr (KIND == kGatedBlend) xp -= p.x.step;
        }
    };
    auto widen = [&](int64_t i0, bool last) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                d[i][v] = static_cast<float>(dyraw[i].v[v]);
                float before = 0.0f, x = 0.0f;
                if constexpr (!PARTIAL) {
                    before = static_cast<float>(yraw[i].v[v]);
                    if (last && i0 + i == top) before = h0[v];
                    if constexpr (KIND == kGatedBlend) x = static_cast<float>(xraw[i].v[v]);
                }
                step_of<S, KIND>(static_cast<float>(graw[i].v[v]), x, before, a[i][v], keep[i][v], side[i][v]);
            }
        }
    };
    int parity = 0;
    float entering[V], first[V];
    auto enter = [&](float (&mu)[V]) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float pa = a[0][v], pb = a[0][v] * d[0][v];
#pragma unroll
            for (int i = 1; i < N; ++i) {
                pa *= a[i][v];
                pb = a[i][v] * (d[i][v] + pb);
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
            mu[v] = first[v] = mine;
        }
        parity ^= 1;
    };
    auto gradient = [&](int i, float (&mu)[V], Vec<S, V>& dg, Vec<S, V>& dx) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float lam = d[i][v] + mu[v];
            mu[v] = a[i][v] * lam;
            dg.v[v] = static_cast<S>(lam * side[i][v]);
            dx.v[v] = static_cast<S>(KIND == kGatedBlend ? lam * keep[i][v] : lam);
        }
    };

    // whole passes, but for one that holds the axis's last position
    const int64_t reach = end < top ? end : top;
    const int64_t passes = reach > begin ? (reach - begin) / (W * N) : 0;
    int64_t i0 = begin + wave * N;
    // (after enter has turned to the other half of lds)
    auto repair = [&](int64_t past) {
        repair_pass<V, W>(lds[parity], wave, lane, entering, carry, first, [&](float (&mu)[V]) {
            S* dgp = p.dg.base + (top - i0) * p.dg.step;
            S* dxp = p.dx.base + (top - i0) * p.dx.step;
#pragma unroll
            for (int i = 0; i < N; ++i, dgp -= p.dg.step, dxp -= p.dx.step) {
                Vec<S, V> dg, dx;
                gradient(i, mu, dg, dx);
                if (i0 + i < past) {
                    store_at<false, S, V>(dgp, dgo, dg);
                    store_at<false, S, V>(dxp, dxo, dx);
                }
            }
        });
    };
    auto walk = [&] {
        float mu[V];
        enter(mu);
        if constexpr (!PARTIAL) {
            S* dgp = p.dg.base + (top - i0) * p.dg.step;
            S* dxp = p.dx.base + (top - i0) * p.dx.step;
            const OFF dgi = as_it_is(dgo), dxi = as_it_is(dxo);
#pragma unroll
            for (int i = 0; i < N; ++i, dgp -= p.dg.step, dxp -= p.dx.step) {
                Vec<S, V> dg, dx;
                gradient(i, mu, dg, dx);
                store_at<NT, S, V>(dgp, dgi, dg);
                store_at<NT, S, V>(dxp, dxi, dx);
            }
            repair(i0 + N);
        }
        i0 += W * N;
    };
    if (passes > 0) {
        fetch(i0);
        for (int64_t pass = 1; pass < passes; ++pass) {
            widen(i0, false);
            fetch(i0 + W * N);
            walk();
        }
        widen(i0, false);
        walk();
    }
    if (begin + passes * (W * N) < end) {
        // the last, shorter pass: positions past the end read the last one and become neutral, without a branch
        const OFF gi = as_it_is(go), dyi = as_it_is(dyo), yi = as_it_is(yo), xi = as_it_is(xo);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t t = top - (i0 + i < end ? i0 + i : end - 1);
            fetch_one(i, p.g.base + t * p.g.step, p.dy.base + t * p.dy.step, p.y.base + (t > 0 ? t - 1 : 0) * p.y.step,
                      KIND == kGatedBlend ? p.x.base + t * p.x.step : nullptr, gi, dyi, yi, xi);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                graw[i].v[v] = i0 + i < end ? graw[i].v[v] : neutral_gate<S, KIND>();
                dyraw[i].v[v] = i0 + i < end ? dyraw[i].v[v] : static_cast<S>(0.0f);
            }
        }
        widen(i0, true);
        float mu[V];
        enter(mu);
        if constexpr (!PARTIAL) {
            S* dgp = p.dg.base + (top - i0) * p.dg.step;
            S* dxp = p.dx.base + (top - i0) * p.dx.step;
#pragma unroll
            for (int i = 0; i < N; ++i, dgp -= p.dg.step, dxp -= p.dx.step) {
                Vec<S, V> dg, dx;
                gradient(i, mu, dg, dx);
                if (i0 + i < end) {
                    store_at<NT, S, V>(dgp, dgo, dg);
                    store_at<NT, S, V>(dxp, dxo, dx);
                }
            }
            repair(end);
        }
    }
    if constexpr (PARTIAL) {
        // a segment whose state got lost (as in repair_pass) or whose product passed the range once more, step after step
        if (wave == 0 && !(finite(carry[0]) && in_range(product[0]))) {
            float state = 0.0f;
            double far = 1.0;
            for (int64_t t = top - begin; t > top - end; --t) {
                float factor, rest = 1.0f;
                gate_of<S, KIND>(static_cast<float>(load_at<false, S, 1>(p.g.base + t * p.g.step, go).v[0]), factor, rest);
                state = factor * (static_cast<float>(load_at<false, S, 1>(p.dy.base + t * p.dy.step, dyo).v[0]) + state);
                far = times(far, static_cast<double>(factor));
            }
            carry[0] = state;
            product[0] = far;
        }
    }
    if (wave == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (PARTIAL) p.records[segment * p.cut.m + r + v] = {product[v], carry[v]};
            else if (p.dinitial.base && segment == p.cut.segments - 1) p.dinitial.base[p.dinitial.row.at(r + v)] = carry[v];
        }
    }
}

template <typename S, int KIND, int V, int W, typename OFF, bool NT>
int launch_cols(GradCall<S> p, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    p.cut.blocks = ceil_div(p.cut.m, kWave * V);
    int64_t segments = cut_columns<V, W>() ? column_segments<S>(p.cut.blocks, p.cut.n, W * kGradSteps) : 1;
    if (segments > 1 && (!scratch || scratch_bytes < records_bytes(p.cut.m, segments))) return DLFX_ERR_SCRATCH_TOO_SMALL;
    p.cut.length = align_up(ceil_div(p.cut.n, segments), W * kGradSteps);
    segments = p.cut.segments = ceil_div(p.cut.n, p.cut.length);
    if (grid_of(p.cut.blocks * segments) > kMostThreads / (W * kWave)) return DLFX_ERR_TOO_LARGE;
    if constexpr (cut_columns<V, W>()) {
        if (segments > 1) {
            p.records = static_cast<Stretch*>(scratch);
            p.entering = reinterpret_cast<float*>(static_cast<char*>(scratch) + align_up(static_cast<size_t>(p.cut.m * (segments - 1)) * sizeof(Stretch), 256));
            gated_grad_cols<S, KIND, V, W, OFF, NT, true><<<dim3(static_cast<unsigned>(grid_of(p.cut.blocks * (segments - 1)))), dim3(W * kWave), 0, stream>>>(p);
            DLFX_CHECK_LAUNCH();
        }
    }
    gated_grad_cols<S, KIND, V, W, OFF, NT, false><<<dim3(static_cast<unsigned>(grid_of(p.cut.blocks * segments))), dim3(W * kWave), 0, stream>>>(p);
    DLFX_CHECK_LAUNCH();
    return DLFX_OK;
}

// Rows along memory, as in the forward kernel, from the last step to the first; DIR is the direction
// of the walk in memory.  bf16 [16384, 4096] 139 us (4.8 TB/s), fp32 [1000000, 64] 236 us (5.4 TB/s).
template <typename S, int KIND, int G, int W, int DIR, bool PARTIAL>
__global__ __launch_bounds__(W > 4 ? W * kWave : 256) void gated_grad_rows(GradCall<S> p) {
    static_assert(W == 1 || G == kWave, "whole wavefronts share a row");
    constexpr int N = run_length<S>();
    constexpr int BLOCK = W > 4 ? W * kWave : 256, TEAM = W * G, TEAMS = BLOCK / TEAM;
    constexpr int PASS = TEAM * N;
    __shared__ Stretch lds[W > 1 ? 2 : 1][W > 1 ? TEAMS : 1][W];
    const int team = threadIdx.x / TEAM, place = threadIdx.x % TEAM, wave = place / kWave;
    const int64_t segment = PARTIAL ? blockIdx.x / p.cut.blocks : p.cut.segments - 1 - blockIdx.x / p.cut.blocks;
    const int64_t wanted = (blockIdx.x % p.cut.blocks) * TEAMS + team;
    if (wanted - (W == 1 ? threadIdx.x % kWave / G : 0) >= p.cut.m) return;      // (as in the forward kernel)
    const int64_t r = wanted < p.cut.m ? wanted : p.cut.m - 1;
    const int64_t n = p.cut.n, top = n - 1;
    // position i of the walk is step n - 1 - i, DIR elements further on in memory each
    auto start = [&](const auto& track) { return track.base + track.row.at(r) - DIR * top; };
    const S* gp = start(p.g);
    const S* dyp = start(p.dy);
    const S* xp = KIND == kGatedBlend ? start(p.x) : nullptr;
    const S* before_p = start(p.y) + DIR;            // the state before position i is the one of position i + 1
    S* dgp = start(p.dg);
    S* dxp = start(p.dx);
    const int64_t begin = segment * p.cut.length;
    const int64_t end = begin + p.cut.length < n ? begin + p.cut.length : n;

    float carry = 0.0f, h0 = 0.0f;
    double product = 1.0;
    if constexpr (!PARTIAL) {
        if (segment == p.cut.segments - 1 && p.initial.base) h0 = p.initial.base[p.initial.row.at(r)];
    }
    if (p.cut.segments == 1 || (PARTIAL && segment == 0)) {
        const float d = p.dlast.base ? p.dlast.base[p.dlast.row.at(r)] : 0.0f;
        if constexpr (PARTIAL) {
            if (place == 0) p.entering[r] = d;
        } else {
            carry = d;
        }
    } else if (!PARTIAL) {
        carry = p.entering[r];
        if constexpr (W > 4) carry = enter_segment(p.records, p.cut.m, r, segment, carry);
    }

    S graw[N], dyraw[N], yraw[N], xraw[N];
    float a[N], d[N], keep[N], side[N];
    auto fetch = [&](int64_t i) {
        load_run<true, DIR>(gp, i, end, graw);
        load_run<true, DIR>(dyp, i, end, dyraw);
        if constexpr (!PARTIAL) {
            load_run<true, DIR>(before_p, i, end, yraw);
            if constexpr (KIND == kGatedBlend) load_run<true, DIR>(xp, i, end, xraw);
        }
    };
    auto widen = [&](int64_t i0, bool last) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            d[i] = static_cast<float>(dyraw[i]);
            float before = 0.0f, x = 0.0f;
            if constexpr (!PARTIAL) {
                before = static_cast<float>(yraw[i]);
                if (last && i0 + i == top) before = h0;
                if constexpr (KIND == kGatedBlend) x = static_cast<float>(xraw[i]);
            }
            step_of<S, KIND>(static_cast<float>(graw[i]), x, before, a[i], keep[i], side[i]);
        }
    };
    int parity = 0;
    auto enter = [&]() -> float {
        float pa = a[0], pb = a[0] * d[0];
#pragma unroll
        for (int i = 1; i < N; ++i) {
            pa *= a[i];
            pb = a[i] * (d[i] + pb);
        }
        Stretch before, all;
        join_lanes<G>({pa, pb}, before, all, [&] { return product_of(pa, a); });
        float mu = carry;
        if constexpr (W > 1) {
            if (lane_id() == 0) lds[parity][team][wave] = all;
            __syncthreads();
            float c = carry;
            double far = product;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (w == wave) mu = c;
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
        return through(before, mu);
    };
    auto gradients = [&](float mu, S (&dg)[N], S (&dx)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float lam = d[i] + mu;
            mu = a[i] * lam;
            dg[i] = static_cast<S>(lam * side[i]);
            dx[i] = static_cast<S>(KIND == kGatedBlend ? lam * keep[i] : lam);
        }
    };

    // whole passes, but for one that holds the axis's last position
    const int64_t reach = end < top ? end : top;
    const int64_t passes = reach > begin ? (reach - begin) / PASS : 0;
    int64_t i0 = begin + place * N;
    auto walk = [&] {
        const float mu = enter();
        if constexpr (!PARTIAL) {
            S dg[N], dx[N];
            gradients(mu, dg, dx);
            store_run<true, DIR>(dgp, i0, end, dg);
            store_run<true, DIR>(dxp, i0, end, dx);
        }
        i0 += PASS;
    };
    if (passes > 0) {
        fetch(i0);
        for (int64_t pass = 1; pass < passes; ++pass) {
            widen(i0, false);
            fetch(i0 + PASS);
            walk();
        }
        widen(i0, false);
        walk();
    }
    if (begin + passes * PASS < end) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            graw[i] = neutral_gate<S, KIND>();
            dyraw[i] = yraw[i] = xraw[i] = static_cast<S>(0.0f);
        }
        load_run<false, DIR>(gp, i0, end, graw);
        load_run<false, DIR>(dyp, i0, end, dyraw);
        if constexpr (!PARTIAL) {
            load_run<false, DIR>(before_p, i0, reach, yraw);
            if constexpr (KIND == kGatedBlend) load_run<false, DIR>(xp, i0, end, xraw);
        }
        widen(i0, true);
        const float mu = enter();
        if constexpr (!PARTIAL) {
            S dg[N], dx[N];
            gradients(mu, dg, dx);
            store_run<false, DIR>(dgp, i0, end, dg);
            store_run<false, DIR>(dxp, i0, end, dx);
        }
    }
    if (place == 0) {
        if constexpr (PARTIAL) p.records[segment * p.cut.m + r] = {product, carry};
        else if (p.dinitial.base && segment == p.cut.segments - 1) p.dinitial.base[p.dinitial.row.at(r)] = carry;
    }
}

template <typename S, int KIND, int G, int W, int DIR>
int launch_rows(GradCall<S> p, void* scratch, size_t scratch_bytes, hipStream_t stream) {
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
            gated_grad_rows<S, KIND, G, W, DIR, true><<<dim3(static_cast<unsigned>(p.cut.blocks * (segments - 1))), dim3(BLOCK), 0, stream>>>(p);
            DLFX_CHECK_LAUNCH();
        }
    }
    gated_grad_rows<S, KIND, G, W, DIR, false><<<dim3(static_cast<unsigned>(p.cut.blocks * segments)), dim3(BLOCK), 0, stream>>>(p);
    DLFX_CHECK_LAUNCH();
    return DLFX_OK;
}

template <typename S, int KIND, int DIR>
int launch_direction(const GradCall<S>& p, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    const int64_t runs = p.cut.n / run_length<S>();
    if (runs < 16) return launch_rows<S, KIND, 4, 1, DIR>(p, scratch, scratch_bytes, stream);
    if (runs < 32) return launch_rows<S, KIND, 16, 1, DIR>(p, scratch, scratch_bytes, stream);
    if (runs < kWave) return launch_rows<S, KIND, 32, 1, DIR>(p, scratch, scratch_bytes, stream);
    if (p.cut.m >= 2048 && runs < 32 * kWave) return launch_rows<S, KIND, kWave, 1, DIR>(p, scratch, scratch_bytes, stream);
    if (p.cut.m >= 512 || runs <= 4 * kWave) return launch_rows<S, KIND, kWave, 4, DIR>(p, scratch, scratch_bytes, stream);
    return launch_rows<S, KIND, kWave, 16, DIR>(p, scratch, scratch_bytes, stream);
}

template <typename S, int KIND>
int launch_grad(const GradCall<S>& p, void* scratch, size_t scratch_bytes, hipStream_t stream) {
    const int64_t m = p.cut.m, n = p.cut.n;
    if (n <= kWalked) {
        if (ceil_div(m, 256) > kMostThreads / 256) return DLFX_ERR_TOO_LARGE;
        gated_grad_walk<S, KIND><<<dim3(static_cast<unsigned>(ceil_div(m, 256))), dim3(256), 0, stream>>>(p);
        DLFX_CHECK_LAUNCH();
        return DLFX_OK;
    }
    const int d = direction(p.y);
    if (d != 0 && d == direction(p.g) && d == direction(p.dy) && d == direction(p.dg) && d == direction(p.dx) && (KIND != kGatedBlend || d == direction(p.x)))
        return d > 0 ? launch_direction<S, KIND, -1>(p, scratch, scratch_bytes, stream) : launch_direction<S, KIND, 1>(p, scratch, scratch_bytes, stream);
    if (!(short_offsets(p.g) && short_offsets(p.x) && short_offsets(p.y) && short_offsets(p.dy) && short_offsets(p.dg) && short_offsets(p.dx)))
        return launch_cols<S, KIND, 1, 16, int64_t, false>(p, scratch, scratch_bytes, stream);
    const bool lines = whole_lines(p.g) && whole_lines(p.x) && whole_lines(p.y) && whole_lines(p.dy) && whole_lines(p.dg) && whole_lines(p.dx);
    if constexpr (sizeof(S) == 2) {
        if (m >= kManyPairs && pairs_of_rows(p.g) && pairs_of_rows(p.x) && pairs_of_rows(p.y) && pairs_of_rows(p.dy) &&
            pairs_of_rows(p.dg) && pairs_of_rows(p.dx))
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

extern "C" int dlfx_gated_scan_grad(dlfx_stream_t stream, const char* name, int dtype, int64_t m, int64_t n,
                                    int rank, const int64_t* dims,
                                    const void* gate, int64_t gate_offset, const int64_t* gate_strides,
                                    const void* x, int64_t x_offset, const int64_t* x_strides,
                                    const float* initial, int64_t initial_offset, const int64_t* initial_strides,
                                    const void* y, int64_t y_offset, const int64_t* y_strides,
                                    const void* dy, int64_t dy_offset, const int64_t* dy_strides,
                                    const float* dlast, int64_t dlast_offset, const int64_t* dlast_strides,
                                    void* dgate, int64_t dgate_offset, const int64_t* dgate_strides,
                                    void* dx, int64_t dx_offset, const int64_t* dx_strides,
                                    float* dinitial, int64_t dinitial_offset, const int64_t* dinitial_strides,
                                    void* scratch, size_t scratch_bytes) {
    if (!name || !gate || !y || !dy || !dgate || !dx || !gate_strides || !y_strides || !dy_strides || !dgate_strides || !dx_strides)
        return DLFX_ERR_INVALID_ARGUMENT;
    const int kind = kind_of(name);
    if (kind < 0) return DLFX_ERR_UNKNOWN_OP;
    if (kind == kGatedBlend && (!x || !x_strides)) return DLFX_ERR_INVALID_ARGUMENT;
    if (!shape_ok(m, n, rank, dims, dx_strides) || !strides_distinct(rank, dims, dx_strides) || !strides_distinct(rank, dims, dgate_strides))
        return DLFX_ERR_INVALID_ARGUMENT;
    if (rank > 1 && ((initial && !initial_strides) || (dlast && !dlast_strides) || (dinitial && !dinitial_strides))) return DLFX_ERR_INVALID_ARGUMENT;
    if (dinitial && !strides_distinct(rank - 1, dims, dinitial_strides)) return DLFX_ERR_INVALID_ARGUMENT;
    if (kind != kGatedBlend) x = nullptr;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        GradCall<S> p{};
        p.cut.m = m;
        p.cut.n = n;
        if (!make_track(rank, dims, gate, gate_offset, gate_strides, false, &p.g) || !make_track(rank, dims, x, x_offset, x_strides, false, &p.x) ||
            !make_track(rank, dims, y, y_offset, y_strides, false, &p.y) || !make_track(rank, dims, dy, dy_offset, dy_strides, false, &p.dy) ||
            !make_track(rank, dims, dgate, dgate_offset, dgate_strides, false, &p.dg) ||
            !make_track(rank, dims, dx, dx_offset, dx_strides, false, &p.dx) ||
            !make_track(rank, dims, initial, initial_offset, initial_strides, true, &p.initial) ||
            !make_track(rank, dims, dlast, dlast_offset, dlast_strides, true, &p.dlast) ||
            !make_track(rank, dims, dinitial, dinitial_offset, dinitial_strides, true, &p.dinitial))
            return static_cast<int>(DLFX_ERR_RANK);
        return dispatch_kind(kind, [&](auto k) { return launch_grad<S, decltype(k)::value>(p, scratch, scratch_bytes, s); });
    });
}
