// Group normalisation, forward: see norm.cuh.
#include "norm.cuh"

namespace stdml::collective::train
{
namespace
{
constexpr int kAhead = 4;  // rows that a thread has on their way

template <typename T, int kCh, int kAct, bool kResidual>
__global__ void __launch_bounds__(kNormThreads, 4) forward_kernel(NormArgs a)
{
    extern __shared__ __align__(16) unsigned char raw[];
    using V = Vec<T, kCh>;
    const bool cluster = a.walks == 3 && a.slices > 1;
    if (cluster) { cluster_begin(); }
    const Part p(a);
    const Grid<kCh> g(p.width);
    float2 *lines = reinterpret_cast<float2 *>(raw);
    float *lines_first = reinterpret_cast<float *>(raw) + 2 * kNormThreads * kCh;  // each channel's first value in the slice
    double2 *shares = reinterpret_cast<double2 *>(lines_first + (a.width + 3) / 4 * 4), *total = shares + kNormThreads, *all = total + a.width;
    const int groups = p.width / a.per, g0 = p.c0 / a.per;
    const long long count = p.to - p.from;
    // (here, where the loads below hide what a division in 64 bits takes)
    const double each = count > 0 ? 1.0 / static_cast<double>(count) : 0.0;
    const T *x = static_cast<const T *>(a.x.ptr) + p.n * a.x.image + p.c0;

    if ((a.walks & 1) != 0) {
        // ---- sums of x less the slice's first value of the channel, and of their squares
        for (int pass = 0; pass < g.passes; ++pass) {
            const int col = g.column(pass);
            float s1[kCh] = {}, s2[kCh] = {};
            if (col < g.columns && g.row() < g.down && count > 0) {
                const V base = *reinterpret_cast<const V *>(x + p.from * a.x.row + col * kCh);
                if (g.row() == 0) {
#pragma unroll
                    for (int i = 0; i < kCh; ++i) { lines_first[col * kCh + i] = base.at(i); }
                }
                Walker<V> wx(x, a.x.row, p.from + g.row(), col, kCh, g.down);
                const int rows = static_cast<int>((count - g.row() + g.down - 1) / g.down);
                const auto add = [&](const V &v) {
#pragma unroll
                    for (int i = 0; i < kCh; ++i) {
                        const float d = v.at(i) - base.at(i);
                        s1[i] += d;
                        s2[i] += d * d;
                    }
                };
                int it = 0;
                for (; it + kAhead <= rows; it += kAhead, wx.next(kAhead)) {
                    V v[kAhead];
#pragma unroll
                    for (int k = 0; k < kAhead; ++k) { v[k] = wx.load(k); }
#pragma unroll
                    for (int k = 0; k < kAhead; ++k) {
                        add(v[k]);
                    }
                }
                for (; it < rows; ++it, wx.next(1)) {
                    const V v = wx.load(0);
                    add(v);
                }
            }
            column_sums<kCh>(g, pass, p.width, s1, s2, lines, shares, total);
        }
        __syncthreads();
        // ---- mean and sum of squared deviations of each group in the slice
        const double share = a.per_value * static_cast<double>(a.positions);
        if (cluster) { cluster_runs(); }
        each_group(groups, a.per, [&](int k, int lane, int lanes, auto gather) {
            // (a channel's mean: its first value in the slice, and the mean of what lies above it)
            const auto mean_of = [&](int c) { return count > 0 ? lines_first[c] + total[c].x * each : 0.0; };
            double mean = 0, dev = 0;
            for (int c = k * a.per + lane; c < (k + 1) * a.per; c += lanes) { mean += mean_of(c); }
            mean = gather(mean) * share;
            for (int c = k * a.per + lane; c < (k + 1) * a.per; c += lanes) {
                const double2 t = total[c];
                const double off = mean_of(c) - mean;
                dev += t.y - t.x * t.x * each + off * off * count;
            }
            dev = gather(dev);
            if (lane == 0) { publish(a, p, all, groups, g0, k, make_double2(mean, dev)); }
        });
        if (a.walks == 1) { return; }
        if (cluster) {
            cluster_sync();
        } else {
            __syncthreads();
        }
    }
    // ---- of the slices together: total[group] = mean, 1 / deviation
    for (int k = threadIdx.x; k < groups; k += blockDim.x) {
        double mean = 0, dev = 0;
        const auto rows_in = [&](int i) {
            return static_cast<double>(a.slices <= 32 ? portion(a.positions, i + 1, a.slices) - portion(a.positions, i, a.slices)
                                                      : a.positions * (i + 1) / a.slices - a.positions * i / a.slices);
        };
        for (int i = 0; i < a.slices; ++i) { mean += published(a, p, all, groups, g0, k, i).x * (rows_in(i) * a.per_position); }
        for (int i = 0; i < a.slices; ++i) {
            const double2 v = published(a, p, all, groups, g0, k, i);
            dev += v.y + (v.x - mean) * (v.x - mean) * rows_in(i) * a.per;
        }
        const double rstd = rsqrt(dev * a.per_value + a.eps);
        total[k] = make_double2(mean, rstd);
        if (p.slice == 0) { reinterpret_cast<double2 *>(a.stats)[p.n * a.groups + g0 + k] = total[k]; }
    }
    __syncthreads();
    // ---- results
    const T *r = static_cast<const T *>(a.r.ptr);
    if (kResidual) { r += p.n * a.r.image + p.c0; }
    T *y = static_cast<T *>(const_cast<void *>(a.y.ptr)) + p.n * a.y.image + p.c0;
    for (int pass = 0; pass < g.passes; ++pass) {
        const int col = g.column(pass);
        if (col >= g.columns || g.row() >= g.down) { continue; }
        // (x - mean) * scale + bias as one multiply-add: either way what is lost is what 32 bits lose of mean * scale
        float scale[kCh], shift[kCh];
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            const int c = col * kCh + i;
            const double2 st = total[c / a.per];
            const double k = st.y * weight_of(a, p.c0 + c);
            scale[i] = static_cast<float>(k);
            shift[i] = static_cast<float>(bias_of(a, p.c0 + c) - st.x * k);
        }
        Walker<V> wx(x, a.x.row, p.from + g.row(), col, kCh, g.down), wy(y, a.y.row, p.from + g.row(), col, kCh, g.down),
            wr = wy;
        if (kResidual) { wr = Walker<V>(r, a.r.row, p.from + g.row(), col, kCh, g.down); }
        const int rows = static_cast<int>(max(0ll, (count - g.row() + g.down - 1) / g.down));
        wx.turn(rows);  // (what was read last is in the L2 still)
        wy.turn(rows);
        wr.turn(rows);
        const auto finish = [&](const V &v, const V &res, int k) {
            float out[kCh];
#pragma unroll
            for (int i = 0; i < kCh; ++i) {
                float z = fmaf(v.at(i), scale[i], shift[i]);
                if (kResidual) { z += res.at(i); }
                out[i] = act<T, kAct>(z);
            }
            V o;
            o.set(out);
            wy.store(k, o);
        };
        int it = 0;
        for (; it + kAhead <= rows; it += kAhead) {
            V v[kAhead], res[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                v[k] = wx.load(k);
                if (kResidual) { res[k] = wr.load(k); }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) { finish(v[k], res[k], k); }
            wx.next(kAhead);
            wy.next(kAhead);
            wr.next(kAhead);
        }
        for (; it < rows; ++it) {
            V res;
            if (kResidual) { res = wr.load(0); }
            finish(wx.load(0), res, 0);
            wx.next(1);
            wy.next(1);
            wr.next(1);
        }
    }
}
template <typename T, int kCh, int kAct>
void forward(const NormArgs &n, cudaStream_t s)
{
    if (n.r.ptr != nullptr) {
        norm_walks(forward_kernel<T, kCh, kAct, true>, n, kCh, s);
    } else {
        norm_walks(forward_kernel<T, kCh, kAct, false>, n, kCh, s);
    }
}
}  // namespace

void norm_forward_launch(const NormArgs &n, int dt, int vector, int act, cudaStream_t s)
{
    by_dtype(dt, [&](auto t) {
        using T = decltype(t);
        by_act(act, [&](auto k) {
            constexpr int kAct = decltype(k)::value, kFull = 16 / sizeof(T);
            if constexpr (kAct != STDMLC_ACT_GELU_TANH) {
                if (vector >= kFull) {
                    forward<T, kFull, kAct>(n, s);
                } else if (vector >= 2) {
                    forward<T, 2, kAct>(n, s);
                } else {
                    forward<T, 1, kAct>(n, s);
                }
            }
        });
    });
}
}  // namespace stdml::collective::train
