// Group normalisation, forward: see norm.cuh.
#include "norm.cuh"

namespace stdml::collective::train
{
namespace
{
constexpr int kAhead = 4;  // rows that a thread has on their way
constexpr int kRun = 16;   // rows whose sums are taken in 32 bits

// Sums of a thread's channels, in 32 bits over a run of rows: of x less a base, and of its square.  s2 - s1^2 / n cancels what the base is
// off by, so the base is a mean of the thread's own: of the first kAhead rows, which are the first run, and of the last run from then
// on.  A value that lies D from all others adds D^2 to what is summed, and its run's mean is off by D / 4 at most, so that the next
// run's 16 squares add up to D^2 before they cancel: 32 bits lose some 2^-21 of D^2 at the worst.  (One base for a whole slice, its first
// value, was off by D in all of the slice's rows; 64 images of 112 x 112 x 64 in bf16 took 61 us with it and take 67.)
template <typename T, int kCh>
struct Run {
    float base[kCh], s1[kCh] = {}, s2[kCh] = {};

    __device__ __forceinline__ void add(const Vec<T, kCh> &v)
    {
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            const float d = v.at(i) - base[i];
            s1[i] += d;
            s2[i] += d * d;
        }
    }
    // A run of `rows`: into the sums in 64 bits, of x less `first` (a value of each channel) and of squared deviations from `first`.
    __device__ __forceinline__ void end(int rows, const float *first, double2 *lines)
    {
        const double n = rows, each = rows == kRun ? 1.0 / kRun : rows == kAhead ? 1.0 / kAhead : 1.0 / n;
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            double2 &l = lines[line_of(i)];
            const double sum = s1[i], off = static_cast<double>(base[i]) - first[i], mean = off + sum * each;
            l = make_double2(l.x + n * mean, l.y + (s2[i] - sum * sum * each + n * mean * mean));
            base[i] += static_cast<float>(sum * each);
            s1[i] = s2[i] = 0;
        }
    }
};

template <typename T, int kCh, int kAct, bool kResidual>
__global__ void __launch_bounds__(kNormThreads, 4) forward_kernel(NormArgs a)
{
    extern __shared__ __align__(16) unsigned char raw[];
    using V = Vec<T, kCh>;
    const bool cluster = a.walks == 3 && a.slices > 1;
    if (cluster) { cluster_begin(); }
    const Part p(a);
    const Grid<kCh> g(p.width);
    double2 *lines = reinterpret_cast<double2 *>(raw);
    float *lines_first = reinterpret_cast<float *>(lines + kNormThreads * kCh);  // each channel's first value in the slice
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
#pragma unroll
            for (int i = 0; i < kCh; ++i) { lines[line_of(i)] = make_double2(0, 0); }
            if (col < g.columns && g.row() == 0 && count > 0) {
                const V v = *reinterpret_cast<const V *>(x + p.from * a.x.row + col * kCh);
#pragma unroll
                for (int i = 0; i < kCh; ++i) { lines_first[col * kCh + i] = v.at(i); }
            }
            __syncthreads();
            if (col < g.columns && g.row() < g.down && count > 0) {
                const float *first = lines_first + col * kCh;
                Walker<V> wx(x, a.x.row, p.from + g.row(), col, kCh, g.down);
                const int rows = static_cast<int>((count - g.row() + g.down - 1) / g.down);
                Run<T, kCh> run;
                int left = rows;
#pragma unroll 1
                while (left >= kAhead) {
                    const int many = left == rows ? kAhead : min(left, kRun) / kAhead * kAhead;
#pragma unroll 1
                    for (int it = 0; it < many; it += kAhead, wx.next(kAhead)) {
                        V v[kAhead];
#pragma unroll
                        for (int k = 0; k < kAhead; ++k) { v[k] = wx.load(k); }
                        if (left == rows) {
#pragma unroll
                            for (int i = 0; i < kCh; ++i) { run.base[i] = 0.25f * v[0].at(i) + 0.25f * v[1].at(i) + 0.25f * v[2].at(i) + 0.25f * v[3].at(i); }
                        }
#pragma unroll
                        for (int k = 0; k < kAhead; ++k) { run.add(v[k]); }
                    }
                    run.end(many, first, lines);
                    left -= many;
                }
                if (left > 0) {
#pragma unroll 1
                    for (int k = 0; k < left; ++k, wx.next(1)) {
                        const V v = wx.load(0);
                        if (k == 0 && left == rows) {
#pragma unroll
                            for (int i = 0; i < kCh; ++i) { run.base[i] = v.at(i); }
                        }
                        run.add(v);
                    }
                    run.end(left, first, lines);
                }
            }
            column_sums<kCh>(g, pass, p.width, lines, shares, total);
        }
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
        // (x - mean) * scale + bias as one multiply-add, whose second term goes with the scale as it was rounded: what is lost is half
        // a step of mean * scale.
        float scale[kCh], shift[kCh];
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            const int c = col * kCh + i;
            const double2 st = total[c / a.per];
            scale[i] = static_cast<float>(st.y * weight_of(a, p.c0 + c));
            shift[i] = static_cast<float>(bias_of(a, p.c0 + c) - st.x * scale[i]);
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
        norm_walks(forward_kernel<T, kCh, kAct, true>, n, kCh, true, s);
    } else {
        norm_walks(forward_kernel<T, kCh, kAct, false>, n, kCh, true, s);
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
