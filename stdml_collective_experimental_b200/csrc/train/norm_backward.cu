// Group normalisation, backward: see norm.cuh.
#include "norm.cuh"

namespace stdml::collective::train
{
namespace
{
constexpr int kAhead = 2;  // rows that a thread has on their way
constexpr int kRun = 64;   // rows whose sums are taken in 32 bits, before 64 take over

// Factors of a thread's channels (four at most: with eight they would not leave room for four blocks on an SM).
// z = x * scale + shift [+ r]; below `near` (and what r adds) its sign is in doubt.
template <int kCh>
struct Factors {
    float mean[kCh], scale[kCh], shift[kCh], near[kCh];
};

// z where 32 bits leave its sign in doubt.
__device__ __noinline__ float placed(float x, float add, double mean, double rstd, float w, float b)
{
    return static_cast<float>((x - mean) * rstd * w + b + add);
}

// dz of a thread's channels in a row, and x - mean.
template <typename T, int kCh, int kAct, bool kResidual>
__device__ __forceinline__ void grad_z(const NormArgs &a, const Part &p, int col, const Factors<kCh> &f, const double2 *stats,
                                       const Vec<T, kCh> &x, const Vec<T, kCh> &r, const Vec<T, kCh> &dy, float (&dz)[kCh], float (&off)[kCh])
{
    constexpr float kDoubt = 4e-6f;  // of the terms that z is made of: some 64 steps of 32 bits
    float z[kCh];
    bool doubt = false;
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
        off[i] = x.at(i) - f.mean[i];
        if constexpr (kAct != STDMLC_ACT_NONE) {
            z[i] = fmaf(x.at(i), f.scale[i], f.shift[i]);
            float near = f.near[i];
            if (kResidual) {
                z[i] += r.at(i);
                if (kAct == STDMLC_ACT_RELU) { near = fmaf(fabsf(r.at(i)), kDoubt, near); }
            }
            if (kAct == STDMLC_ACT_RELU) { doubt = doubt | (fabsf(z[i]) <= near); }
        }
    }
    if (kAct == STDMLC_ACT_RELU && doubt) {
        // the derivative of relu jumps at zero: values that 32 bits leave in doubt are placed in 64
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            const int c = col * kCh + i;
            const double2 st = stats[c / a.per];
            z[i] = placed(x.at(i), kResidual ? r.at(i) : 0.f, st.x, st.y, weight_of(a, p.c0 + c), bias_of(a, p.c0 + c));
        }
    }
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
        dz[i] = dy.at(i);
        if constexpr (kAct == STDMLC_ACT_RELU) {
            dz[i] = z[i] > 0.f ? dz[i] : 0.f;
        } else if constexpr (kAct != STDMLC_ACT_NONE) {
            dz[i] *= act_grad<T, kAct>(z[i]);
        }
    }
}

template <typename T, int kCh, int kAct, bool kResidual>
__global__ void __launch_bounds__(kNormThreads, 4) backward_kernel(NormArgs a)
{
    extern __shared__ __align__(16) unsigned char raw[];
    using V = Vec<T, kCh>;
    const bool cluster = a.walks == 3 && a.slices > 1;
    if (cluster) { cluster_begin(); }
    const Part p(a);
    const Grid<kCh> g(p.width);
    double2 *lines = reinterpret_cast<double2 *>(raw), *shares = lines + kNormThreads * kCh, *total = shares + kNormThreads, *all = total + a.width;
    const int groups = p.width / a.per, g0 = p.c0 / a.per;
    const double2 *stats = reinterpret_cast<const double2 *>(a.stats) + p.n * a.groups + g0;
    const T *x = static_cast<const T *>(a.x.ptr) + p.n * a.x.image + p.c0, *dy = static_cast<const T *>(a.dy.ptr) + p.n * a.dy.image + p.c0;
    const T *r = static_cast<const T *>(a.r.ptr);
    if (kResidual) { r += p.n * a.r.image + p.c0; }

    const auto factors = [&](int col) {
        Factors<kCh> f;
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            const int c = col * kCh + i;
            const double2 st = stats[c / a.per];
            const double k = st.y * weight_of(a, p.c0 + c), bias = bias_of(a, p.c0 + c);
            const float scale = static_cast<float>(k);
            f.mean[i] = static_cast<float>(st.x);
            f.scale[i] = scale;
            f.shift[i] = static_cast<float>(bias - st.x * scale);  // (as in the forward pass)
            f.near[i] = static_cast<float>(4e-6 * (fabs(st.x * k) + fabs(bias)));
        }
        return f;
    };
    // All rows of a thread's: what(x, residual, dy, which of the rows ahead), then next(how many); pause() after each kRun of them.
    const auto walk = [&](int col, bool back, auto what, auto next, auto pause) {
        const long long first = p.from + g.row();
        const int rows = static_cast<int>(max(0ll, (p.to - first + g.down - 1) / g.down));
        Walker<V> wx(x, a.x.row, first, col, kCh, g.down), wd(dy, a.dy.row, first, col, kCh, g.down), wr = wx;
        if (kResidual) { wr = Walker<V>(r, a.r.row, first, col, kCh, g.down); }
        if (back) {  // (what was read last is in the L2 still)
            wx.turn(rows);
            wd.turn(rows);
            wr.turn(rows);
        }
        const auto load = [&](int k, V &vx, V &vr, V &vd) {
            vx = wx.load(k);
            vd = wd.load(k);
            if (kResidual) { vr = wr.load(k); }
        };
        int left = rows;
        while (left >= kAhead) {
            const int rest = max(0, left - kRun);
            for (; left >= rest + kAhead; left -= kAhead) {
                V vx[kAhead], vr[kAhead], vd[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) { load(k, vx[k], vr[k], vd[k]); }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) { what(vx[k], vr[k], vd[k], k); }
                wx.next(kAhead);
                wd.next(kAhead);
                wr.next(kAhead);
                next(kAhead);
            }
            pause();
        }
        for (; left > 0; --left) {
            V vx, vr, vd;
            load(0, vx, vr, vd);
            what(vx, vr, vd, 0);
            wx.next(1);
            wd.next(1);
            wr.next(1);
            next(1);
        }
    };

    if ((a.walks & 1) != 0) {
        // ---- sums of dz and of dz * xh
        for (int pass = 0; pass < g.passes; ++pass) {
            const int col = g.column(pass);
#pragma unroll
            for (int i = 0; i < kCh; ++i) { lines[line_of(i)] = make_double2(0, 0); }
            if (col < g.columns && g.row() < g.down) {
                float s1[kCh] = {}, s2[kCh] = {};
                const auto keep = [&] {
#pragma unroll
                    for (int i = 0; i < kCh; ++i) {
                        double2 &l = lines[line_of(i)];
                        l = make_double2(l.x + s1[i], l.y + s2[i]);
                        s1[i] = s2[i] = 0;
                    }
                };
                const Factors<kCh> f = factors(col);
                const auto add = [&](const V &vx, const V &vr, const V &vd, int) {
                    float dz[kCh], off[kCh];
                    grad_z<T, kCh, kAct, kResidual>(a, p, col, f, stats, vx, vr, vd, dz, off);
#pragma unroll
                    for (int i = 0; i < kCh; ++i) {
                        s1[i] += dz[i];
                        s2[i] += dz[i] * off[i];
                    }
                };
                walk(col, false, add, [](int) {}, keep);
                keep();
            }
            column_sums<kCh>(g, pass, p.width, lines, shares, total);
        }
        for (int c = threadIdx.x; c < p.width; c += kNormThreads) { total[c].y *= stats[c / a.per].y; }  // off * rstd = xh
        __syncthreads();
        if (a.param_sums != nullptr) {
            float *out = a.param_sums + (p.n * a.slices + p.slice) * 2 * a.channels + p.c0;
            for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
                out[c] = static_cast<float>(total[c].x);
                out[a.channels + c] = static_cast<float>(total[c].y);
            }
        }
        if (a.dx.ptr == nullptr && a.dr.ptr == nullptr) {  // (in all blocks)
            if (cluster) { cluster_runs(); }
            return;
        }
        if (cluster) { cluster_runs(); }
        each_group(groups, a.per, [&](int k, int lane, int lanes, auto gather) {
            double m1 = 0, m2 = 0;
            for (int c = k * a.per + lane; c < (k + 1) * a.per; c += lanes) {
                const double w = weight_of(a, p.c0 + c);
                m1 += w * total[c].x;
                m2 += w * total[c].y;
            }
            m1 = gather(m1);
            m2 = gather(m2);
            if (lane == 0) { publish(a, p, all, groups, g0, k, make_double2(m1, m2)); }
        });
        if (a.walks == 1) { return; }
        if (cluster) {
            cluster_sync();
        } else {
            __syncthreads();
        }
    }
    // ---- of the slices together: total[group] = m1, m2
    for (int k = threadIdx.x; k < groups; k += blockDim.x) {
        double m1 = 0, m2 = 0;
        for (int i = 0; i < a.slices; ++i) {
            const double2 v = published(a, p, all, groups, g0, k, i);
            m1 += v.x;
            m2 += v.y;
        }
        total[k] = make_double2(m1 * a.per_value, m2 * a.per_value);
    }
    __syncthreads();
    // ---- results
    T *dx = static_cast<T *>(const_cast<void *>(a.dx.ptr)), *dr = static_cast<T *>(const_cast<void *>(a.dr.ptr));
    if (dx != nullptr) { dx += p.n * a.dx.image + p.c0; }
    if (dr != nullptr) { dr += p.n * a.dr.image + p.c0; }
    for (int pass = 0; pass < g.passes; ++pass) {
        const int col = g.column(pass);
        if (col >= g.columns || g.row() >= g.down) { continue; }
        const Factors<kCh> f = factors(col);
        float c1[kCh], c2[kCh];
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            const int k = (col * kCh + i) / a.per;
            const double rstd = stats[k].y;
            c1[i] = static_cast<float>(-rstd * total[k].x);
            c2[i] = static_cast<float>(-rstd * rstd * total[k].y);
        }
        const long long first = p.from + g.row();
        Walker<V> wo(dx != nullptr ? dx : dr, dx != nullptr ? a.dx.row : a.dr.row, first, col, kCh, g.down), wr = wo;
        if (dr != nullptr) { wr = Walker<V>(dr, a.dr.row, first, col, kCh, g.down); }
        const int rows = static_cast<int>(max(0ll, (p.to - first + g.down - 1) / g.down));
        wo.turn(rows);
        wr.turn(rows);
        const auto write = [&](const V &vx, const V &vr, const V &vd, int k) {
            float dz[kCh], off[kCh];
            grad_z<T, kCh, kAct, kResidual>(a, p, col, f, stats, vx, vr, vd, dz, off);
            V o;
            if (dr != nullptr) {
                o.set(dz);
                wr.store(k, o);
            }
            if (dx != nullptr) {
#pragma unroll
                for (int i = 0; i < kCh; ++i) { dz[i] = fmaf(f.scale[i], dz[i], fmaf(off[i], c2[i], c1[i])); }
                o.set(dz);
                wo.store(k, o);
            }
        };
        walk(col, true, write, [&](int k) {
            wo.next(k);
            wr.next(k);
        }, [] {});
    }
}

// dweight and dbias: the slices' sums, in their order (a warp's lanes take channels side by side, its warps every 32nd slice).
__global__ void __launch_bounds__(1024) params_kernel(const float *sums, long long slices, int channels, void *dweight, void *dbias, int dt)
{
    __shared__ double shares[2][32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    double db = 0, dw = 0;
    if (c < channels) {
#pragma unroll 4
        for (long long i = warp; i < slices; i += 32) {
            db += sums[2 * i * channels + c];
            dw += sums[(2 * i + 1) * channels + c];
        }
    }
    shares[0][lane][warp] = db;
    shares[1][lane][warp] = dw;
    __syncthreads();
    for (int which = 0; which < 2; ++which) {  // a warp adds up a channel
        const double sum = warp_sum(shares[which][warp][lane]);
        void *out = which == 0 ? dbias : dweight;
        const int of = blockIdx.x * 32 + warp;
        if (lane == 0 && out != nullptr && of < channels) { store_any(out, of, dt, static_cast<float>(sum)); }
    }
}
template <typename T, int kCh, int kAct>
void backward(const NormArgs &n, cudaStream_t s)
{
    const bool results = n.dx.ptr != nullptr || n.dr.ptr != nullptr;
    if constexpr (kAct != STDMLC_ACT_NONE) {
        if (n.r.ptr != nullptr) { return norm_walks(backward_kernel<T, kCh, kAct, true>, n, kCh, results, s); }
    }
    norm_walks(backward_kernel<T, kCh, kAct, false>, n, kCh, results, s);
}
}  // namespace

void norm_params_launch(const NormArgs &n, void *dweight, void *dbias, cudaStream_t s)
{
    params_kernel<<<static_cast<unsigned int>((n.channels + 31) / 32), 1024, 0, s>>>(n.param_sums, n.images * n.slices, n.channels, dweight,
                                                                                   dbias, n.weight_dt);
}

void norm_backward_launch(const NormArgs &n, int dt, int vector, int act, cudaStream_t s)
{
    by_dtype(dt, [&](auto t) {
        using T = decltype(t);
        by_act(act, [&](auto k) {
            constexpr int kAct = decltype(k)::value;
            if constexpr (kAct != STDMLC_ACT_GELU_TANH) {
                if (vector >= 4) {
                    backward<T, 4, kAct>(n, s);
                } else if (vector >= 2) {
                    backward<T, 2, kAct>(n, s);
                } else {
                    backward<T, 1, kAct>(n, s);
                }
            }
        });
    });
}
}  // namespace stdml::collective::train
