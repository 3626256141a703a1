// Group normalisation, forward: see norm.cuh.
#include "norm.cuh"

namespace stdml::collective::train
{
namespace
{
constexpr int kAhead = 4;  // rows that a thread has on their way

template <typename T, int kCh, int kAct>
__global__ void __launch_bounds__(kNormThreads, 2) forward_kernel(NormArgs a)
{
    extern __shared__ __align__(16) unsigned char raw[];
    using V = Vec<T, kCh>;
    const Part p(a);
    const Grid<kCh> g(p.width);
    float2 *lines = reinterpret_cast<float2 *>(raw);
    double2 *total = reinterpret_cast<double2 *>(lines + kNormThreads * kCh), *group = total + a.width;
    const int groups = p.width / a.per, g0 = p.c0 / a.per;
    const long long count = p.to - p.from;
    const T *x = static_cast<const T *>(a.x.ptr) + p.n * a.x.image + p.c0;

    if ((a.walks & 1) != 0) {
        // ---- sums of x less the slice's first value of the channel, and of their squares
        for (int pass = 0; pass < g.passes; ++pass) {
            const int col = g.column(pass);
            float s1[kCh] = {}, s2[kCh] = {};
            if (col < g.columns && g.row() < g.down && count > 0) {
                const V base = *reinterpret_cast<const V *>(x + p.from * a.x.row + col * kCh);
                long long s = p.from + g.row();
                for (; s + (kAhead - 1) * g.down < p.to; s += kAhead * g.down) {
                    V v[kAhead];
#pragma unroll
                    for (int k = 0; k < kAhead; ++k) { v[k] = *reinterpret_cast<const V *>(x + (s + k * g.down) * a.x.row + col * kCh); }
#pragma unroll
                    for (int k = 0; k < kAhead; ++k) {
#pragma unroll
                        for (int i = 0; i < kCh; ++i) {
                            const float d = v[k].at(i) - base.at(i);
                            s1[i] += d;
                            s2[i] += d * d;
                        }
                    }
                }
                for (; s < p.to; s += g.down) {
                    const V v = *reinterpret_cast<const V *>(x + s * a.x.row + col * kCh);
#pragma unroll
                    for (int i = 0; i < kCh; ++i) {
                        const float d = v.at(i) - base.at(i);
                        s1[i] += d;
                        s2[i] += d * d;
                    }
                }
            }
            column_sums<kCh>(g, pass, p.width, s1, s2, lines, total);
        }
        __syncthreads();
        // ---- mean and sum of squared deviations of each group in the slice
        for (int k = threadIdx.x; k < groups; k += blockDim.x) {
            double mean = 0, dev = 0;
            if (count > 0) {
                for (int c = 0; c < a.per; ++c) {
                    const double2 t = total[k * a.per + c];
                    mean += to_f32(x[p.from * a.x.row + k * a.per + c]) + t.x / count;
                }
                mean /= a.per;
                for (int c = 0; c < a.per; ++c) {
                    const double2 t = total[k * a.per + c];
                    const double off = to_f32(x[p.from * a.x.row + k * a.per + c]) + t.x / count - mean;
                    dev += t.y - t.x * t.x / count + off * off * count;
                }
            }
            group[k] = make_double2(mean, dev);
            if (a.walks == 1) {
                reinterpret_cast<double2 *>(a.sums)[(p.n * a.slices + p.slice) * a.groups + g0 + k] = group[k];
            }
        }
        if (a.walks == 1) { return; }
        if (a.slices > 1) {
            cluster_sync();
        } else {
            __syncthreads();
        }
    }
    // ---- of the slices together: total[group] = mean, 1 / deviation
    for (int k = threadIdx.x; k < groups; k += blockDim.x) {
        double mean = 0, dev = 0;
        const double2 *in_memory = reinterpret_cast<const double2 *>(a.sums) + p.n * a.slices * a.groups + g0 + k;
        const auto slice_of = [&](int i) {
            return a.walks == 2 ? in_memory[static_cast<long long>(i) * a.groups] : a.slices > 1 ? of_block(group + k, i) : group[k];
        };
        const auto rows_in = [&](int i) { return a.positions * (i + 1) / a.slices - a.positions * i / a.slices; };
        for (int i = 0; i < a.slices; ++i) { mean += slice_of(i).x * rows_in(i); }
        mean /= a.positions;
        for (int i = 0; i < a.slices; ++i) {
            const double2 v = slice_of(i);
            dev += v.y + (v.x - mean) * (v.x - mean) * rows_in(i) * a.per;
        }
        const double rstd = 1.0 / sqrt(dev / (static_cast<double>(a.positions) * a.per) + a.eps);
        total[k] = make_double2(mean, rstd);
        if (p.slice == 0) { reinterpret_cast<double2 *>(a.stats)[p.n * a.groups + g0 + k] = total[k]; }
    }
    __syncthreads();
    // ---- results
    const T *r = static_cast<const T *>(a.r.ptr);
    if (r != nullptr) { r += p.n * a.r.image + p.c0; }
    T *y = static_cast<T *>(const_cast<void *>(a.y.ptr)) + p.n * a.y.image + p.c0;
    for (int pass = 0; pass < g.passes; ++pass) {
        const int col = g.column(pass);
        if (col >= g.columns || g.row() >= g.down) { continue; }
        float scale[kCh], mean[kCh], bias[kCh];
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            const int c = col * kCh + i;
            const double2 st = total[c / a.per];
            mean[i] = static_cast<float>(st.x);
            scale[i] = static_cast<float>(st.y) * weight_of(a, p.c0 + c);
            bias[i] = bias_of(a, p.c0 + c);
        }
        const auto finish = [&](const V &v, const V &res, long long s) {
            float out[kCh];
#pragma unroll
            for (int i = 0; i < kCh; ++i) {
                const float add = r != nullptr ? res.at(i) : 0.f, z = (v.at(i) - mean[i]) * scale[i] + bias[i] + add;
                out[i] = act<T, kAct>(z);
            }
            V o;
            o.set(out);
            *reinterpret_cast<V *>(y + s * a.y.row + col * kCh) = o;
        };
        long long s = p.from + g.row();
        for (; s + (kAhead - 1) * g.down < p.to; s += kAhead * g.down) {
            V v[kAhead], res[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                v[k] = *reinterpret_cast<const V *>(x + (s + k * g.down) * a.x.row + col * kCh);
                if (r != nullptr) { res[k] = *reinterpret_cast<const V *>(r + (s + k * g.down) * a.r.row + col * kCh); }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) { finish(v[k], res[k], s + k * g.down); }
        }
        for (; s < p.to; s += g.down) {
            V res;
            if (r != nullptr) { res = *reinterpret_cast<const V *>(r + s * a.r.row + col * kCh); }
            finish(*reinterpret_cast<const V *>(x + s * a.x.row + col * kCh), res, s);
        }
    }
    if (a.walks == 3 && a.slices > 1) { cluster_sync(); }  // (nobody leaves while another reads its sums)
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
                    norm_walks(forward_kernel<T, kFull, kAct>, n, kFull, s);
                } else if (vector >= 2) {
                    norm_walks(forward_kernel<T, 2, kAct>, n, 2, s);
                } else {
                    norm_walks(forward_kernel<T, 1, kAct>, n, 1, s);
                }
            }
        });
    });
}
}  // namespace stdml::collective::train
