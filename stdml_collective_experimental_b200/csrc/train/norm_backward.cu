// Group normalisation, backward: see norm.cuh.
#include "norm.cuh"

namespace stdml::collective::train
{
namespace
{
constexpr int kAhead = 2;  // rows that a thread has on their way

// Factors of a thread's channels (four at most: with eight they would not leave room for two blocks on an SM).
template <int kCh>
struct Factors {
    float mean[kCh], rstd[kCh], scale[kCh], bias[kCh];
};

// dz of a thread's channels in a row, and (x - mean).
template <typename T, int kCh, int kAct>
__device__ __forceinline__ void grad_z(const NormArgs &a, const Part &p, int col, const Factors<kCh> &f, const double2 *stats,
                                       const Vec<T, kCh> &x, const Vec<T, kCh> &r, const Vec<T, kCh> &dy, float (&dz)[kCh], float (&off)[kCh])
{
#pragma unroll
    for (int i = 0; i < kCh; ++i) {
        off[i] = x.at(i) - f.mean[i];
        dz[i] = dy.at(i);
        if constexpr (kAct != STDMLC_ACT_NONE) {
            const float add = a.r.ptr != nullptr ? r.at(i) : 0.f;
            float z = off[i] * f.scale[i] + f.bias[i] + add;
            if constexpr (kAct == STDMLC_ACT_RELU) {
                // the derivative jumps at zero: a value that 32 bits leave in doubt is placed in 64
                if (fabsf(z) <= 1e-5f * ((fabsf(x.at(i)) + fabsf(f.mean[i])) * fabsf(f.scale[i]) + fabsf(f.bias[i]) + fabsf(add))) {
                    const int c = col * kCh + i;
                    const double2 st = stats[c / a.per];
                    z = static_cast<float>((x.at(i) - st.x) * st.y * weight_of(a, p.c0 + c) + f.bias[i] + add);
                }
            }
            dz[i] *= act_grad<T, kAct>(z);
        }
    }
}

template <typename T, int kCh, int kAct>
__global__ void __launch_bounds__(kNormThreads, 2) backward_kernel(NormArgs a)
{
    extern __shared__ __align__(16) unsigned char raw[];
    using V = Vec<T, kCh>;
    const Part p(a);
    const Grid<kCh> g(p.width);
    float2 *lines = reinterpret_cast<float2 *>(raw);
    double2 *total = reinterpret_cast<double2 *>(lines + kNormThreads * kCh), *group = total + a.width;
    const int groups = p.width / a.per, g0 = p.c0 / a.per;
    const double2 *stats = reinterpret_cast<const double2 *>(a.stats) + p.n * a.groups + g0;
    const T *x = static_cast<const T *>(a.x.ptr) + p.n * a.x.image + p.c0, *dy = static_cast<const T *>(a.dy.ptr) + p.n * a.dy.image + p.c0;
    const T *r = static_cast<const T *>(a.r.ptr);
    if (r != nullptr) { r += p.n * a.r.image + p.c0; }

    const auto factors = [&](int col) {
        Factors<kCh> f;
#pragma unroll
        for (int i = 0; i < kCh; ++i) {
            const int c = col * kCh + i;
            const double2 st = stats[c / a.per];
            f.mean[i] = static_cast<float>(st.x);
            f.rstd[i] = static_cast<float>(st.y);
            f.scale[i] = static_cast<float>(st.y) * weight_of(a, p.c0 + c);
            f.bias[i] = bias_of(a, p.c0 + c);
        }
        return f;
    };
    // All rows of a thread's: what(row, x, residual, dy).
    const auto walk = [&](int col, auto what) {
        const auto load = [&](long long s, V &vx, V &vr, V &vd) {
            vx = *reinterpret_cast<const V *>(x + s * a.x.row + col * kCh);
            if (kAct != STDMLC_ACT_NONE && r != nullptr) { vr = *reinterpret_cast<const V *>(r + s * a.r.row + col * kCh); }
            vd = *reinterpret_cast<const V *>(dy + s * a.dy.row + col * kCh);
        };
        long long s = p.from + g.row();
        for (; s + (kAhead - 1) * g.down < p.to; s += kAhead * g.down) {
            V vx[kAhead], vr[kAhead], vd[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) { load(s + k * g.down, vx[k], vr[k], vd[k]); }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) { what(s + k * g.down, vx[k], vr[k], vd[k]); }
        }
        for (; s < p.to; s += g.down) {
            V vx, vr, vd;
            load(s, vx, vr, vd);
            what(s, vx, vr, vd);
        }
    };

    if ((a.walks & 1) != 0) {
        // ---- sums of dz and of dz * xh
        for (int pass = 0; pass < g.passes; ++pass) {
            const int col = g.column(pass);
            float s1[kCh] = {}, s2[kCh] = {};
            if (col < g.columns && g.row() < g.down) {
                const Factors<kCh> f = factors(col);
                walk(col, [&](long long, const V &vx, const V &vr, const V &vd) {
                    float dz[kCh], off[kCh];
                    grad_z<T, kCh, kAct>(a, p, col, f, stats, vx, vr, vd, dz, off);
#pragma unroll
                    for (int i = 0; i < kCh; ++i) {
                        s1[i] += dz[i];
                        s2[i] += dz[i] * (off[i] * f.rstd[i]);
                    }
                });
            }
            column_sums<kCh>(g, pass, p.width, s1, s2, lines, total);
        }
        __syncthreads();
        if (a.param_sums != nullptr) {
            float *out = a.param_sums + (p.n * a.slices + p.slice) * 2 * a.channels + p.c0;
            for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
                out[c] = static_cast<float>(total[c].x);
                out[a.channels + c] = static_cast<float>(total[c].y);
            }
        }
        if (a.dx.ptr == nullptr && a.dr.ptr == nullptr) { return; }  // (all blocks)
        for (int k = threadIdx.x; k < groups; k += blockDim.x) {
            double m1 = 0, m2 = 0;
            for (int c = k * a.per; c < (k + 1) * a.per; ++c) {
                const double w = weight_of(a, p.c0 + c);
                m1 += w * total[c].x;
                m2 += w * total[c].y;
            }
            group[k] = make_double2(m1, m2);
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
    // ---- of the slices together: total[group] = m1, m2
    const double many = static_cast<double>(a.positions) * a.per;
    for (int k = threadIdx.x; k < groups; k += blockDim.x) {
        double m1 = 0, m2 = 0;
        const double2 *in_memory = reinterpret_cast<const double2 *>(a.sums) + p.n * a.slices * a.groups + g0 + k;
        for (int i = 0; i < a.slices; ++i) {
            const double2 v = a.walks == 2 ? in_memory[static_cast<long long>(i) * a.groups]
                              : a.slices > 1 ? of_block(group + k, i) : group[k];
            m1 += v.x;
            m2 += v.y;
        }
        total[k] = make_double2(m1 / many, m2 / many);
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
            const double2 m = total[(col * kCh + i) / a.per];
            c1[i] = f.rstd[i] * static_cast<float>(m.x);
            c2[i] = f.rstd[i] * f.rstd[i] * static_cast<float>(m.y);
        }
        walk(col, [&](long long s, const V &vx, const V &vr, const V &vd) {
            float dz[kCh], off[kCh];
            grad_z<T, kCh, kAct>(a, p, col, f, stats, vx, vr, vd, dz, off);
            V o;
            if (dr != nullptr) {
                o.set(dz);
                *reinterpret_cast<V *>(dr + s * a.dr.row + col * kCh) = o;
            }
            if (dx != nullptr) {
#pragma unroll
                for (int i = 0; i < kCh; ++i) { dz[i] = f.scale[i] * dz[i] - c1[i] - off[i] * c2[i]; }
                o.set(dz);
                *reinterpret_cast<V *>(dx + s * a.dx.row + col * kCh) = o;
            }
        });
    }
    if (a.walks == 3 && a.slices > 1) { cluster_sync(); }  // (nobody leaves while another reads its sums)
}

// dweight and dbias: the slices' sums, in their order.
__global__ void __launch_bounds__(256) params_kernel(const float *sums, long long slices, int channels, void *dweight, void *dbias, int dt)
{
    __shared__ double shares[2][8][32];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
    double db = 0, dw = 0;
    if (c < channels) {
        for (long long i = lane; i < slices; i += 8) {
            db += sums[2 * i * channels + c];
            dw += sums[(2 * i + 1) * channels + c];
        }
    }
    shares[0][lane][threadIdx.x & 31] = db;
    shares[1][lane][threadIdx.x & 31] = dw;
    __syncthreads();
    if (lane > 1 || c >= channels) { return; }
    double sum = 0;
    for (int i = 0; i < 8; ++i) { sum += shares[lane][i][threadIdx.x & 31]; }
    void *out = lane == 0 ? dbias : dweight;
    if (out != nullptr) { store_any(out, c, dt, static_cast<float>(sum)); }
}
}  // namespace

void norm_params_launch(const NormArgs &n, void *dweight, void *dbias, cudaStream_t s)
{
    params_kernel<<<static_cast<unsigned int>((n.channels + 31) / 32), 256, 0, s>>>(n.param_sums, n.images * n.slices, n.channels, dweight,
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
                    norm_walks(backward_kernel<T, 4, kAct>, n, 4, s);
                } else if (vector >= 2) {
                    norm_walks(backward_kernel<T, 2, kAct>, n, 2, s);
                } else {
                    norm_walks(backward_kernel<T, 1, kAct>, n, 1, s);
                }
            }
        });
    });
}
}  // namespace stdml::collective::train
