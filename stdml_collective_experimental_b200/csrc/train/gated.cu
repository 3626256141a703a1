// The gated projection of a feed-forward block, forward and backward:
//   g = x Wg^T + bg, u = x Wu^T + bu, h = act(g) * u
//   dg = dh * u * act'(g), du = dh * act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dbg = sum dg, dbu = sum du
#include "dispatch.cuh"
#include "host.hpp"

namespace stdml::collective::train
{
namespace
{
constexpr int kTile = 64, kStep = 16;

struct Operand {
    const void *ptr;
    long long row, col;  // element (i, k) at i * row + k * col
    int dt;
};

// acc[4][4] of one thread of 16 x 16: rows m0 + 4 ty.., columns n0 + 4 tx.. of A B^T.
__device__ __forceinline__ void tile_product(const Operand &a, const Operand &b, long long m0, long long n0,
                                             long long m, long long n, long long k, float (&acc)[4][4])
{
    __shared__ float sa[kStep][kTile + 1], sb[kStep][kTile + 1];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (long long k0 = 0; k0 < k; k0 += kStep) {
        __syncthreads();
        for (int e = threadIdx.x; e < kTile * kStep; e += 256) {
            const int i = e / kStep, j = e % kStep;
            sa[j][i] = m0 + i < m && k0 + j < k ? load_any(a.ptr, (m0 + i) * a.row + (k0 + j) * a.col, a.dt) : 0.f;
            sb[j][i] = n0 + i < n && k0 + j < k ? load_any(b.ptr, (n0 + i) * b.row + (k0 + j) * b.col, b.dt) : 0.f;
        }
        __syncthreads();
        for (int j = 0; j < kStep; ++j) {
            for (int p = 0; p < 4; ++p) {
                for (int q = 0; q < 4; ++q) { acc[p][q] += sa[j][4 * ty + p] * sb[j][4 * tx + q]; }
            }
        }
    }
}

template <int kAct>
__global__ void __launch_bounds__(256) forward_kernel(stdmlc_gated a)
{
    const long long m0 = static_cast<long long>(blockIdx.y) * kTile, n0 = static_cast<long long>(blockIdx.x) * kTile;
    float g[4][4] = {}, u[4][4] = {};
    const Operand x{a.x, a.x_row, 1, a.dt};
    tile_product(x, {a.w_gate, a.w_gate_row, 1, a.dt}, m0, n0, a.tokens, a.ffn, a.hidden, g);
    tile_product(x, {a.w_up, a.w_up_row, 1, a.dt}, m0, n0, a.tokens, a.ffn, a.hidden, u);
    for (int p = 0; p < 4; ++p) {
        for (int q = 0; q < 4; ++q) {
            const long long i = m0 + 4 * (threadIdx.x >> 4) + p, j = n0 + 4 * (threadIdx.x & 15) + q;
            if (i >= a.tokens || j >= a.ffn) { continue; }
            const float gv = g[p][q] + (a.b_gate != nullptr ? load_any(a.b_gate, j, a.dt) : 0.f);
            const float uv = u[p][q] + (a.b_up != nullptr ? load_any(a.b_up, j, a.dt) : 0.f);
            store_any(a.h, i * a.ffn + j, a.dt, act<kAct>(gv) * uv);
            if (a.saved != nullptr) {
                float *s = static_cast<float *>(a.saved);
                s[i * a.ffn + j] = gv;
                s[(a.tokens + i) * a.ffn + j] = uv;
            }
        }
    }
}

// dg, du in 32 bits, [2][tokens][ffn].
template <int kAct>
__global__ void gate_grad_kernel(stdmlc_gated a, float *d)
{
    const long long many = a.tokens * a.ffn, step = static_cast<long long>(gridDim.x) * blockDim.x;
    const float *s = static_cast<const float *>(a.saved);
    for (long long e = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; e < many; e += step) {
        const float dh = load_any(a.dh, e / a.ffn * a.dh_row + e % a.ffn, a.dt);
        d[e] = dh * s[many + e] * act_grad<kAct>(s[e]);
        d[many + e] = dh * act<kAct>(s[e]);
    }
}

__global__ void __launch_bounds__(256) product_kernel(Operand a, Operand b, Operand a2, Operand b2, void *out, long long m,
                                                      long long n, long long k, int dt)
{
    const long long m0 = static_cast<long long>(blockIdx.y) * kTile, n0 = static_cast<long long>(blockIdx.x) * kTile;
    float acc[4][4] = {};
    tile_product(a, b, m0, n0, m, n, k, acc);
    if (a2.ptr != nullptr) { tile_product(a2, b2, m0, n0, m, n, k, acc); }
    for (int p = 0; p < 4; ++p) {
        for (int q = 0; q < 4; ++q) {
            const long long i = m0 + 4 * (threadIdx.x >> 4) + p, j = n0 + 4 * (threadIdx.x & 15) + q;
            if (i < m && j < n) { store_any(out, i * n + j, dt, acc[p][q]); }
        }
    }
}

__global__ void column_sums_kernel(const float *d, long long tokens, long long ffn, void *out, int dt)
{
    const long long j = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    if (j >= ffn) { return; }
    double sum = 0;
    for (long long i = 0; i < tokens; ++i) { sum += d[i * ffn + j]; }
    store_any(out, j, dt, static_cast<float>(sum));
}

dim3 tiles(long long m, long long n)
{
    return dim3(static_cast<unsigned int>((n + kTile - 1) / kTile), static_cast<unsigned int>((m + kTile - 1) / kTile));
}

void check(const stdmlc_gated *a)
{
    require(a != nullptr, "gated_linear: null arguments");
    require(float_type(a->dt), "gated_linear: bf16, f16 or f32 expected");
    require(a->act >= STDMLC_ACT_SILU && a->act <= STDMLC_ACT_GELU_TANH, "gated_linear: unknown activation");
    require(a->tokens >= 0 && a->tokens <= (1ll << 22) && a->hidden > 0 && a->hidden <= (1ll << 22) && a->ffn > 0 &&
                a->ffn <= (1ll << 22),
            "gated_linear: sizes must lie between 1 and 2^22");
    require((a->b_gate == nullptr) == (a->b_up == nullptr), "gated_linear: both biases or none");
}
}  // namespace
}  // namespace stdml::collective::train

using namespace stdml::collective::train;

extern "C" long long stdmlc_gated_saved(const stdmlc_gated *a) { return a == nullptr ? -1 : 8 * a->tokens * a->ffn; }

extern "C" long long stdmlc_gated_workspace(const stdmlc_gated *a, int backward)
{
    return a == nullptr ? -1 : backward ? 8 * a->tokens * a->ffn : 0;
}

extern "C" int stdmlc_gated_forward(const stdmlc_gated *a, int device, void *stream)
{
    return entry(device, [&] {
        check(a);
        if (a->tokens == 0) { return; }
        by_act(a->act, [&](auto k) {
            forward_kernel<decltype(k)::value>
                <<<tiles(a->tokens, a->ffn), 256, 0, static_cast<cudaStream_t>(stream)>>>(*a);
        });
    });
}

extern "C" int stdmlc_gated_backward(const stdmlc_gated *a, int device, void *stream)
{
    return entry(device, [&] {
        check(a);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        float *dg = static_cast<float *>(a->workspace), *du = dg + a->tokens * a->ffn;
        const long long m = a->tokens, f = a->ffn, k = a->hidden;
        if (m > 0) {
            by_act(a->act, [&](auto act) { gate_grad_kernel<decltype(act)::value><<<1024, 256, 0, s>>>(*a, dg); });
        }
        if (a->dx != nullptr && m > 0) {
            product_kernel<<<tiles(m, k), 256, 0, s>>>({dg, f, 1, kF32}, {a->w_gate, 1, a->w_gate_row, a->dt}, {du, f, 1, kF32},
                                                       {a->w_up, 1, a->w_up_row, a->dt}, a->dx, m, k, f, a->dt);
        }
        const Operand none{}, x{a->x, 1, a->x_row, a->dt};
        if (a->dw_gate != nullptr) {
            product_kernel<<<tiles(f, k), 256, 0, s>>>({dg, 1, f, kF32}, x, none, none, a->dw_gate, f, k, m, a->dt);
        }
        if (a->dw_up != nullptr) {
            product_kernel<<<tiles(f, k), 256, 0, s>>>({du, 1, f, kF32}, x, none, none, a->dw_up, f, k, m, a->dt);
        }
        const unsigned int blocks = static_cast<unsigned int>((f + 255) / 256);
        if (a->db_gate != nullptr) { column_sums_kernel<<<blocks, 256, 0, s>>>(dg, m, f, a->db_gate, a->dt); }
        if (a->db_up != nullptr) { column_sums_kernel<<<blocks, 256, 0, s>>>(du, m, f, a->db_up, a->dt); }
    });
}
