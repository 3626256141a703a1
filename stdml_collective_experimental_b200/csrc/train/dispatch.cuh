// From run-time types and activations to template arguments.
#pragma once
#include "math.cuh"

namespace stdml::collective::train
{
template <typename F>
void by_dtype(int dt, F f)
{
    switch (dt) {
    case kBf16:
        f(__nv_bfloat16{});
        break;
    case kF16:
        f(__half{});
        break;
    default:
        f(float{});
        break;
    }
}

template <int N>
struct Int {
    static constexpr int value = N;
};

template <typename F>
void by_act(int act, F f)
{
    switch (act) {
    case STDMLC_ACT_RELU:
        f(Int<STDMLC_ACT_RELU>{});
        break;
    case STDMLC_ACT_SILU:
        f(Int<STDMLC_ACT_SILU>{});
        break;
    case STDMLC_ACT_GELU:
        f(Int<STDMLC_ACT_GELU>{});
        break;
    case STDMLC_ACT_GELU_TANH:
        f(Int<STDMLC_ACT_GELU_TANH>{});
        break;
    default:
        f(Int<STDMLC_ACT_NONE>{});
        break;
    }
}
}  // namespace stdml::collective::train
