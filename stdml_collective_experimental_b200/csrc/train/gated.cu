// The gated projection of a feed-forward block, forward and backward:
//   g = x Wg^T + bg, u = x Wu^T + bu, h = act(g) * u
//   dg = dh * u * act'(g), du = dh * act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dbg = sum dg, dbu = sum du
//
// All five products run on the tensor cores (product.cuh), whose operands are 16-bit.  A tile of the forward
// product holds 128 columns of g beside the same 128 of u, so that the activation and the product are
// its epilogue.  32-bit operands are cut into three bf16 pieces of 8 bits each, which together are
// the operand, and the six products of pieces that reach 2^-24 are summed.
#include <algorithm>
#include <mutex>

#include "dispatch.cuh"
#include "host.hpp"
#include "product.cuh"

namespace stdml::collective::train
{
namespace
{
__device__ unsigned int g_status, g_taken;

// Asked and cleared in one step, so that nothing is lost that is reported meanwhile.
__global__ void take_status_kernel() { g_taken = atomicExch(&g_status, 0u); }

// ------------------------------------------------------------ what the backward pass needs of g and u
// Blocks of some columns of a row, both values together.  16-bit types: 24 bits of each, the upper 16 and the next 8
// apart (16 bits would put two more roundings as large as a result's own into every gradient; 32 would cost a
// third more bytes).  They are cut, not rounded: less by 2^-15 at most, 1/16 of half a step of f16 and 1/128 of bf16, which no gradient
// shows.  32-bit types: all of them.
template <typename T>
struct Saved {
    static constexpr int kCols = 16;
    static constexpr int kBytes = sizeof(T) == 4 ? 128 : 96;  // g, u in 32 bits | upper g, upper u, lower g, lower u
    __host__ __device__ static long long row_bytes(long long ffn) { return (ffn + kCols - 1) / kCols * kBytes; }
};

// ------------------------------------------------------------ the range of dg and du
// dg and du are rounded to the operands' type for the tensor cores, half a step of it each: an error of the size of a result's own rounding, and not
// more in sums of them, where it is of either sign.  (As two 16-bit pieces each they would take the gradients' products twice.)  In f16 they would
// also overflow where dh u does, and vanish where a sum over many tokens does not: they are multiplied by a power of two that
// puts the largest at 2^14, which the results are divided by in 32 bits.  So values down to 2^-28 of the largest keep all their bits.
__device__ __forceinline__ int scale_exponent(unsigned int most)  // of what `most`, the bits of a float, is multiplied by
{
    return most == 0u ? 0 : min(126, 14 - (static_cast<int>(most >> 23) - 127));
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<unsigned int>(e + 127) << 23); }

// ------------------------------------------------------------ results of a tile
// An epilogue warp has 32 rows of a tile, one to a thread; through 32 rows of 128 bytes in shared memory they reach
// global memory 32 bytes and more in a row (stores of 16 bytes from 32 rows at a time took longer than the products).
// Pieces of 16 bytes lie swizzled, so that neither side meets bank conflicts.
__device__ __forceinline__ uint4 *piece_at(unsigned char *mem, int row, int piece)
{
    return reinterpret_cast<uint4 *>(mem + 128 * row + 16 * (piece ^ (row & 7)));
}

template <typename T>
__device__ __forceinline__ void put16(unsigned char *mem, int row, int piece, const float (&v)[16])
{
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 16 / kPer; ++j) { *piece_at(mem, row, piece + j) = pack16<T>(v + kPer * j); }
}

// Where kPieces pieces of each of 32 rows go, 32 / kPieces rows at a time: to + r * pitch + 16 * piece.
template <int kPieces>
struct RowsOut {
    unsigned char *to;  // this thread's first piece
    long long step;     // from one of its rows to the next
    int left;           // rows of this thread's row and those below

    __device__ __forceinline__ RowsOut(void *base, long long pitch, int row0, int m)
    {
        const int r = (threadIdx.x & 31) / kPieces;
        to = static_cast<unsigned char *>(base) + (row0 + r) * pitch + 16 * (threadIdx.x % kPieces);
        step = 32 / kPieces * pitch;
        left = m - row0 - r;
    }
    // From pieces `first` on in shared memory, `bytes` further on in each row.
    __device__ __forceinline__ void copy(unsigned char *mem, int first, long long bytes) const
    {
        const int r = (threadIdx.x & 31) / kPieces, q = threadIdx.x % kPieces;
        unsigned char *at = to + bytes;
#pragma unroll
        for (int k = 0; k < kPieces; ++k, at += step) {
            if (32 / kPieces * k < left) { *reinterpret_cast<uint4 *>(at) = *piece_at(mem, r + 32 / kPieces * k, first + q); }
        }
    }
};

// The same for rows at any address, element by element: columns [col, col + kBytes / sizeof(T)) of a result of n.
template <typename T, int kBytes>
__device__ __noinline__ void rows_out_any(unsigned char *mem, T *out, int row0, int m, long long n, long long col)
{
    constexpr int kWords = kBytes / 4;
    for (int i = threadIdx.x & 31; i < 32 * kWords; i += 32) {
        const int r = i / kWords, q = i % kWords;
        const long long c = col + q * static_cast<int>(4 / sizeof(T));
        if (row0 + r >= m || c >= n) { continue; }
        const uint32_t word = reinterpret_cast<const uint32_t *>(piece_at(mem, r, q / 4))[q % 4];
        T *to = out + (row0 + r) * n + c;
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<uint32_t *>(to) = word;
        } else if (c + 1 < n && reinterpret_cast<uintptr_t>(to) % 4 == 0) {
            *reinterpret_cast<uint32_t *>(to) = word;
        } else {
            reinterpret_cast<uint16_t *>(to)[0] = static_cast<uint16_t>(word);
            if (c + 1 < n) { reinterpret_cast<uint16_t *>(to)[1] = static_cast<uint16_t>(word >> 16); }
        }
    }
}

// g and u of the same columns side by side in a tile: h, and what the backward pass needs of them.
template <typename T, int kAct>
struct GatedTile {
    T *h;
    const T *b_gate, *b_up;
    unsigned char *saved;
    bool vec_h, vec_b;

    __device__ __forceinline__ void add_bias(const T *bias, long long col, int n, float (&v)[16]) const
    {
        if (vec_b && col + 16 <= n) {
            constexpr int kPer = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < 16 / kPer; ++j) {
                float t[kPer];
                unpack16<T>(reinterpret_cast<const uint4 *>(bias + col)[j], t);
#pragma unroll
                for (int i = 0; i < kPer; ++i) { v[kPer * j + i] += t[i]; }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) { v[i] += col + i < n ? to_f32(bias[col + i]) : 0.f; }
        }
    }
    // The upper 16 bits of 16 values into two pieces, the next 8 into one.
    __device__ __forceinline__ static void keep24(unsigned char *mem, int row, int upper, int lower, const float (&v)[16])
    {
        uint32_t up[8], low[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            up[i] = __byte_perm(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), 0x7632);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t a = __byte_perm(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), 0x0051),
                           b = __byte_perm(__float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]), 0x0051);
            low[i] = __byte_perm(a, b, 0x5410);
        }
        *piece_at(mem, row, upper) = make_uint4(up[0], up[1], up[2], up[3]);
        *piece_at(mem, row, upper + 1) = make_uint4(up[4], up[5], up[6], up[7]);
        *piece_at(mem, row, lower) = make_uint4(low[0], low[1], low[2], low[3]);
    }

    template <int kN, typename Source>
    __device__ __forceinline__ void tile(const Product &p, int, int row0, int nt, int, int slice, unsigned char *mem,
                                         const Source &from) const
    {
        constexpr int kCols = Saved<T>::kCols, kPasses = Shape<kN, false>::kBlocks / 2, kPieces = sizeof(T);
        const int lane = threadIdx.x & 31;
        const long long first = nt * (kN / 2ll) + kPasses * kCols * slice;
        const RowsOut<kPieces> rows_h(h + first, p.n * static_cast<long long>(sizeof(T)), row0, p.m);
        const RowsOut<kPieces> rows_s(saved + first / kCols * Saved<T>::kBytes, Saved<T>::row_bytes(p.n), row0, p.m);
        const int passes = static_cast<int>(min(static_cast<long long>(kPasses), (p.n - first + kCols - 1) / kCols));
        if (passes <= 0) { from.done(); }
#pragma unroll 1
        for (int b = 0; b < passes; ++b) {
            const long long col = first + kCols * b;
            float g[16], u[16];
            from.load(b, g);
            from.load(kPasses + b, u);
            from.loaded(g);
            from.loaded(u);
            if (b == passes - 1) { from.done(); }
            if (b_gate != nullptr) {
                add_bias(b_gate, col, p.n, g);
                add_bias(b_up, col, p.n, u);
            }
            if (saved != nullptr) {
                if constexpr (sizeof(T) == 4) {
                    put16<T>(mem, lane, 0, g);
                    put16<T>(mem, lane, 4, u);
                } else {
                    keep24(mem, lane, 2, 6, g);
                    keep24(mem, lane, 4, 7, u);
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < Saved<T>::kBytes / (16 * kPieces); ++j) {
                    rows_s.copy(mem, (sizeof(T) == 4 ? 0 : 2) + kPieces * j, Saved<T>::kBytes * b + 16 * kPieces * j);
                }
                if constexpr (sizeof(T) == 4) { __syncwarp(); }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) { u[i] *= act<T, kAct>(g[i]); }
            put16<T>(mem, lane, 0, u);
            __syncwarp();
            if (vec_h && col + kCols <= p.n) {
                rows_h.copy(mem, 0, kCols * static_cast<int>(sizeof(T)) * b);
            } else {
                rows_out_any<T, kCols * sizeof(T)>(mem, h, row0, p.m, p.n, col);
            }
            __syncwarp();
        }
    }
};

template <typename T>
struct PlainTile {
    T *out[2][2];  // [product][z]
    const unsigned int *most;  // f16: what dg and du were scaled by
    bool vec;

    template <int kN, typename Source>
    __device__ __forceinline__ void tile(const Product &p, int product, int row0, int nt, int z, int slice, unsigned char *mem,
                                         const Source &from) const
    {
        constexpr int kCols = Shape<kN, false>::kValues, kBytes = kCols * static_cast<int>(sizeof(T));
        static_assert(kBytes <= 128, "one row in shared memory");
        T *to = product == 0 ? (z == 0 ? out[0][0] : out[0][1]) : (z == 0 ? out[1][0] : out[1][1]);
        const long long first = nt * static_cast<long long>(kN) + kCols * slice;
        if (first >= p.n) {
            from.done();
            return;
        }
        const float by = std::is_same_v<T, __half> ? power_of_two(-scale_exponent(__ldg(most))) : 1.f;
#pragma unroll
        for (int b = 0; b < kCols / 16; ++b) {
            float v[16];
            from.load(b, v);
            from.loaded(v);
            if constexpr (std::is_same_v<T, __half>) {
#pragma unroll
                for (int i = 0; i < 16; ++i) { v[i] *= by; }
            }
            put16<T>(mem, threadIdx.x & 31, b * static_cast<int>(sizeof(T)), v);
        }
        from.done();
        __syncwarp();
        if (vec && first + kCols <= p.n) {
            RowsOut<kBytes / 16>(to + first, p.n * static_cast<long long>(sizeof(T)), row0, p.m).copy(mem, 0, 0);
        } else {
            rows_out_any<T, kBytes>(mem, to, row0, p.m, p.n, first);
        }
        __syncwarp();
    }
};

// ------------------------------------------------------------ operands of the tensor cores
// v as the sum of three bf16 numbers of 8 bits each, largest first (what is not finite in the first alone).
__device__ __forceinline__ void cut(float v, uint16_t (&piece)[kPieces])
{
    const uint32_t b = __float_as_uint(v), top = b & 0xFFFF0000u;
    if ((b & 0x7F800000u) == 0x7F800000u) {
        piece[0] = static_cast<uint16_t>((b >> 16) | ((b & 0x7FFFFFu) != 0u ? 0x40u : 0u));
        piece[1] = piece[2] = 0;
        return;
    }
    const float rest = v - __uint_as_float(top);
    const uint32_t mid = __float_as_uint(rest) & 0xFFFF0000u;
    const uint32_t low = __float_as_uint(rest - __uint_as_float(mid));
    piece[0] = static_cast<uint16_t>(top >> 16);
    piece[1] = static_cast<uint16_t>(mid >> 16);
    piece[2] = static_cast<uint16_t>(low >> 16);
}

// Rows of a pitch that TMA takes; 32-bit values as pieces: [pieces][rows][pitch].  A thread takes eight columns (all of them
// are written, up to the pitch), blockIdx.y an operand.
struct Packed {
    const void *from;
    long long row, rows, cols, pitch;
    uint16_t *to;
    bool vec;
};
struct Packs {
    Packed of[3];
};

template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Packs packs)
{
    const Packed &p = packs.of[blockIdx.y];
    const int across = static_cast<int>((p.pitch + 7) / 8);
    const long long many = p.rows * across, step = static_cast<long long>(gridDim.x) * 256;
    for (long long e = blockIdx.x * 256ll + threadIdx.x; e < many; e += step) {
        const long long r = many < (1ll << 31) ? static_cast<unsigned int>(e) / static_cast<unsigned int>(across) : e / across;
        const long long c = (e - r * across) * 8;
        const T *from = static_cast<const T *>(p.from) + r * p.row + c;
        uint16_t *to = p.to + r * p.pitch + c;
        if constexpr (sizeof(T) == 4) {
            float v[8];
            if (p.vec && c + 8 <= p.cols) {
                reinterpret_cast<float4 *>(v)[0] = reinterpret_cast<const float4 *>(from)[0];
                reinterpret_cast<float4 *>(v)[1] = reinterpret_cast<const float4 *>(from)[1];
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) { v[i] = c + i < p.cols ? from[i] : 0.f; }
            }
            __align__(16) uint16_t out[kPieces][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint16_t piece[kPieces];
                cut(v[i], piece);
#pragma unroll
                for (int k = 0; k < kPieces; ++k) { out[k][i] = piece[k]; }
            }
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                *reinterpret_cast<uint4 *>(to + k * p.rows * p.pitch) = *reinterpret_cast<const uint4 *>(out[k]);
            }
        } else {
            __align__(16) uint16_t out[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) { out[i] = c + i < p.cols ? reinterpret_cast<const uint16_t *>(from)[i] : 0; }
            *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(out);
        }
    }
}

// ------------------------------------------------------------ dg and du
constexpr int kGradRows = 64, kGradCols = 256;  // of a block: 8 rows of 32 threads with 8 columns each

struct GateGrad {
    const void *dh;
    long long dh_row;
    const unsigned char *saved;
    long long tokens, ffn, pitch;
    uint16_t *d;      // [gate, up][pieces][tokens][pitch]
    float *partial;   // [row blocks][gate, up][ffn]; null: no sums
    unsigned int *most;  // f16: bits of a bound of |dg| and |du|
    bool vec;
};

// 8 columns of a row of dh, and the saved g and u.
template <typename T>
struct GateGradRow {
    __align__(16) T dh[8];
    __align__(16) uint32_t g[sizeof(T) == 4 ? 8 : 4], u[sizeof(T) == 4 ? 8 : 4];
    uint2 low_g, low_u;

    __device__ __forceinline__ void load(const GateGrad &a, long long r, long long col)
    {
        const T *from = static_cast<const T *>(a.dh) + r * a.dh_row + col;
        if (a.vec) {  // (and so ffn is a multiple of 16 bytes)
#pragma unroll
            for (int i = 0; i < static_cast<int>(8 * sizeof(T) / 16); ++i) {
                const bool in = col + (i + 1) * static_cast<int>(16 / sizeof(T)) <= a.ffn;
                reinterpret_cast<uint4 *>(dh)[i] = in ? reinterpret_cast<const uint4 *>(from)[i] : make_uint4(0, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) { dh[i] = col + i < a.ffn ? from[i] : from_f32<T>(0.f); }
        }
        constexpr int kCols = Saved<T>::kCols;
        const unsigned char *s = a.saved + r * Saved<T>::row_bytes(a.ffn) + col / kCols * Saved<T>::kBytes;
        const int at = static_cast<int>(col % kCols);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                reinterpret_cast<uint4 *>(g)[i] = reinterpret_cast<const uint4 *>(s + 4 * at)[i];
                reinterpret_cast<uint4 *>(u)[i] = reinterpret_cast<const uint4 *>(s + 64 + 4 * at)[i];
            }
        } else {
            *reinterpret_cast<uint4 *>(g) = *reinterpret_cast<const uint4 *>(s + 2 * at);
            *reinterpret_cast<uint4 *>(u) = *reinterpret_cast<const uint4 *>(s + 32 + 2 * at);
            low_g = *reinterpret_cast<const uint2 *>(s + 64 + at);
            low_u = *reinterpret_cast<const uint2 *>(s + 80 + at);
        }
    }
    __device__ __forceinline__ static float value(const uint32_t *v, const uint2 &low, int i)
    {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(v[i]);
        } else {
            // bytes: 0, the next 8 bits, the upper 16
            const uint32_t lo = __byte_perm(i < 4 ? low.x : low.y, 0u, 0x4404 | ((i & 3) << 4));
            return __uint_as_float(__byte_perm(v[i / 2], lo, (i & 1) != 0 ? 0x3254 : 0x1054));
        }
    }
};

constexpr int kMostRows = 16;  // of a block (1037 x 2730: with 64 of them 8.4 us)

// a.most, which is zero: |act'| <= 1.13 and |act(g)| <= |g|.  What is not finite stays so, and bounds nothing.
template <typename T>
__global__ void __launch_bounds__(256) gate_most_kernel(GateGrad a)
{
    const int across = static_cast<int>((a.ffn + kGradCols - 1) / kGradCols), down = blockIdx.x / across;
    const long long col = (blockIdx.x - down * across) * static_cast<long long>(kGradCols) + 8 * (threadIdx.x & 31);
    const long long first = down * static_cast<long long>(kMostRows), end = min(first + kMostRows, a.tokens);
    float most = 0;
    if (col < a.ffn) {
#pragma unroll 2
        for (long long r = first + (threadIdx.x >> 5); r < end; r += 8) {
            GateGradRow<T> row;
            row.load(a, r, col);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float g = row.value(row.g, make_uint2(0, 0), i), u = row.value(row.u, make_uint2(0, 0), i);
                // (the upper bits alone: 1 % less at most)
                const float v = fabsf(to_f32(row.dh[i])) * fmaxf(1.15f * fabsf(u), 1.02f * fabsf(g));
                if (col + i < a.ffn && v > most && v < INFINITY) { most = v; }
            }
        }
    }
    most = warp_max(most);
    if ((threadIdx.x & 31) == 0 && most > 0.f) { atomicMax(a.most, __float_as_uint(most)); }
}

template <typename T, int kAct>
__global__ void __launch_bounds__(256) gate_grad_kernel(GateGrad a)
{
    const float scale = std::is_same_v<T, __half> ? power_of_two(scale_exponent(*a.most)) : 1.f;
    __shared__ float sums[2][8][kGradCols];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int across = static_cast<int>((a.ffn + kGradCols - 1) / kGradCols), down = blockIdx.x / across;
    const long long base = (blockIdx.x - down * across) * static_cast<long long>(kGradCols), col = base + 8 * tx;
    const long long first = down * static_cast<long long>(kGradRows);
    const long long end = min(first + kGradRows, a.tokens), slab = a.tokens * a.pitch;
    float sg[8] = {}, su[8] = {};
    if (col < a.ffn) {
        GateGradRow<T> row;
        if (first + ty < end) { row.load(a, first + ty, col); }
        for (long long r = first + ty; r < end; r += 8) {
            const GateGradRow<T> now = row;
            if (r + 8 < end) { row.load(a, r + 8, col); }
            constexpr int kSlabs = sizeof(T) == 4 ? kPieces : 1;
            __align__(16) uint16_t out[2][kSlabs][8];
            float both[2][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float dh = to_f32(now.dh[i]), g = now.value(now.g, now.low_g, i), u = now.value(now.u, now.low_u, i);
                float act, grad;
                act_both<T, kAct>(g, act, grad);
                const float dg = dh * u * grad, du = dh * act;
                if (col + i < a.ffn) {
                    sg[i] += dg;
                    su[i] += du;
                }
                if constexpr (sizeof(T) == 4) {
                    uint16_t piece[kPieces];
                    cut(dg, piece);
#pragma unroll
                    for (int j = 0; j < kPieces; ++j) { out[0][j][i] = piece[j]; }
                    cut(du, piece);
#pragma unroll
                    for (int j = 0; j < kPieces; ++j) { out[1][j][i] = piece[j]; }
                } else {
                    both[0][i] = std::is_same_v<T, __half> ? dg * scale : dg;
                    both[1][i] = std::is_same_v<T, __half> ? du * scale : du;
                }
            }
            if constexpr (sizeof(T) == 2) {
                *reinterpret_cast<uint4 *>(out[0][0]) = pack16<T>(both[0]);
                *reinterpret_cast<uint4 *>(out[1][0]) = pack16<T>(both[1]);
            }
            uint16_t *at = a.d + r * a.pitch + col;
#pragma unroll
            for (int z = 0; z < 2; ++z) {
#pragma unroll
                for (int j = 0; j < kSlabs; ++j) {
                    *reinterpret_cast<uint4 *>(at + (z * kSlabs + j) * slab) = *reinterpret_cast<const uint4 *>(out[z][j]);
                }
            }
        }
    }
    if (a.partial == nullptr) { return; }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        sums[0][ty][8 * tx + i] = sg[i];
        sums[1][ty][8 * tx + i] = su[i];
    }
    __syncthreads();
    const long long mine = base + threadIdx.x;
    if (mine >= a.ffn) { return; }
    for (int z = 0; z < 2; ++z) {
        float sum = 0;
        for (int i = 0; i < 8; ++i) { sum += sums[z][i][threadIdx.x]; }
        a.partial[(2ll * down + z) * a.ffn + mine] = sum;
    }
}

// The sums of all row blocks (blockIdx.y: gate, up).
__global__ void bias_sums_kernel(const float *partial, long long blocks, long long ffn, void *db_gate, void *db_up, int dt)
{
    void *out = blockIdx.y == 0 ? db_gate : db_up;
    const long long j = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x;
    if (out == nullptr || j >= ffn) { return; }
    double sum = 0;
    for (long long b = 0; b < blocks; ++b) { sum += partial[(2 * b + blockIdx.y) * ffn + j]; }
    store_any(out, j, dt, static_cast<float>(sum));
}

// ------------------------------------------------------------ few tokens
// The weights' way from memory is all that counts: a warp takes a row of both, for all tokens.
constexpr int kFewTokens = 4;

template <typename T, int kAct, int kTokens, bool kVec>
__global__ void __launch_bounds__(256) few_kernel(stdmlc_gated a)
{
    const long long f = blockIdx.x * 8ll + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (f >= a.ffn) { return; }
    const T *wg = static_cast<const T *>(a.w_gate) + f * a.w_gate_row, *wu = static_cast<const T *>(a.w_up) + f * a.w_up_row;
    const T *x = static_cast<const T *>(a.x);
    float g[kTokens] = {}, u[kTokens] = {};
    constexpr int kPer = kVec ? 16 / static_cast<int>(sizeof(T)) : 1;
    struct alignas(kVec ? 16 : sizeof(T)) Vec {
        T v[kPer];
    };
#pragma unroll 4
    for (long long k = lane * kPer; k < a.hidden; k += 32 * kPer) {
        const Vec vg = *reinterpret_cast<const Vec *>(wg + k), vu = *reinterpret_cast<const Vec *>(wu + k);
#pragma unroll
        for (int t = 0; t < kTokens; ++t) {
            const Vec vx = *reinterpret_cast<const Vec *>(x + t * a.x_row + k);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                g[t] += to_f32(vx.v[i]) * to_f32(vg.v[i]);
                u[t] += to_f32(vx.v[i]) * to_f32(vu.v[i]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
        g[t] = warp_sum(g[t]);
        u[t] = warp_sum(u[t]);
        if (lane != t) { continue; }
        if (a.b_gate != nullptr) {
            g[t] += to_f32(static_cast<const T *>(a.b_gate)[f]);
            u[t] += to_f32(static_cast<const T *>(a.b_up)[f]);
        }
        static_cast<T *>(a.h)[t * a.ffn + f] = from_f32<T>(u[t] * act<T, kAct>(g[t]));
        if (a.saved != nullptr) {
            constexpr int kCols = Saved<T>::kCols;
            unsigned char *s = static_cast<unsigned char *>(a.saved) + t * Saved<T>::row_bytes(a.ffn) + f / kCols * Saved<T>::kBytes;
            const int at = static_cast<int>(f % kCols);
            const uint32_t bg = __float_as_uint(g[t]), bu = __float_as_uint(u[t]);
            if constexpr (sizeof(T) == 4) {
                reinterpret_cast<uint32_t *>(s)[at] = bg;
                reinterpret_cast<uint32_t *>(s + 64)[at] = bu;
            } else {
                reinterpret_cast<uint16_t *>(s)[at] = static_cast<uint16_t>(bg >> 16);
                reinterpret_cast<uint16_t *>(s + 32)[at] = static_cast<uint16_t>(bu >> 16);
                s[64 + at] = static_cast<unsigned char>(bg >> 8);
                s[80 + at] = static_cast<unsigned char>(bu >> 8);
            }
        }
    }
}

// ------------------------------------------------------------ host side
using Encode = decltype(&cuTensorMapEncodeTiled);

Encode encoder()
{
    static const Encode fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            (void)cudaGetLastError();
            p = nullptr;
        }
        return reinterpret_cast<Encode>(p);
    }();
    if (fn == nullptr) { throw std::runtime_error("cuTensorMapEncodeTiled is not available"); }
    return fn;
}

constexpr long long up_to(long long n, long long multiple) { return (n + multiple - 1) / multiple * multiple; }

// A 16-bit matrix in slabs, as TMA reads it.
struct Matrix {
    const void *ptr;
    long long rows, cols, pitch, slabs;

    CUtensorMap map(CUtensorMapDataType type, int box_rows) const
    {
        CUtensorMap m;
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(slabs)};
        const cuuint64_t strides[2] = {static_cast<cuuint64_t>(2 * pitch), static_cast<cuuint64_t>(2 * pitch * rows)};
        const cuuint32_t box[3] = {kStepK, static_cast<cuuint32_t>(box_rows), 1}, steps[3] = {1, 1, 1};
        const CUresult r = encoder()(&m, type, 3, const_cast<void *>(ptr), dims, strides, box, steps,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) { throw std::runtime_error("gated_linear: tensor map refused: " + std::to_string(r)); }
        return m;
    }
};

// Memory of a workspace, handed out in order (256 bytes apart); without one it only counts.
class Bump
{
  public:
    explicit Bump(void *base) : base_(static_cast<char *>(base)) {}
    template <typename T>
    T *take(long long count)
    {
        T *p = reinterpret_cast<T *>(base_ + used_);
        used_ += up_to(count * static_cast<long long>(sizeof(T)), 256);
        return p;
    }
    long long used() const { return used_; }

  private:
    char *base_;
    long long used_ = 0;
};

int pieces_of(int dt) { return dt == kF32 ? kPieces : 1; }

// An operand as TMA can read it: where it lies, or in the workspace.
struct Operand {
    const void *from;
    long long row, rows, cols;
    int dt;
    Matrix as{};
    bool packed = false;

    Operand(const void *p, long long row_, long long rows_, long long cols_, int dt_, Bump &work)
        : from(p), row(row_), rows(rows_), cols(cols_), dt(dt_)
    {
        const bool fits = dt != kF32 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || (row % 8 == 0 && row >= cols));
        if (fits) {
            as = {p, rows, cols, rows == 1 ? up_to(cols, 8) : row, 1};
        } else {
            packed = true;
            const long long pitch = up_to(cols, 8);
            as = {work.take<uint16_t>(pieces_of(dt) * rows * pitch), rows, cols, pitch, pieces_of(dt)};
        }
    }
};

// Those of the operands that have to be, in one launch.
void pack(std::initializer_list<const Operand *> all, cudaStream_t s)
{
    Packs packs{};
    unsigned int count = 0;
    long long most = 0;
    int dt = kF32;
    for (const Operand *o : all) {
        if (!o->packed) { continue; }
        dt = o->dt;
        packs.of[count++] = {o->from, o->row, o->rows, o->cols, o->as.pitch, static_cast<uint16_t *>(const_cast<void *>(o->as.ptr)),
                             reinterpret_cast<uintptr_t>(o->from) % 16 == 0 && (o->row * element_size(o->dt)) % 16 == 0};
        most = std::max(most, o->rows * (o->as.pitch / 8));
    }
    if (count == 0) { return; }
    const unsigned int blocks = static_cast<unsigned int>(std::min((most + 255) / 256, 2048ll));
    by_dtype(dt, [&](auto t) { pack_kernel<decltype(t)><<<dim3(blocks, count), 256, 0, s>>>(packs); });
}

struct Operands {
    Bump work;
    Operand x, w_gate, w_up;

    explicit Operands(const stdmlc_gated *a)
        : work(a->workspace), x(a->x, a->x_row, a->tokens, a->hidden, a->dt, work),
          w_gate(a->w_gate, a->w_gate_row, a->ffn, a->hidden, a->dt, work),
          w_up(a->w_up, a->w_up_row, a->ffn, a->hidden, a->dt, work)
    {
    }
};

long long row_blocks(const stdmlc_gated *a) { return (a->tokens + kGradRows - 1) / kGradRows; }

unsigned int *status_word()
{
    void *p = nullptr;
    cuda_ok(cudaGetSymbolAddress(&p, g_status), "status word");
    return static_cast<unsigned int *>(p);
}

unsigned long long wait_limit(const stdmlc_gated *a)
{
    return a->wait_limit_ns == 0 ? 10ull * 1000 * 1000 * 1000 : a->wait_limit_ns < 0 ? 0 : static_cast<unsigned long long>(a->wait_limit_ns);
}

// Sizes of a product, without its operands.
Product sizes(long long m, long long n, long long reduction, int halves, int z, bool two_b)
{
    Product p{};
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(n);
    p.steps = static_cast<int>((reduction + kStepK - 1) / kStepK);
    p.halves = halves;
    p.z = z;
    p.two_b = two_b ? 1 : 0;
    p.m_tiles = static_cast<int>((m + kTileM * kCtas - 1) / (kTileM * kCtas));
    p.split = 1;
    return p;
}

int columns_of(const Product &p, int width)
{
    const int w = p.two_b != 0 ? width / 2 : width;
    return (p.n + w - 1) / w;
}

// How wide a launch's tiles are and into how many parts those of each product are cut.  C clusters take units in
// turn, so the launch lasts for
//   sum over rounds of C units of the longest of each.
// A unit lasts for its steps (one of a 256-wide tile takes 0.45 us, which is its way from the L2, and of a 128-wide one
// 0.75 of that, as its bytes; of 32-bit operands, six products, 1 us), or for the epilogue of the one before it, which runs beside it; the last epilogue runs alone.  The parts
// of a tile are written (kWrite steps' time), and read by the last (kRead for each).
int cut_tiles(Work &w, int clusters, bool wide)
{
    constexpr int kCuts[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32};
    constexpr double kStart = 1, kEpilogue = 6, kWrite = 4, kRead = 4;
    double least = 1e30;
    int best[3] = {256, 1, 1};
    for (int width : {256, 128}) {
        if (wide && width == 256) { continue; }
        const double step = wide ? 2.2 : width == 256 ? 1.0 : 0.75, area = width / 256.0;
        int most[2] = {1, 1};
        long long tiles[2] = {0, 0}, steps[2] = {0, 0};
        for (int q = 0; q < w.products; ++q) {
            const Product &p = w.product[q];
            tiles[q] = static_cast<long long>(p.m_tiles) * columns_of(p, width) * p.z;
            steps[q] = static_cast<long long>(p.steps) * p.halves;
            // (parts of 4 steps at least; memory for at most four parts for each cluster)
            if (tiles[q] <= 2 * clusters) {
                most[q] = static_cast<int>(std::clamp<long long>(4ll * clusters / tiles[q], 1, std::max(1ll, steps[q] / 4)));
            }
        }
        for (int s0 : kCuts) {
            for (int s1 : kCuts) {
                if (s0 > most[0] || s1 > most[1]) { break; }
                double main[2] = {0, 0}, after[2] = {0, 0};
                const int s[2] = {s0, s1};
                for (int q = 0; q < w.products; ++q) {
                    main[q] = step * steps[q] / s[q] + kStart;
                    after[q] = area * (s[q] > 1 || wide ? kWrite + kRead * s[q] + kEpilogue : kEpilogue);
                }
                const long long u0 = tiles[0] * s0, u1 = tiles[1] * s1;
                const long long rounds = (u0 + clusters - 1) / clusters, all = (u0 + u1 + clusters - 1) / clusters;
                const int mixed = u0 % clusters != 0 && u1 > 0 ? 1 : 0;
                const double unit[2] = {std::max(main[0], after[0]), std::max(main[1], after[1])};
                const double cost = (rounds - mixed) * unit[0] + mixed * std::max(unit[0], unit[1]) + (all - rounds) * unit[1] +
                                    (all > rounds ? after[1] : mixed != 0 ? std::max(after[0], after[1]) : after[0]);
                if (cost < least) {
                    least = cost;
                    best[0] = width;
                    best[1] = s0;
                    best[2] = s1;
                }
            }
        }
    }
    int parts = 0;
    w.units = 0;
    for (int q = 0, tile = 0; q < 2; ++q) {
        Product &p = w.product[q];
        p.first_unit = q < w.products ? w.units : 0x7fffffff;
        if (q >= w.products) { break; }
        p.n_tiles = columns_of(p, best[0]);
        p.split = best[1 + q];
        p.first_tile = tile;
        p.first_part = parts;
        const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles * p.z;
        require(w.units + tiles * p.split < (1ll << 23), "gated_linear: too large");
        tile += static_cast<int>(tiles);
        w.units += static_cast<int>(tiles) * p.split;
        if (p.split > 1) { parts += static_cast<int>(tiles) * p.split; }
    }
    w.own_part = parts;
    return best[0];
}

long long tiles_of(const Product &p) { return static_cast<long long>(p.m_tiles) * p.n_tiles * p.z; }

// Memory of a launch's own: parts and tickets (none where nothing is split), and words that begin as zero like them.
struct Scratch {
    long long tickets = 0, words;
    unsigned int *most;

    Scratch(Work &w, int clusters, int width, bool wide, Bump &work, int more = 0)
    {
        bool split = false;
        for (int q = 0; q < w.products; ++q) {
            tickets += tiles_of(w.product[q]) * kCtas * kEpilogueWarps;
            split = split || w.product[q].split > 1;
        }
        if (!split) { tickets = 0; }
        words = tickets + more;
        w.tickets = work.take<unsigned int>(words);
        most = w.tickets + tickets;
        w.parts = work.take<float>((w.own_part + (wide ? clusters : 0)) * (width == 256 ? Shape<256, false>::kPart : Shape<128, true>::kPart));
    }
    void clear(const Work &w, cudaStream_t s) const
    {
        if (words > 0) { cuda_ok(cudaMemsetAsync(w.tickets, 0, 4 * words, s), "cudaMemsetAsync"); }
    }
};

void set_kind(Product &p, int dt, int width)
{
    const uint32_t type = dt == kF16 ? 0u : 1u;
    p.kind = (1u << 4) | (type << 7) | (type << 10) | (p.across_a != 0 ? 1u << 15 : 0u) | (p.across_b != 0 ? 1u << 16 : 0u) |
             (static_cast<uint32_t>(width >> 3) << 17) | (static_cast<uint32_t>(kTileM * kCtas >> 4) << 24);
}

template <bool kWide, int kN, typename Epilogue>
void launch_as(const Work &w, const Epilogue &epilogue, int clusters, cudaStream_t s)
{
    auto kernel = product_kernel<kWide, kN, Epilogue>;
    constexpr int kSmem = Shape<kN, kWide>::kSmem;
    cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem), "shared memory");
    kernel<<<static_cast<unsigned int>(std::min(w.units, clusters) * kCtas), kProductThreads, kSmem, s>>>(w, epilogue);
}

// (32-bit operands take narrow tiles alone: their sums need the registers)
template <bool kWide, typename Epilogue>
void launch(const Work &w, const Epilogue &epilogue, int clusters, int width, cudaStream_t s)
{
    if constexpr (!kWide) {
        if (width == 256) { return launch_as<false, 256>(w, epilogue, clusters, s); }
    }
    launch_as<kWide, 128>(w, epilogue, clusters, s);
}

bool aligned_rows(const void *p, long long row, int dt)
{
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row * element_size(dt) % 16 == 0;
}

void check(const stdmlc_gated *a)
{
    require(a != nullptr, "gated_linear: null arguments");
    require(float_type(a->dt), "gated_linear: bf16, f16 or f32 expected");
    require(a->act >= STDMLC_ACT_SILU && a->act <= STDMLC_ACT_GELU_TANH, "gated_linear: unknown activation");
    require(a->tokens >= 0 && a->tokens <= (1ll << 22) && a->hidden > 0 && a->hidden <= (1ll << 20) && a->ffn > 0 &&
                a->ffn <= (1ll << 20),
            "gated_linear: at most 2^22 tokens, 2^20 hidden and 2^20 ffn");
    require((a->b_gate == nullptr) == (a->b_up == nullptr), "gated_linear: both biases or none");
    require(a->tokens == 0 || (a->x != nullptr && a->w_gate != nullptr && a->w_up != nullptr), "gated_linear: null operand");
}

CUtensorMapDataType map_type(int dt) { return dt == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; }

// 32-bit sums of pieces are added up in registers after so many steps (one; at two, gradients of 512 x 1024 x 2736 were 1.3e-6 off and not 2.9e-7, for 16 us of 207): the tensor cores cut what they add to a
// sum of its size, a step of 2^-24 each time, always towards zero.
constexpr int kWideChunk = 1;

template <typename F>
void by_gate(int act, F f)
{
    switch (act) {
    case STDMLC_ACT_SILU:
        f(Int<STDMLC_ACT_SILU>{});
        break;
    case STDMLC_ACT_GELU:
        f(Int<STDMLC_ACT_GELU>{});
        break;
    default:
        f(Int<STDMLC_ACT_GELU_TANH>{});
        break;
    }
}

struct Forward : Operands {
    int clusters = sm_count() / kCtas, width = 0;
    Work w{};
    Scratch scratch;

    explicit Forward(const stdmlc_gated *a) : Operands(a), scratch{plan(a), clusters, width, a->dt == kF32, work} {}

  private:
    Work &plan(const stdmlc_gated *a)
    {
        w.product[0] = sizes(a->tokens, a->ffn, a->hidden, 1, 1, true);
        w.products = 1;
        w.chunk = kWideChunk;
        width = cut_tiles(w, clusters, a->dt == kF32);
        return w;
    }
};

struct Backward : Operands {
    int clusters = sm_count() / kCtas, width = 0, dx = -1, dw = -1;
    Matrix d;
    float *partial;
    Work w{};
    Scratch scratch;

    explicit Backward(const stdmlc_gated *a) : Operands(a), d(grads(a)), partial(work.take<float>(2 * row_blocks(a) * a->ffn)),
          scratch{plan(a), clusters, width, a->dt == kF32, work, a->dt == kF16 ? 1 : 0}
    {
    }

  private:
    Matrix grads(const stdmlc_gated *a)
    {
        const long long pitch = up_to(a->ffn, 8);
        return {work.take<uint16_t>(2 * pieces_of(a->dt) * a->tokens * pitch), a->tokens, a->ffn, pitch, 2 * pieces_of(a->dt)};
    }
    Work &plan(const stdmlc_gated *a)
    {
        const int pieces = pieces_of(a->dt), z = (a->dw_gate != nullptr ? 1 : 0) + (a->dw_up != nullptr ? 1 : 0);
        Product px = sizes(a->tokens, a->hidden, a->ffn, 2, 1, false), pw = sizes(a->ffn, a->hidden, a->tokens, 1, z, false);
        px.half_slabs = pieces;
        px.across_b = 1;
        pw.z_slabs = pieces;
        pw.z_first = a->dw_gate != nullptr ? 0 : 1;
        pw.across_a = pw.across_b = 1;
        // (the longer units first: they run beside the shorter ones of the other product)
        const bool x_first = 2 * px.steps >= pw.steps;
        for (int turn = 0; turn < 2; ++turn) {
            const bool x = (turn == 0) == x_first;
            if (x && a->dx != nullptr) { w.product[dx = w.products++] = px; }
            if (!x && z > 0) { w.product[dw = w.products++] = pw; }
        }
        w.chunk = kWideChunk;
        if (w.products > 0) { width = cut_tiles(w, clusters, a->dt == kF32); }
        return w;
    }
};

template <typename T, int kTokens>
void few(const stdmlc_gated *a, cudaStream_t s)
{
    const bool vec = aligned_rows(a->x, a->tokens > 1 ? a->x_row : 8, a->dt) && aligned_rows(a->w_gate, a->w_gate_row, a->dt) &&
                     aligned_rows(a->w_up, a->w_up_row, a->dt) && a->hidden * sizeof(T) % 16 == 0;
    const unsigned int blocks = static_cast<unsigned int>((a->ffn + 7) / 8);
    by_gate(a->act, [&](auto k) {
        constexpr int kAct = decltype(k)::value;
        if (vec) {
            few_kernel<T, kAct, kTokens, true><<<blocks, 256, 0, s>>>(*a);
        } else {
            few_kernel<T, kAct, kTokens, false><<<blocks, 256, 0, s>>>(*a);
        }
    });
}

void forward(const stdmlc_gated *a, cudaStream_t s)
{
    if (a->tokens <= kFewTokens) {
        by_dtype(a->dt, [&](auto t) {
            using T = decltype(t);
            switch (a->tokens) {
            case 1:
                return few<T, 1>(a, s);
            case 2:
                return few<T, 2>(a, s);
            case 3:
                return few<T, 3>(a, s);
            default:
                return few<T, 4>(a, s);
            }
        });
        return;
    }
    Forward f(a);
    pack({&f.x, &f.w_gate, &f.w_up}, s);
    Product &p = f.w.product[0];
    p.a = f.x.as.map(map_type(a->dt), kTileM);
    p.b[0] = f.w_gate.as.map(map_type(a->dt), f.width / kCtas);
    p.b[1] = f.w_up.as.map(map_type(a->dt), f.width / kCtas);
    set_kind(p, a->dt, f.width);
    f.w.status = status_word();
    f.w.wait_ns = wait_limit(a);
    f.scratch.clear(f.w, s);
    by_dtype(a->dt, [&](auto t) {
        using T = decltype(t);
        by_gate(a->act, [&](auto k) {
            const GatedTile<T, decltype(k)::value> tile{
                static_cast<T *>(a->h),           static_cast<const T *>(a->b_gate),
                static_cast<const T *>(a->b_up),  static_cast<unsigned char *>(a->saved),
                aligned_rows(a->h, a->ffn, a->dt), aligned_rows(a->b_gate, 8, a->dt) && aligned_rows(a->b_up, 8, a->dt)};
            launch<sizeof(T) == 4>(f.w, tile, f.clusters, f.width, s);
        });
    });
}

void backward(const stdmlc_gated *a, cudaStream_t s)
{
    Backward b(a);
    const bool sums = a->db_gate != nullptr || a->db_up != nullptr;
    const GateGrad gg{a->dh, a->dh_row, static_cast<const unsigned char *>(a->saved), a->tokens, a->ffn, b.d.pitch,
                      static_cast<uint16_t *>(const_cast<void *>(b.d.ptr)), sums ? b.partial : nullptr, b.scratch.most,
                      aligned_rows(a->dh, a->dh_row, a->dt) && a->ffn * element_size(a->dt) % 16 == 0};
    const CUtensorMapDataType type = map_type(a->dt);
    b.scratch.clear(b.w, s);
    by_dtype(a->dt, [&](auto t) {
        using T = decltype(t);
        const long long across = (a->ffn + kGradCols - 1) / kGradCols, grid = across * row_blocks(a);
        if constexpr (std::is_same_v<T, __half>) {
            const long long down = (a->tokens + kMostRows - 1) / kMostRows;
            gate_most_kernel<T><<<static_cast<unsigned int>(across * down), 256, 0, s>>>(gg);
        }
        by_gate(a->act, [&](auto k) {
            gate_grad_kernel<T, decltype(k)::value><<<static_cast<unsigned int>(grid), 256, 0, s>>>(gg);
        });
        if (sums) {
            bias_sums_kernel<<<dim3(static_cast<unsigned int>((a->ffn + 255) / 256), 2), 256, 0, s>>>(
                b.partial, row_blocks(a), a->ffn, a->db_gate, a->db_up, a->dt);
        }
        if (b.w.products == 0) { return; }
        if (b.dx >= 0 && b.dw >= 0) {
            pack({&b.x, &b.w_gate, &b.w_up}, s);
        } else if (b.dx >= 0) {
            pack({&b.w_gate, &b.w_up}, s);
        } else {
            pack({&b.x}, s);
        }
        PlainTile<T> tile{{{nullptr, nullptr}, {nullptr, nullptr}}, b.scratch.most, true};
        if (b.dx >= 0) {
            Product &p = b.w.product[b.dx];
            p.a = b.d.map(type, kTileM);
            p.b[0] = b.w_gate.as.map(type, kStepK);
            p.b[1] = b.w_up.as.map(type, kStepK);
            set_kind(p, a->dt, b.width);
            tile.out[b.dx][0] = static_cast<T *>(a->dx);
            tile.vec = tile.vec && aligned_rows(a->dx, a->hidden, a->dt);
        }
        if (b.dw >= 0) {
            Product &p = b.w.product[b.dw];
            p.a = b.d.map(type, kStepK);
            p.b[0] = b.x.as.map(type, kStepK);
            set_kind(p, a->dt, b.width);
            tile.out[b.dw][0] = static_cast<T *>(a->dw_gate);
            tile.out[b.dw][1] = static_cast<T *>(a->dw_up);
            for (const void *p : {a->dw_gate, a->dw_up}) { tile.vec = tile.vec && (p == nullptr || aligned_rows(p, a->hidden, a->dt)); }
        }
        b.w.status = status_word();
        b.w.wait_ns = wait_limit(a);
        launch<sizeof(T) == 4>(b.w, tile, b.clusters, b.width, s);
    });
}
}  // namespace
}  // namespace stdml::collective::train

using namespace stdml::collective::train;

extern "C" long long stdmlc_gated_saved(const stdmlc_gated *a)
{
    if (a == nullptr) { return -1; }
    return a->tokens * (a->dt == kF32 ? Saved<float>::row_bytes(a->ffn) : Saved<__half>::row_bytes(a->ffn));
}

extern "C" long long stdmlc_gated_workspace(const stdmlc_gated *a, int backward)
{
    if (a == nullptr || a->tokens < 0 || a->hidden <= 0 || a->ffn <= 0) { return -1; }
    if (a->tokens == 0 || (!backward && a->tokens <= kFewTokens)) { return 0; }
    return bytes_entry([&] { return backward != 0 ? Backward(a).work.used() : Forward(a).work.used(); });
}

extern "C" int stdmlc_gated_forward(const stdmlc_gated *a, int device, void *stream)
{
    return entry(device, [&] {
        check(a);
        if (a->tokens == 0) { return; }
        require(a->h != nullptr, "gated_linear: null operand");
        forward(a, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int stdmlc_gated_backward(const stdmlc_gated *a, int device, void *stream)
{
    return entry(device, [&] {
        check(a);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if (a->tokens == 0) {  // sums of nothing
            const size_t w = static_cast<size_t>(element_size(a->dt)) * a->ffn;
            for (void *p : {a->dw_gate, a->dw_up}) {
                if (p != nullptr) { cuda_ok(cudaMemsetAsync(p, 0, w * a->hidden, s), "cudaMemsetAsync"); }
            }
            for (void *p : {a->db_gate, a->db_up}) {
                if (p != nullptr) { cuda_ok(cudaMemsetAsync(p, 0, w, s), "cudaMemsetAsync"); }
            }
            return;
        }
        require(a->dh != nullptr && a->saved != nullptr && a->workspace != nullptr, "gated_linear: null operand");
        backward(a, s);
    });
}

extern "C" int stdmlc_train_status(int device, int *out)
{
    return entry(device, [&] {
        require(out != nullptr, "status: null output");
        static std::mutex one_at_a_time;  // g_taken has one place
        const std::lock_guard<std::mutex> lock(one_at_a_time);
        cuda_ok(cudaDeviceSynchronize(), "status");  // (a copy alone waits for no stream that was made non-blocking)
        take_status_kernel<<<1, 1>>>();
        unsigned int v = 0;
        cuda_ok(cudaMemcpyFromSymbol(&v, g_taken, sizeof v), "status");
        *out = v != 0 ? 1 : 0;
    });
}
