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

#include "dispatch.cuh"
#include "host.hpp"
#include "product.cuh"

namespace stdml::collective::train
{
namespace
{
constexpr int kPieces = 3;

__device__ unsigned int g_status;

// ------------------------------------------------------------ results of a tile
template <typename T>
__device__ __forceinline__ void store16(T *to, const float (&v)[16], long long left, bool vec)
{
    if (vec && left >= 16) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                reinterpret_cast<float4 *>(to)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
        } else {
            __align__(16) T t[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) { t[i] = from_f32<T>(v[i]); }
            reinterpret_cast<uint4 *>(to)[0] = reinterpret_cast<const uint4 *>(t)[0];
            reinterpret_cast<uint4 *>(to)[1] = reinterpret_cast<const uint4 *>(t)[1];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i < left) { to[i] = from_f32<T>(v[i]); }
        }
    }
}

// g and u of 128 columns side by side in a tile: h, and what the backward pass needs of them.
template <typename T, int kAct>
struct GatedTile {
    T *h;
    const T *b_gate, *b_up;
    float *saved;  // g, u: [2][tokens][pitch]
    long long pitch;
    bool vec;

    __device__ __forceinline__ void tile(const Product &p, long long m0, long long nt, int, int warp, uint32_t tmem) const
    {
        const long long row = m0 + 32 * (warp & 3) + (threadIdx.x & 31);
        const int half = warp >> 2;
        tmem += (32u * (warp & 3) << 16) + 64 * half;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
            const long long col = nt * 128 + 64 * half + 16 * c;
            if (col >= p.n) { break; }
            float g[16], u[16];
            tmem_load16(tmem + 16 * c, g);
            tmem_load16(tmem + 128 + 16 * c, u);
            tmem_loaded(g);
            tmem_loaded(u);
            if (row < p.m) {
                if (b_gate != nullptr) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if (col + i < p.n) {
                            g[i] += to_f32(b_gate[col + i]);
                            u[i] += to_f32(b_up[col + i]);
                        }
                    }
                }
                if (saved != nullptr) {
                    store16(saved + row * pitch + col, g, 16, true);
                    store16(saved + (p.m + row) * pitch + col, u, 16, true);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) { u[i] *= act<kAct>(g[i]); }
                store16(h + row * p.n + col, u, p.n - col, vec);
            }
            __syncwarp();
        }
    }
};

template <typename T>
struct PlainTile {
    T *out[2];  // of each z
    bool vec;

    __device__ __forceinline__ void tile(const Product &p, long long m0, long long nt, int z, int warp, uint32_t tmem) const
    {
        const long long row = m0 + 32 * (warp & 3) + (threadIdx.x & 31);
        const int half = warp >> 2;
        tmem += (32u * (warp & 3) << 16) + 128 * half;
        T *to = out[z] + row * p.n;
#pragma unroll 1
        for (int c = 0; c < 8; ++c) {
            const long long col = nt * kTileN + 128 * half + 16 * c;
            if (col >= p.n) { break; }
            float v[16];
            tmem_load16(tmem + 16 * c, v);
            tmem_loaded(v);
            if (row < p.m) { store16(to + col, v, p.n - col, vec); }
            __syncwarp();
        }
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

// Rows of a pitch that TMA takes; 32-bit values as pieces: [pieces][rows][pitch].
template <typename T>
__global__ void pack_kernel(const T *from, long long from_row, long long rows, long long cols, long long pitch, uint16_t *to)
{
    const long long many = rows * cols, step = static_cast<long long>(gridDim.x) * blockDim.x;
    for (long long e = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; e < many; e += step) {
        const long long r = e / cols, c = e - r * cols;
        const T v = from[r * from_row + c];
        uint16_t *at = to + r * pitch + c;
        if constexpr (sizeof(T) == 4) {
            uint16_t piece[kPieces];
            cut(v, piece);
            for (int i = 0; i < kPieces; ++i) { at[i * rows * pitch] = piece[i]; }
        } else {
            *at = *reinterpret_cast<const uint16_t *>(&v);
        }
    }
}

// ------------------------------------------------------------ dg and du
constexpr int kGradRows = 64, kGradCols = 256;  // of a block: 8 rows of 32 threads with 8 columns each

struct GateGrad {
    const void *dh;
    long long dh_row;
    const float *saved;
    long long tokens, ffn, pitch;
    uint16_t *d;      // [gate, up][pieces][tokens][pitch]
    float *partial;   // [row blocks][gate, up][ffn]; null: no sums
    bool vec;
};

template <typename T, int kAct>
__global__ void __launch_bounds__(256) gate_grad_kernel(GateGrad a)
{
    __shared__ float sums[2][8][kGradCols];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const long long col = blockIdx.x * static_cast<long long>(kGradCols) + 8 * tx;
    const long long first = blockIdx.y * static_cast<long long>(kGradRows);
    float sg[8] = {}, su[8] = {};
    if (col < a.ffn) {
        for (long long r = first + ty; r < min(first + kGradRows, a.tokens); r += 8) {
            float dh[8], g[8], u[8];
            const T *from = static_cast<const T *>(a.dh) + r * a.dh_row + col;
            if (a.vec && col + 8 <= a.ffn) {
                __align__(16) T t[8];
                for (int i = 0; i < static_cast<int>(8 * sizeof(T) / 16); ++i) {
                    reinterpret_cast<uint4 *>(t)[i] = reinterpret_cast<const uint4 *>(from)[i];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) { dh[i] = to_f32(t[i]); }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) { dh[i] = col + i < a.ffn ? to_f32(from[i]) : 0.f; }
            }
            const float4 *pg = reinterpret_cast<const float4 *>(a.saved + r * a.pitch + col);
            const float4 *pu = reinterpret_cast<const float4 *>(a.saved + (a.tokens + r) * a.pitch + col);
            reinterpret_cast<float4 *>(g)[0] = pg[0];
            reinterpret_cast<float4 *>(g)[1] = pg[1];
            reinterpret_cast<float4 *>(u)[0] = pu[0];
            reinterpret_cast<float4 *>(u)[1] = pu[1];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float dg = dh[i] * u[i] * act_grad<kAct>(g[i]), du = dh[i] * act<kAct>(g[i]);
                g[i] = dg;
                u[i] = du;
                sg[i] += dg;
                su[i] += du;
            }
            constexpr int kSlabs = sizeof(T) == 4 ? kPieces : 1;
            const long long slab = a.tokens * a.pitch;
            uint16_t *at = a.d + r * a.pitch + col;
            __align__(16) uint16_t out[2][kSlabs][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (sizeof(T) == 4) {
                    uint16_t piece[kPieces];
                    cut(g[i], piece);
                    for (int j = 0; j < kPieces; ++j) { out[0][j][i] = piece[j]; }
                    cut(u[i], piece);
                    for (int j = 0; j < kPieces; ++j) { out[1][j][i] = piece[j]; }
                } else {
                    const T x = from_f32<T>(g[i]), y = from_f32<T>(u[i]);
                    out[0][0][i] = *reinterpret_cast<const uint16_t *>(&x);
                    out[1][0][i] = *reinterpret_cast<const uint16_t *>(&y);
                }
            }
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
    const long long mine = blockIdx.x * static_cast<long long>(kGradCols) + threadIdx.x;
    if (mine >= a.ffn) { return; }
    for (int z = 0; z < 2; ++z) {
        float sum = 0;
        for (int i = 0; i < 8; ++i) { sum += sums[z][i][threadIdx.x]; }
        a.partial[(2ll * blockIdx.y + z) * a.ffn + mine] = sum;
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
    void pack(cudaStream_t s) const
    {
        if (!packed || rows == 0) { return; }
        const long long blocks = (rows * cols + 255) / 256;
        by_dtype(dt, [&](auto t) {
            using T = decltype(t);
            pack_kernel<T><<<static_cast<unsigned int>(std::min(blocks, 8192ll)), 256, 0, s>>>(
                static_cast<const T *>(from), row, rows, cols, as.pitch, static_cast<uint16_t *>(const_cast<void *>(as.ptr)));
        });
    }
};

struct Forward {
    Bump work;
    Operand x, w_gate, w_up;

    explicit Forward(const stdmlc_gated *a)
        : work(a->workspace), x(a->x, a->x_row, a->tokens, a->hidden, a->dt, work),
          w_gate(a->w_gate, a->w_gate_row, a->ffn, a->hidden, a->dt, work),
          w_up(a->w_up, a->w_up_row, a->ffn, a->hidden, a->dt, work)
    {
    }
};

long long row_blocks(const stdmlc_gated *a) { return (a->tokens + kGradRows - 1) / kGradRows; }
long long saved_pitch(const stdmlc_gated *a) { return up_to(a->ffn, 16); }

struct Backward : Forward {
    Matrix d;
    float *partial;

    explicit Backward(const stdmlc_gated *a) : Forward(a)
    {
        d = {work.take<uint16_t>(2 * pieces_of(a->dt) * a->tokens * saved_pitch(a)), a->tokens, a->ffn, saved_pitch(a),
             2 * pieces_of(a->dt)};
        partial = work.take<float>(2 * row_blocks(a) * a->ffn);
    }
};

unsigned int *status_word()
{
    void *p = nullptr;
    cuda_ok(cudaGetSymbolAddress(&p, g_status), "status word");
    return static_cast<unsigned int *>(p);
}

// The pairs of pieces whose products are summed, smallest first.
constexpr signed char kPairs[6][2] = {{0, 2}, {2, 0}, {1, 1}, {0, 1}, {1, 0}, {0, 0}};

template <int kCtas, bool kAcrossA, bool kAcrossB, bool kTwoB, typename Epilogue>
void launch(Product &p, const Epilogue &epilogue, int dt, long long reduction, cudaStream_t s)
{
    p.steps = static_cast<int>((reduction + kStepK - 1) / kStepK);
    p.m_tiles = static_cast<int>((p.m + kTileM * kCtas - 1) / (kTileM * kCtas));
    const int width = kTwoB ? 128 : kTileN;
    p.n_tiles = static_cast<int>((p.n + width - 1) / width);
    const uint32_t type = dt == kF16 ? 0u : 1u;
    p.kind = (1u << 4) | (type << 7) | (type << 10) | (kAcrossA ? 1u << 15 : 0u) | (kAcrossB ? 1u << 16 : 0u) |
             (static_cast<uint32_t>(kTileN >> 3) << 17) | (static_cast<uint32_t>(kTileM * kCtas >> 4) << 24);
    p.status = status_word();
    const long long tiles = static_cast<long long>(p.m_tiles) * p.n_tiles * p.z;
    require(tiles < (1ll << 30), "gated_linear: too large");
    auto kernel = product_kernel<kCtas, kAcrossA, kAcrossB, kTwoB, Epilogue>;
    constexpr int kSmem = product_smem<kCtas>();
    cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem), "shared memory");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned int>(std::min<long long>(tiles, sm_count() / kCtas) * kCtas));
    cfg.blockDim = dim3(kProductThreads);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = s;
    cudaLaunchAttribute pair[1];
    pair[0].id = cudaLaunchAttributeClusterDimension;
    pair[0].val.clusterDim = {static_cast<unsigned int>(kCtas), 1, 1};
    cfg.attrs = pair;
    cfg.numAttrs = 1;
    cuda_ok(cudaLaunchKernelEx(&cfg, kernel, p, epilogue), "gated_linear: launch");
}

constexpr int kCtas = 2;

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

void forward(const stdmlc_gated *a, cudaStream_t s)
{
    const Forward f(a);
    f.x.pack(s);
    f.w_gate.pack(s);
    f.w_up.pack(s);
    Product p{};
    p.a = f.x.as.map(map_type(a->dt), kTileM);
    p.b[0] = f.w_gate.as.map(map_type(a->dt), 128);
    p.b[1] = f.w_up.as.map(map_type(a->dt), 128);
    const bool wide = a->dt == kF32;
    for (int i = wide ? 0 : 5; i < 6; ++i) { p.segments[p.segment_count++] = {kPairs[i][0], 0, kPairs[i][1]}; }
    p.m = a->tokens;
    p.n = a->ffn;
    p.z = 1;
    by_dtype(a->dt, [&](auto t) {
        using T = decltype(t);
        by_gate(a->act, [&](auto k) {
            const GatedTile<T, decltype(k)::value> tile{static_cast<T *>(a->h), static_cast<const T *>(a->b_gate),
                                                        static_cast<const T *>(a->b_up), static_cast<float *>(a->saved),
                                                        saved_pitch(a), aligned_rows(a->h, a->ffn, a->dt)};
            launch<kCtas, false, false, true>(p, tile, a->dt, a->hidden, s);
        });
    });
}

void backward(const stdmlc_gated *a, cudaStream_t s)
{
    const Backward b(a);
    const bool sums = a->db_gate != nullptr || a->db_up != nullptr;
    const GateGrad gg{a->dh, a->dh_row, static_cast<const float *>(a->saved), a->tokens, a->ffn, b.d.pitch,
                      static_cast<uint16_t *>(const_cast<void *>(b.d.ptr)), sums ? b.partial : nullptr,
                      aligned_rows(a->dh, a->dh_row, a->dt)};
    const bool wide = a->dt == kF32;
    const int pieces = pieces_of(a->dt);
    const CUtensorMapDataType type = map_type(a->dt);
    by_dtype(a->dt, [&](auto t) {
        using T = decltype(t);
        by_gate(a->act, [&](auto k) {
            const dim3 grid(static_cast<unsigned int>((a->ffn + kGradCols - 1) / kGradCols), static_cast<unsigned int>(row_blocks(a)));
            gate_grad_kernel<T, decltype(k)::value><<<grid, 256, 0, s>>>(gg);
        });
        if (sums) {
            bias_sums_kernel<<<dim3(static_cast<unsigned int>((a->ffn + 255) / 256), 2), 256, 0, s>>>(
                b.partial, row_blocks(a), a->ffn, a->db_gate, a->db_up, a->dt);
        }
        if (a->dx != nullptr) {
            b.w_gate.pack(s);
            b.w_up.pack(s);
            Product p{};
            p.a = b.d.map(type, kTileM);
            p.b[0] = b.w_gate.as.map(type, kStepK);
            p.b[1] = b.w_up.as.map(type, kStepK);
            for (int i = wide ? 0 : 5; i < 6; ++i) {
                for (int z = 0; z < 2; ++z) {
                    p.segments[p.segment_count++] = {static_cast<signed char>(z * pieces + kPairs[i][0]),
                                                     static_cast<signed char>(z), kPairs[i][1]};
                }
            }
            p.m = a->tokens;
            p.n = a->hidden;
            p.z = 1;
            const PlainTile<T> tile{{static_cast<T *>(a->dx), nullptr}, aligned_rows(a->dx, a->hidden, a->dt)};
            launch<kCtas, false, true, false>(p, tile, a->dt, a->ffn, s);
        }
        if (a->dw_gate != nullptr || a->dw_up != nullptr) {
            b.x.pack(s);
            Product p{};
            p.a = b.d.map(type, kStepK);
            p.b[0] = p.b[1] = b.x.as.map(type, kStepK);
            for (int i = wide ? 0 : 5; i < 6; ++i) { p.segments[p.segment_count++] = {kPairs[i][0], 0, kPairs[i][1]}; }
            p.m = a->ffn;
            p.n = a->hidden;
            p.z_slabs = pieces;
            p.z_first = a->dw_gate != nullptr ? 0 : 1;
            p.z = a->dw_gate != nullptr && a->dw_up != nullptr ? 2 : 1;
            const PlainTile<T> tile{{static_cast<T *>(a->dw_gate), static_cast<T *>(a->dw_up)},
                                    (a->dw_gate == nullptr || aligned_rows(a->dw_gate, a->hidden, a->dt)) &&
                                        (a->dw_up == nullptr || aligned_rows(a->dw_up, a->hidden, a->dt))};
            launch<kCtas, true, true, false>(p, tile, a->dt, a->tokens, s);
        }
    });
}
}  // namespace
}  // namespace stdml::collective::train

using namespace stdml::collective::train;

extern "C" long long stdmlc_gated_saved(const stdmlc_gated *a)
{
    return a == nullptr ? -1 : 8 * a->tokens * saved_pitch(a);
}

extern "C" long long stdmlc_gated_workspace(const stdmlc_gated *a, int backward)
{
    if (a == nullptr) { return -1; }
    return backward ? Backward(a).work.used() : Forward(a).work.used();
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
        unsigned int v = 0;
        cuda_ok(cudaMemcpyFromSymbol(&v, g_status, sizeof v), "status");
        if (v != 0) {
            const unsigned int none = 0;
            cuda_ok(cudaMemcpyToSymbol(g_status, &none, sizeof none), "status");
        }
        *out = static_cast<int>(v);
    });
}
