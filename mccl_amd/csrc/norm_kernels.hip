// norm_kernels.hip -- layer norm, dropout and both in one pass over the seam of a transformer block,
// forward and backward.
//
//   forward    t = dropout(x) + residual (either left out on demand), s = t
//              m = sum t / D,  v = sum (t - m)^2 / D,  r = 1 / sqrt(v + eps),  y = (t - m) r w + b
//   backward   g = dy w,  u = (s - m) r
//              dt = r (g - sum g / D - u sum(g u) / D) + ds,  dresidual = dt,  dx = dropout(dt)
//              dw = sum over rows of dy u,  db = sum over rows of dy
//
// HBM-bound: one read of every input and one write of every output, two to five flops a byte.  A row
// stays in the registers of the lanes that share it, so that its mean, the squares about it and the result
// come from one read; sums and statistics are held in 32 bits, and each output is rounded once.  A lane holds
// packets of eight elements: 16 bytes of a 16-bit type, and the 128 bits of one call of the generator.
//
// What large matrices reach, of the bytes they have to move (a copy of that size moves 5.5 TB/s here): the seam of 16384 x 4096 bf16 forward
// 94 us, 5.7 TB/s; layer norm's backward 82 us, 4.9; dropout of 16384 x 8192 bf16 94 us, 5.7.  Small ones are bound by the launch and a round
// trip or two to memory: 8 x 1024 bf16 forward 6 us a call, of which the kernel takes 3.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "operators.h"

namespace mcclx {
namespace {

constexpr int kPacket = 8;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// A packet as it lies in memory: words, because the compiler takes a vector of halves apart into a register each.
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
template <class T> using Raw = std::conditional_t<sizeof(T) == 4, u32x8, u32x4>;
template <class T> struct Packets;
template <> struct Packets<float> { typedef f32x8 Values; };
template <> struct Packets<_Float16> { typedef f16x8 Values; };
template <> struct Packets<__bf16> { typedef bf16x8 Values; };

template <class T>
__device__ __forceinline__ f32x8 to_f32(const Raw<T>& v) {
    return __builtin_convertvector(__builtin_bit_cast(typename Packets<T>::Values, v), f32x8);
}
template <class T>
__device__ __forceinline__ Raw<T> from_f32(const f32x8& v) {  // round to nearest even
    return __builtin_bit_cast(Raw<T>, __builtin_convertvector(v, typename Packets<T>::Values));
}
// A packet without its first `s` elements (1 .. 7), zeros behind the others.
template <class T>
__device__ __forceinline__ Raw<T> shift_down(Raw<T> v, int s) {
    if constexpr (sizeof(T) == 2) {
        u64x2 d = __builtin_bit_cast(u64x2, v);
        const int bits = s * 16;
        if (bits >= 64) {
            d[0] = d[1] >> (bits - 64);
            d[1] = 0;
        } else {
            d[0] = d[0] >> bits | d[1] << (64 - bits);
            d[1] >>= bits;
        }
        return __builtin_bit_cast(Raw<T>, d);
    } else {
        const Raw<T> zero = {};
        if (s & 4) v = __builtin_shufflevector(v, zero, 4, 5, 6, 7, 8, 9, 10, 11);
        if (s & 2) v = __builtin_shufflevector(v, zero, 2, 3, 4, 5, 6, 7, 8, 9);
        if (s & 1) v = __builtin_shufflevector(v, zero, 1, 2, 3, 4, 5, 6, 7, 8);
        return v;
    }
}
// Element alignment is all that the kernels may assume: any row stride and any number of columns.
// Packet `group` of a row of `cols` elements, zeros past the row's end.  The last packet of a row that is no number of whole
// ones is read in one piece too, from where it still ends with the row: a lane that loads its elements one by one has its whole
// wave wait (4099 rows of 1111 f16 forward 9.0 us, of 1112 7.0).
template <class T>
__device__ __forceinline__ Raw<T> get_packet(const T* row, uint32_t group, uint32_t cols) {
    typedef Raw<T> Loose __attribute__((aligned(sizeof(T))));
    const int left = (int)cols - (int)(group * kPacket);
    Raw<T> v = {};
    if (left <= 0) return v;
    if (cols < kPacket) {
        for (int i = left - 1; i >= 0; --i) {  // the first element ends up in front
            if constexpr (sizeof(T) == 2) {
                u64x2 d = __builtin_bit_cast(u64x2, v);
                d[1] = d[1] << 16 | d[0] >> 48;
                d[0] = d[0] << 16 | reinterpret_cast<const uint16_t*>(row)[i];
                v = __builtin_bit_cast(Raw<T>, d);
            } else {
                v = __builtin_shufflevector(v, v, 0, 0, 1, 2, 3, 4, 5, 6);
                v[0] = reinterpret_cast<const uint32_t*>(row)[i];
            }
        }
        return v;
    }
    v = *reinterpret_cast<const Loose*>(row + (left >= kPacket ? (size_t)group * kPacket : (size_t)cols - kPacket));
    return left >= kPacket ? v : shift_down<T>(v, kPacket - left);
}
template <class T>
__device__ __forceinline__ void put_packet(T* row, uint32_t group, uint32_t cols, Raw<T> v) {
    typedef Raw<T> Loose __attribute__((aligned(sizeof(T))));
    const int left = (int)cols - (int)(group * kPacket);
    T* to = row + (size_t)group * kPacket;
    if (left >= kPacket) {
        *reinterpret_cast<Loose*>(to) = v;
    } else if (left > 0) {  // four, two and one
        typedef std::conditional_t<sizeof(T) == 4, u32x4, u32x2> Four;
        typedef std::conditional_t<sizeof(T) == 4, u32x2, uint32_t> Two;
        typedef std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t> One;
        typedef Four LooseFour __attribute__((aligned(sizeof(T))));
        typedef Two LooseTwo __attribute__((aligned(sizeof(T))));
        if (left & 4) {
            Four f;
            if constexpr (sizeof(T) == 4) f = __builtin_shufflevector(v, v, 0, 1, 2, 3);
            else f = __builtin_shufflevector(v, v, 0, 1);
            *reinterpret_cast<LooseFour*>(to) = f;
            v = shift_down<T>(v, 4);
            to += 4;
        }
        if (left & 2) {
            Two f;
            if constexpr (sizeof(T) == 4) f = __builtin_shufflevector(v, v, 0, 1);
            else f = v[0];
            *reinterpret_cast<LooseTwo*>(to) = f;
            v = shift_down<T>(v, 2);
            to += 2;
        }
        if (left & 1) *reinterpret_cast<One*>(to) = (One)v[0];
    }
}
// The compiler knows nothing of `v` from here on: what was made of it is made again, rather than kept in registers.
template <class R>
__device__ __forceinline__ void forget(R& v) {
    asm volatile("" : "+v"(v));
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten
// rounds of two 32 x 32 -> 64 bit products.  One call serves the eight elements of a packet with 16 bits each: the
// products run at a quarter of the rate, and at 32 bits an element they, not HBM, would set the time.
__device__ __forceinline__ uint4 philox(uint32_t group, uint32_t row, const DropArgs& d) {
    uint32_t c0 = group, c1 = row, c2 = d.offset[0], c3 = d.offset[1], k0 = d.key[0], k1 = d.key[1];
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}
// v, with the elements that the mask drops zero (whatever they held) and the others scaled.
__device__ __forceinline__ f32x8 drop(f32x8 v, uint32_t group, uint32_t row, const DropArgs& d) {
    const uint4 bits = philox(group, row, d);
    const uint32_t w[4] = {bits.x, bits.y, bits.z, bits.w};
#pragma unroll
    for (int i = 0; i < kPacket; ++i) {
        const uint32_t u = (i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu;
        v[i] = u >= d.threshold ? v[i] * d.factor : 0.f;
    }
    return v;
}

// v + the same of the lane that CTRL names, in the vector unit (a trip through LDS takes ten times as long).
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}
// The sum over groups of LANES lanes of a wave, in each of them: the neighbour, the other pair, the other four, the
// other eight (in mirrored order, when fours and eights hold one value each), the other row of 16, the other half.
template <int LANES>
__device__ __forceinline__ float wave_sum(float v) {
    if constexpr (LANES > 1) v = add_dpp<0xB1>(v);   // quad_perm 1 0 3 2
    if constexpr (LANES > 2) v = add_dpp<0x4E>(v);   // quad_perm 2 3 0 1
    if constexpr (LANES > 4) v = add_dpp<0x141>(v);  // row_half_mirror
    if constexpr (LANES > 8) v = add_dpp<0x140>(v);  // row_mirror
    if constexpr (LANES > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if constexpr (LANES > 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}
// The sum over the LANES lanes of a row, in each of them.  Rows of several waves go through `scratch`, a place
// of its own for each sum between two barriers, which the whole block has to reach.
template <int LANES, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* scratch) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum<LANES < 64 ? LANES : 64>(v[i]);
    if constexpr (LANES > 64) {
        constexpr int kWaves = LANES / 64;
        scratch += threadIdx.x / LANES * (N * kWaves);
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) scratch[i * kWaves + threadIdx.x % LANES / 64] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) v[i] += scratch[i * kWaves + w];
        }
    }
}

// What lane `lane` of a row holds in its packet j: `full` elements of it lie in the row.
template <int LANES>
struct Place {
    uint32_t lane, cols;
    __device__ __forceinline__ uint32_t group(int j) const { return lane + (uint32_t)j * LANES; }
    __device__ __forceinline__ int full(int j) const {
        const int left = (int)cols - (int)(group(j) * kPacket);
        return left < 0 ? 0 : left < kPacket ? left : kPacket;
    }
    template <class T>
    __device__ __forceinline__ Raw<T> get(const T* row, int j) const {
        return get_packet<T>(row, group(j), cols);
    }
    template <class T>
    __device__ __forceinline__ void put(T* row, int j, const Raw<T>& v) const {
        put_packet<T>(row, group(j), cols, v);
    }
};

// A row to LANES lanes and NV packets a lane, read once.  The squares are those about the mean that the row's first sum has given, so nothing
// cancels where the mean is large.
template <class T, class P, int LANES, int NV, bool SEAM>
__global__ void __launch_bounds__(LANES <= 64 ? 256 : LANES) norm_forward_kernel(NormForwardArgs a) {
    constexpr int kThreads = LANES <= 64 ? 256 : LANES;
    __shared__ float scratch[2][LANES > 64 ? LANES / 64 : 1];
    const Place<LANES> at{threadIdx.x % LANES, a.cols};
    const uint64_t row = a.first_row + (uint64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
    if (row >= a.rows) return;  // (whole blocks only where a row has more than a wave)
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    f32x8 t[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) t[j] = to_f32<T>(at.template get<T>(x, j));
    // The parameters are on their way while the row is summed (8 x 1024 bf16 3.0 us, behind the sums 3.3; 16384 x 4096 bf16 41.4, 43.0), unless
    // that takes registers which waves need: blocks of 1024 (2048 x 16384 f32 62.7, 48.9), f32 rows with the seam (65536 x 512 102, 100),
    // three packets a lane (32768 x 1280 bf16 33.9, 30.5, with f32 parameters 40.5, 30.0; 8192 x 1280 f32 20.6, 17.0; 146 registers, and 47), and f32
    // parameters beside long 16-bit rows, with the seam those of more than a wave (16384 x 6144 98, 90.5, seam 163, 154; 65536 x 2048 seam 204,
    // 196; but 16384 x 2560 28.4, 29.3, 16384 x 1024 seam 22.4, 22.9).
    constexpr bool kEarly = LANES < 1024 && NV < 3 && (sizeof(T) == sizeof(P) ? sizeof(T) == 2 || !SEAM : LANES <= (SEAM ? 64 : 256));
    Raw<P> w[NV], b[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (kEarly && a.weight) w[j] = at.template get<P>(static_cast<const P*>(a.weight), j);
        if (kEarly && a.bias) b[j] = at.template get<P>(static_cast<const P*>(a.bias), j);
    }
    if constexpr (SEAM) {
        if (a.drop.threshold)
#pragma unroll
            for (int j = 0; j < NV; ++j) t[j] = drop(t[j], at.group(j), (uint32_t)row, a.drop);
        if (a.residual) {
            const T* res = static_cast<const T*>(a.residual) + row * a.residual_stride;
#pragma unroll
            for (int j = 0; j < NV; ++j) t[j] += to_f32<T>(at.template get<T>(res, j));
        }
        if (a.s) {
            T* s = static_cast<T*>(a.s) + row * a.cols;
#pragma unroll
            for (int j = 0; j < NV; ++j) at.template put<T>(s, j, from_f32<T>(t[j]));
        }
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < kPacket; ++i) sum[0] += t[j][i];
    row_sum<LANES>(sum, scratch[0]);
    const float mean = sum[0] / (float)a.cols;
    float square[1] = {0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int n = at.full(j);
#pragma unroll
        for (int i = 0; i < kPacket; ++i) {
            t[j][i] -= mean;
            square[0] = i < n ? __builtin_fmaf(t[j][i], t[j][i], square[0]) : square[0];
        }
    }
    row_sum<LANES>(square, scratch[1]);
    const float rstd = 1.f / __builtin_sqrtf(square[0] / (float)a.cols + a.eps);
    if (at.lane == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        f32x8 v = t[j] * rstd;
        if (a.weight) v *= to_f32<P>(kEarly ? w[j] : at.template get<P>(static_cast<const P*>(a.weight), j));
        if (a.bias) v += to_f32<P>(kEarly ? b[j] : at.template get<P>(static_cast<const P*>(a.bias), j));
        at.template put<T>(y, j, from_f32<T>(v));
    }
}

// Rows too long for the registers of a block: a block of 1024 lanes goes over its row three times.
template <class T, class P, bool SEAM>
__global__ void __launch_bounds__(1024) norm_forward_long_kernel(NormForwardArgs a) {
    __shared__ float scratch[2][16];
    const uint64_t row = a.first_row + blockIdx.x;
    const uint32_t packets = (a.cols + kPacket - 1) / kPacket;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* res = SEAM && a.residual ? static_cast<const T*>(a.residual) + row * a.residual_stride : nullptr;
    auto value = [&](const Place<1>& at) {
        f32x8 t = to_f32<T>(at.template get<T>(x, 0));
        if constexpr (SEAM) {
            if (a.drop.threshold) t = drop(t, at.lane, (uint32_t)row, a.drop);
            if (res) t += to_f32<T>(at.template get<T>(res, 0));
        }
        return t;
    };
    float sum[1] = {0.f};
    for (uint32_t g = threadIdx.x; g < packets; g += 1024) {
        const Place<1> at{g, a.cols};
        const f32x8 t = value(at);
#pragma unroll
        for (int i = 0; i < kPacket; ++i) sum[0] += t[i];
        if (SEAM && a.s) at.template put<T>(static_cast<T*>(a.s) + row * a.cols, 0, from_f32<T>(t));
    }
    row_sum<1024>(sum, scratch[0]);
    const float mean = sum[0] / (float)a.cols;
    float square[1] = {0.f};
    for (uint32_t g = threadIdx.x; g < packets; g += 1024) {
        const Place<1> at{g, a.cols};
        const f32x8 t = value(at) - mean;
        const int n = at.full(0);
#pragma unroll
        for (int i = 0; i < kPacket; ++i) square[0] = i < n ? __builtin_fmaf(t[i], t[i], square[0]) : square[0];
    }
    row_sum<1024>(square, scratch[1]);
    const float rstd = 1.f / __builtin_sqrtf(square[0] / (float)a.cols + a.eps);
    if (threadIdx.x == 0) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
    }
    for (uint32_t g = threadIdx.x; g < packets; g += 1024) {
        const Place<1> at{g, a.cols};
        f32x8 v = (value(at) - mean) * rstd;
        if (a.weight) v *= to_f32<P>(at.template get<P>(static_cast<const P*>(a.weight), 0));
        if (a.bias) v += to_f32<P>(at.template get<P>(static_cast<const P*>(a.bias), 0));
        at.template put<T>(static_cast<T*>(a.y) + row * a.cols, 0, from_f32<T>(v));
    }
}

// A block takes ROWS rows, then as many further on as the grid covers, and sums its share of dweight and dbias in
// the registers of the lanes that own the columns: `parts` rows of partial sums leave the device's registers, not `rows`, and
// their order is the same in every call.  One packet a lane and rows of several waves, rather than more packets:
// what a lane holds (the sums, the row, with AHEAD the next row) decides how many waves a SIMD has.
template <class T, class P, int LANES, int NV, int ROWS, bool SEAM, bool AHEAD>
__global__ void __launch_bounds__(LANES* ROWS) norm_backward_kernel(NormBackwardArgs a) {
    constexpr int kWaves = LANES * ROWS / 64, kSumRows = LANES >= 64 ? ROWS : kWaves;  // rows of sums at the end
    __shared__ float scratch[2][LANES > 64 ? 2 * kWaves : 1];
    const Place<LANES> at{threadIdx.x % LANES, a.cols};
    f32x8 dw[NV], db[NV];
    Raw<P> w[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        dw[j] = db[j] = f32x8{};
        if (a.weight) w[j] = at.template get<P>(static_cast<const P*>(a.weight), j);
    }
    struct Row {
        Raw<T> dy[NV], x[NV], ds[SEAM ? NV : 1];
        float mean, rstd;
    };
    auto fetch = [&](Row& r, uint64_t row) {
        if (row >= a.rows) {  // (a block's last rows: they add nothing)
            r = Row{};
            return;
        }
        const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            r.dy[j] = at.template get<T>(dy, j);
            r.x[j] = at.template get<T>(x, j);
        }
        if constexpr (SEAM)
            if (a.ds)
#pragma unroll
                for (int j = 0; j < NV; ++j) r.ds[j] = at.template get<T>(static_cast<const T*>(a.ds) + row * a.ds_stride, j);
        r.mean = a.mean[row];
        r.rstd = a.rstd[row];
    };
    const uint64_t step = (uint64_t)gridDim.x * ROWS;
    int turn = 0;
    Row next;
    if (AHEAD) fetch(next, (uint64_t)blockIdx.x * ROWS + threadIdx.x / LANES);
    for (uint64_t base = (uint64_t)blockIdx.x * ROWS; base < a.rows; base += step, turn ^= 1) {
        const uint64_t row = base + threadIdx.x / LANES;
        Row now;
        if constexpr (AHEAD) {
            now = next;
            if (base + step < a.rows) fetch(next, row + step);  // on its way while this row is summed and written
        } else {
            fetch(now, row);
        }
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const f32x8 d = to_f32<T>(now.dy[j]);  // zeros past the row's end, and so are its products
            const f32x8 u = (to_f32<T>(now.x[j]) - now.mean) * now.rstd;
            const f32x8 g = a.weight ? d * to_f32<P>(w[j]) : d;
#pragma unroll
            for (int i = 0; i < kPacket; ++i) {
                sum[0] += g[i];
                sum[1] = __builtin_fmaf(g[i], u[i], sum[1]);
                dw[j][i] = __builtin_fmaf(d[i], u[i], dw[j][i]);
                db[j][i] += d[i];
            }
        }
        row_sum<LANES>(sum, scratch[turn]);
        const float m0 = sum[0] / (float)a.cols, m1 = sum[1] / (float)a.cols;
        if (row >= a.rows) continue;  // (the last turn)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            forget(now.dy[j]);
            forget(now.x[j]);
            const f32x8 d = to_f32<T>(now.dy[j]);
            const f32x8 u = (to_f32<T>(now.x[j]) - now.mean) * now.rstd;
            const f32x8 g = a.weight ? d * to_f32<P>(w[j]) : d;
            f32x8 dt = (g - m0 - u * m1) * now.rstd;
            if constexpr (SEAM) {
                if (a.ds) dt += to_f32<T>(now.ds[j]);
                if (a.dresidual) at.template put<T>(static_cast<T*>(a.dresidual) + row * a.cols, j, from_f32<T>(dt));
                if (a.dx && a.drop.threshold) dt = drop(dt, at.group(j), (uint32_t)row, a.drop);
            }
            if (a.dx) at.template put<T>(static_cast<T*>(a.dx) + row * a.cols, j, from_f32<T>(dt));
        }
    }
    if (!a.partial) return;
    float* out = a.partial + (uint64_t)blockIdx.x * 2 * a.cols;
    if constexpr (kSumRows > 1) {  // the block's rows into one, in a fixed order
        constexpr int kCols = LANES * NV * kPacket;
        __shared__ float both[kSumRows][2][kCols];
#pragma unroll
        for (int m = LANES; m < 64; m <<= 1)
#pragma unroll
            for (int i = 0; i < kPacket; ++i) {
                dw[0][i] += __shfl_xor(dw[0][i], m);
                db[0][i] += __shfl_xor(db[0][i], m);
            }
        if (LANES >= 64 || threadIdx.x % 64 < LANES) {
            const int r = LANES >= 64 ? threadIdx.x / LANES : threadIdx.x / 64;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                *reinterpret_cast<f32x8*>(&both[r][0][at.group(j) * kPacket]) = dw[j];
                *reinterpret_cast<f32x8*>(&both[r][1][at.group(j) * kPacket]) = db[j];
            }
        }
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < 2 * a.cols; c += LANES * ROWS) {
            const uint32_t which = c >= a.cols, col = which ? c - a.cols : c;
            float v = both[0][which][col];
#pragma unroll
            for (int r = 1; r < kSumRows; ++r) v += both[r][which][col];
            out[c] = v;
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            at.template put<float>(out, j, from_f32<float>(dw[j]));
            at.template put<float>(out + a.cols, j, from_f32<float>(db[j]));
        }
    }
}

// Rows too long for the registers of a block, in two launches: the two sums of each row, then dx and the partial sums of
// the columns, a block to 256 packets of columns and a share of the rows.
template <class T, class P>
__global__ void __launch_bounds__(1024) norm_backward_sums_kernel(NormBackwardArgs a, float* sums) {
    __shared__ float scratch[32];
    const uint32_t packets = (a.cols + kPacket - 1) / kPacket;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float sum[2] = {0.f, 0.f};
        for (uint32_t p = threadIdx.x; p < packets; p += 1024) {
            const Place<1> at{p, a.cols};
            f32x8 g = to_f32<T>(at.template get<T>(dy, 0));
            const f32x8 u = (to_f32<T>(at.template get<T>(x, 0)) - mean) * rstd;
            if (a.weight) g *= to_f32<P>(at.template get<P>(static_cast<const P*>(a.weight), 0));
            const int n = at.full(0);
#pragma unroll
            for (int i = 0; i < kPacket; ++i) {
                if (i >= n) continue;
                sum[0] += g[i];
                sum[1] = __builtin_fmaf(g[i], u[i], sum[1]);
            }
        }
        row_sum<1024>(sum, scratch);
        if (threadIdx.x == 0) {
            sums[2 * row] = sum[0] / (float)a.cols;
            sums[2 * row + 1] = sum[1] / (float)a.cols;
        }
        __syncthreads();  // `scratch` is read before the next row writes it
    }
}
template <class T, class P, bool SEAM>
__global__ void __launch_bounds__(256) norm_backward_long_kernel(NormBackwardArgs a, const float* sums) {
    const Place<1> at{blockIdx.x * 256 + threadIdx.x, a.cols};
    if (at.full(0) == 0) return;
    const f32x8 w = a.weight ? to_f32<P>(at.template get<P>(static_cast<const P*>(a.weight), 0)) : f32x8{};
    f32x8 dw = {}, db = {};
    for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float mean = a.mean[row], rstd = a.rstd[row], m0 = sums[2 * row], m1 = sums[2 * row + 1];
        const f32x8 d = to_f32<T>(at.template get<T>(static_cast<const T*>(a.dy) + row * a.dy_stride, 0));
        const f32x8 u = (to_f32<T>(at.template get<T>(static_cast<const T*>(a.x) + row * a.x_stride, 0)) - mean) * rstd;
        const f32x8 g = a.weight ? d * w : d;
        dw += d * u;
        db += d;
        f32x8 dt = (g - m0 - u * m1) * rstd;
        if constexpr (SEAM) {
            if (a.ds) dt += to_f32<T>(at.template get<T>(static_cast<const T*>(a.ds) + row * a.ds_stride, 0));
            if (a.dresidual) at.template put<T>(static_cast<T*>(a.dresidual) + row * a.cols, 0, from_f32<T>(dt));
            if (a.dx && a.drop.threshold) dt = drop(dt, at.lane, (uint32_t)row, a.drop);
        }
        if (a.dx) at.template put<T>(static_cast<T*>(a.dx) + row * a.cols, 0, from_f32<T>(dt));
    }
    if (a.partial) {
        float* out = a.partial + (uint64_t)blockIdx.y * 2 * a.cols;
        at.template put<float>(out, 0, from_f32<float>(dw));
        at.template put<float>(out + a.cols, 0, from_f32<float>(db));
    }
}

// dweight and dbias from their partial sums, columns `first` on: a block to 32 columns, its 32 half waves take the parts in turn, eight
// loads under way at a time (512 parts of 4096 columns 4.8 us).
template <class P>
__global__ void __launch_bounds__(1024) norm_join_kernel(const float* partial, uint32_t parts, uint32_t cols, uint32_t first, P* dweight, P* dbias) {
    __shared__ float both[32][33];
    first += blockIdx.x * 32;
    const uint32_t c = first + threadIdx.x % 32, slice = threadIdx.x / 32;
    P* out = blockIdx.y ? dbias : dweight;
    if (!out) return;
    const float* from = partial + (uint64_t)blockIdx.y * cols + (c < cols ? c : cols - 1);
    float sum[8] = {};
    uint32_t i = slice;
    for (; i + 7 * 32 < parts; i += 8 * 32)
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] += from[(uint64_t)(i + k * 32) * 2 * cols];
#pragma unroll
    for (int k = 0; k < 8; ++k)
        if (i + k * 32 < parts) sum[k] += from[(uint64_t)(i + k * 32) * 2 * cols];
    both[slice][threadIdx.x % 32] = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
    __syncthreads();
    float v[1] = {both[threadIdx.x % 32][slice]};  // column `slice` of the block, a slice a lane
    row_sum<32>(v, nullptr);
    if (threadIdx.x % 32 == 0 && first + slice < cols) out[first + slice] = (P)v[0];
}

// A packet a lane.  4096 x 768 f32 with a residual 7.5 us, 5.0 TB/s, 16384 x 8192 bf16 94 us, 5.7 TB/s: the generator's twenty products a packet
// are done while others' loads are on their way.
template <class T>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutArgs a, uint32_t packets) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < a.rows * packets; i += (uint64_t)gridDim.x * 256) {
        const uint64_t row = i / packets;
        const Place<1> at{(uint32_t)(i - row * packets), a.cols};
        f32x8 v = to_f32<T>(at.template get<T>(static_cast<const T*>(a.x) + row * a.x_stride, 0));
        if (a.drop.threshold) v = drop(v, at.lane, (uint32_t)row, a.drop);
        if (a.residual) v += to_f32<T>(at.template get<T>(static_cast<const T*>(a.residual) + row * a.residual_stride, 0));
        at.template put<T>(static_cast<T*>(a.out) + row * a.cols, 0, from_f32<T>(v));
    }
}

// ---- launches ------------------------------------------------------------------------

constexpr uint64_t kRowsALaunch = 1u << 21;            // a grid holds 2^32 lanes at most, and silently leaves out the others
constexpr uint32_t kJoinedALaunch = 1u << 26;          // columns; 32 lanes each, of one dimension
constexpr uint32_t kForwardMost = 1024 * 2 * kPacket;  // columns that a block of norm_forward_kernel holds

template <class T, class P, int LANES, int NV>
void forward(hipStream_t st, const NormForwardArgs& a) {
    constexpr int kThreads = LANES <= 64 ? 256 : LANES;
    const uint64_t rows = a.rows - a.first_row < kRowsALaunch ? a.rows - a.first_row : kRowsALaunch;
    const dim3 grid((uint32_t)((rows + kThreads / LANES - 1) / (kThreads / LANES)));
    if (a.residual || a.s || a.drop.threshold)
        norm_forward_kernel<T, P, LANES, NV, true><<<grid, dim3(kThreads), 0, st>>>(a);
    else
        norm_forward_kernel<T, P, LANES, NV, false><<<grid, dim3(kThreads), 0, st>>>(a);
}
// Two packets a lane from 128 packets on, and rows of several waves: 16384 rows of 4096 bf16 at 8 packets in one wave / 4 in two /
// 2 in four: 50.8 / 43.9 / 43.1 us, with the seam 109 / 102 / 97.  Three in one wave for what that fits: 4099 x 1111 f16 7.3 us,
// at 2 in two waves 8.0.  (All with the parameters behind the sums.)
template <class T, class P>
void forward_for(hipStream_t st, const NormForwardArgs& a) {
    const uint32_t packets = (a.cols + kPacket - 1) / kPacket;
    if (packets <= 8) return forward<T, P, 8, 1>(st, a);
    if (packets <= 16) return forward<T, P, 16, 1>(st, a);
    if (packets <= 32) return forward<T, P, 32, 1>(st, a);
    if (packets <= 64) return forward<T, P, 64, 1>(st, a);
    if (packets <= 128) return forward<T, P, 64, 2>(st, a);
    if (packets <= 192) return forward<T, P, 64, 3>(st, a);
    if (packets <= 256) return forward<T, P, 128, 2>(st, a);
    if (packets <= 384) return forward<T, P, 192, 2>(st, a);
    if (packets <= 512) return forward<T, P, 256, 2>(st, a);
    if (packets <= 768) return forward<T, P, 384, 2>(st, a);
    if (packets <= 1024) return forward<T, P, 512, 2>(st, a);
    if (a.cols <= kForwardMost) return forward<T, P, 1024, 2>(st, a);
    const dim3 grid((uint32_t)(a.rows - a.first_row < kRowsALaunch ? a.rows - a.first_row : kRowsALaunch));
    if (a.residual || a.s || a.drop.threshold)
        norm_forward_long_kernel<T, P, true><<<grid, dim3(1024), 0, st>>>(a);
    else
        norm_forward_long_kernel<T, P, false><<<grid, dim3(1024), 0, st>>>(a);
}

// Lanes to a row of a backward pass, packets a lane and rows a block: rows that fill the sixteen waves of a CU, since every block leaves
// a row of partial sums (4096 x 768 f32 in blocks of four rows / eight 12.3 / 11.2 us, 1000 x 4096 f16 in one / two 18.8 / 15.7,
// with the seam 4099 x 1111 f16 in one / five 24.1 / 24.9, 16384 x 4096 bf16 in one / two 141 / 131; one number that was lost is 16384 x 4096 bf16
// without the seam, 85.0 / 86.8).  The narrowest rows stay at eight waves, for calls of few rows (1000 x 64 6.0 us, at sixteen 7.1).
// Blocks of 960 and 1024 lanes have 128 registers a lane: f32 rows with the seam spill 8 to 24 bytes there (128, 192, 256 and 512 lanes).
struct Shape {
    uint32_t lanes, packets, rows;
};
constexpr Shape kShapes[] = {{8, 1, 64}, {16, 1, 32}, {32, 1, 16}, {64, 1, 16}, {128, 1, 8}, {192, 1, 5}, {256, 1, 4}, {384, 1, 2}, {512, 1, 2},
                             {768, 1, 1}, {1024, 1, 1}};
constexpr int kShapeCount = sizeof kShapes / sizeof kShapes[0];
constexpr uint32_t kBackwardMost = kShapes[kShapeCount - 1].lanes * kShapes[kShapeCount - 1].packets * kPacket;
int shape_for(uint32_t cols) {
    int i = 0;
    while (i < kShapeCount && kShapes[i].lanes * kShapes[i].packets * kPacket < cols) ++i;
    return i;
}
template <class T, class P, int I>
void backward(hipStream_t st, const NormBackwardArgs& a, int shape) {
    if constexpr (I < kShapeCount) {
        if (shape != I) return backward<T, P, I + 1>(st, a, shape);
        constexpr Shape s = kShapes[I];
        constexpr bool kAhead = s.packets == 1 && (sizeof(T) == 2 || s.lanes < 1024);  // (no room for two rows otherwise)
        const dim3 grid(a.parts), block(s.lanes * s.rows);
        if (a.ds || a.dresidual || a.drop.threshold)
            norm_backward_kernel<T, P, s.lanes, s.packets, s.rows, true, kAhead><<<grid, block, 0, st>>>(a);
        else
            norm_backward_kernel<T, P, s.lanes, s.packets, s.rows, false, kAhead><<<grid, block, 0, st>>>(a);
    }
}
template <class T, class P>
int backward_for(hipStream_t st, NormBackwardArgs a) {
    float* sums = a.partial + (uint64_t)a.parts * 2 * a.cols;  // (long rows only)
    if (!a.dweight && !a.dbias) a.partial = nullptr;
    const uint32_t packets = (a.cols + kPacket - 1) / kPacket;
    int launches = a.rows ? 1 : 0;
    if (a.rows == 0) {  // (the sums of no rows are zero)
    } else if (a.cols <= kBackwardMost) {
        backward<T, P, 0>(st, a, shape_for(a.cols));
    } else {
        norm_backward_sums_kernel<T, P><<<dim3((uint32_t)(a.rows < kRowsALaunch ? a.rows : kRowsALaunch)), dim3(1024), 0, st>>>(a, sums);
        const dim3 grid((packets + 255) / 256, a.parts);
        if (a.ds || a.dresidual || a.drop.threshold)
            norm_backward_long_kernel<T, P, true><<<grid, dim3(256), 0, st>>>(a, sums);
        else
            norm_backward_long_kernel<T, P, false><<<grid, dim3(256), 0, st>>>(a, sums);
        launches = 2;
    }
    if (a.dweight || a.dbias)
        for (uint32_t first = 0; first < a.cols; first += kJoinedALaunch, ++launches) {
            const uint32_t some = a.cols - first < kJoinedALaunch ? a.cols - first : kJoinedALaunch;
            norm_join_kernel<P><<<dim3((some + 31) / 32, 2), dim3(1024), 0, st>>>(a.partial, a.parts, a.cols, first, static_cast<P*>(a.dweight),
                                                                                 static_cast<P*>(a.dbias));
        }
    return launches;
}

}  // namespace

uint32_t norm_backward_parts(uint64_t rows, uint32_t cols, int cus) {
    if (cols > kBackwardMost) {
        const uint64_t blocks = (cols + 256 * kPacket - 1) / (256 * kPacket), want = (4 * (uint64_t)cus + blocks - 1) / blocks;
        return (uint32_t)(rows < want ? rows : want);
    }
    // as many blocks as the device holds at sixteen waves a CU, and all with the same number of turns
    const Shape s = kShapes[shape_for(cols)];
    const uint64_t all = (rows + s.rows - 1) / s.rows, most = 16 / (s.lanes * s.rows / 64) * (uint64_t)cus;
    const uint64_t turns = (all + most - 1) / most;
    return turns ? (uint32_t)((all + turns - 1) / turns) : 0;
}
uint64_t norm_backward_scratch(uint64_t rows, uint32_t cols, int cus) {
    const uint64_t partial = (uint64_t)norm_backward_parts(rows, cols, cus) * 2 * cols * sizeof(float);
    return cols > kBackwardMost ? partial + rows * 2 * sizeof(float) : partial;
}

int launch_norm_forward(hipStream_t st, int dtype, int param_dtype, NormForwardArgs a, hipError_t* error) {
    int launches = 0;
    for (a.first_row = 0; a.first_row < a.rows; a.first_row += kRowsALaunch, ++launches) {
        if (dtype == MCCLX_F32) forward_for<float, float>(st, a);
        else if (dtype == MCCLX_F16 && param_dtype == MCCLX_F16) forward_for<_Float16, _Float16>(st, a);
        else if (dtype == MCCLX_F16) forward_for<_Float16, float>(st, a);
        else if (param_dtype == MCCLX_BF16) forward_for<__bf16, __bf16>(st, a);
        else forward_for<__bf16, float>(st, a);
        if ((*error = hipGetLastError()) != hipSuccess) return -1;
    }
    return launches;
}
int launch_norm_backward(hipStream_t st, int dtype, int param_dtype, const NormBackwardArgs& a, hipError_t* error) {
    int n;
    if (dtype == MCCLX_F32) n = backward_for<float, float>(st, a);
    else if (dtype == MCCLX_F16 && param_dtype == MCCLX_F16) n = backward_for<_Float16, _Float16>(st, a);
    else if (dtype == MCCLX_F16) n = backward_for<_Float16, float>(st, a);
    else if (param_dtype == MCCLX_BF16) n = backward_for<__bf16, __bf16>(st, a);
    else n = backward_for<__bf16, float>(st, a);
    *error = hipGetLastError();
    return *error == hipSuccess ? n : -1;
}
int launch_dropout(hipStream_t st, int dtype, const DropoutArgs& a, int cus, hipError_t* error) {
    const uint32_t packets = (a.cols + kPacket - 1) / kPacket;
    const uint64_t blocks = (a.rows * packets + 255) / 256, most = 64 * (uint64_t)cus;
    const dim3 grid((uint32_t)(blocks < most ? blocks : most));
    if (dtype == MCCLX_F32) dropout_kernel<float><<<grid, dim3(256), 0, st>>>(a, packets);
    else if (dtype == MCCLX_F16) dropout_kernel<_Float16><<<grid, dim3(256), 0, st>>>(a, packets);
    else dropout_kernel<__bf16><<<grid, dim3(256), 0, st>>>(a, packets);
    *error = hipGetLastError();
    return *error == hipSuccess ? 1 : -1;
}

}  // namespace mcclx
