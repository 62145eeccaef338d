// loss_kernels.hip -- softmax cross entropy at the end of a language model, without keeping the logits.
//
//   z = h w^T  (tokens x vocab),  lse_i = log sum_v exp z_iv,  loss_i = lse_i - z_i,target
//   dz_iv = (exp(z_iv - lse_i) - [v = target_i]) g_i,  dh = dz w,  dw = dz^T h
//
// Forward: one product whose epilogue keeps, of each tile of logits, a maximum and a sum of exponentials
// a row; a small kernel joins them.  Backward, for pieces of the vocabulary: the same product again, whose epilogue
// writes dz of the piece in 16 bits; then the piece's rows of dw, which no other piece touches, and its share
// of dh, which adds up in fp32.  8 tokens x vocab x width flops in all, on the matrix cores.
//
// fp32 operands, dz among them, are split into three bf16 planes, x = x0 + x1 + x2 exactly, 8 bits each, and six products of planes, x1 y1,
// x0 y2, x2 y0, x0 y1, x1 y0, x0 y0, take the place of one: what is left out is at most 2^-24 of a product, one fp32 rounding.  (The
// matrix cores multiply fp32 at a sixteenth of bf16's rate.)  bf16 has fp32's exponents, so that a large row costs the others
// nothing; all that has to be seen to is that products neither overflow nor vanish, and a power of two that brings a matrix's largest
// value to 2^50 does that for values down to 2^-100 of it (fp32 itself cannot multiply all that it holds).  Two f16 planes and three
// products would take 0.6 of the time (4096 tokens, 32000 x 768, forward and backward 2.4 ms, this way 4.1), but hold 2^-49 of one
// common largest value: a row 2^34 times the others left those with 15 bits, one 2^50 times with none.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

#include "operators.h"

namespace mcclx {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
#define MCCLX_GLOBAL __attribute__((address_space(1)))
#define MCCLX_LDS __attribute__((address_space(3)))

// Element types of a product's operands: bf16, f16, or fp32 as three planes of bf16.  kDzScale: what dz, which lies in -1 .. 1, is multiplied
// by before it is rounded to them.  f16 has most of its numbers below 2^14, and its rare tokens' p keep 11 bits down to 2^-28; fp32's planes
// get the size of the matrices.
struct Bf16 { typedef __bf16 T; typedef bf16x4 T4; typedef bf16x8 T8; static constexpr int kPlanes = 1; static constexpr float kDzScale = 0x1p14f; };
struct F16 { typedef _Float16 T; typedef f16x4 T4; typedef f16x8 T8; static constexpr int kPlanes = 1; static constexpr float kDzScale = 0x1p14f; };
struct Split { typedef __bf16 T; typedef bf16x4 T4; typedef bf16x8 T8; static constexpr int kPlanes = 3; static constexpr float kDzScale = 0x1p50f; };
constexpr int kMostPlanes = 3;
// Of pass n of a split product, the planes of p and q, small terms first.
constexpr int kPasses = 6;
__device__ __forceinline__ uint32_t plane_of_p(uint32_t pass) { return 0x121 >> 2 * pass & 3; }   // 1 0 2 0 1 0
__device__ __forceinline__ uint32_t plane_of_q(uint32_t pass) { return 0x049 >> 2 * pass & 3; }   // 1 2 0 1 0 0

// c += a b on the matrix cores, c in accumulation registers.  Named here, because the compiler, left to choose, moves a
// tile's accumulators to and fro between the two register files in every step; volatile, so that a step's products,
// LDS reads and loads are issued in the order they are written in.  What the compiler otherwise sees to around these
// instructions: `settle`, and a and b come from LDS reads, never from an instruction right in front of them.
template <class E>
__device__ __forceinline__ void mfma(const i16x8& a, const i16x8& b, f32x4& c) {
    if constexpr (std::is_same_v<typename E::T, __bf16>)
        asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    else
        asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
// Loads 16 bytes a lane from a buffer straight into LDS at `to` + OFFSET (the same in all lanes) + 16 lane; what lies past
// the buffer's end, lane_offset and the scalar offset together, reads as zero.  In assembly, because the compiler would wait for all such loads at the next transposing
// read; they return nothing in registers, and `arrive` does the waiting.  (m0 and its use need an instruction between them.)
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <int OFFSET>
__device__ __forceinline__ void load_to_lds(uint32_t to, uint32_t lane_offset, const i32x4& buffer, uint32_t offset) {
    asm volatile("s_add_u32 m0, %0, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(to), "v"(lane_offset), "s"(buffer), "s"(offset), "n"(OFFSET) : "memory", "scc");
}

// f(0), f(1) ... f(N - 1), each number a constant of its own type.
template <class F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}

// ---- a 256 x 256 tile of out[q][p] = sum_k P[p][k] Q[q][k] ------------------------------
//
// Four waves, 128 x 128 each, in 256 accumulators a lane: at that size a step reads 64 KB of LDS for 1024 cycles of products, half of
// what LDS can give (eight waves of 128 x 64 would need three quarters, and the loads into it come on top).  K goes in steps of 32
// through four stages of LDS of 32 KB, filled by loads that go there directly, two to four steps ahead.  While a step is
// multiplied, the next one's operands are read into the other half of the wave's operand registers.
//
// An operand lies in memory with K innermost or with K outermost.  K outermost: a stage is [32][256] (of a small tile [32][128]), read
// with the transposing LDS read, the 32-byte unit u of row k at u ^ ((k & 3) | (k >> 1 & 4)).  K innermost: two stages are one
// [256][64], eight 16-byte chunks a row, chunk c of row r at c ^ (r & 7), because a load should take whole lines of 128 bytes
// (stage by stage they are halves, asked for twice: 1260 TFLOP/s of the logits' product, this way 1390).  Both keep the lanes of a read on
// different banks (no conflicts are counted).
//
// 8192 tokens, 131072 x 4096 bf16: logits 6.3 ms, 1390 TFLOP/s; dz 6.8, 1290; dw 5.9 and dh 6.0, 1500 and 1470, near the 1500 to 1580 that a large
// library product of bf16 reaches on this card, whose clock falls as its matrix cores fill (they are busy three quarters of dw's cycles).
// The logits' and dz's epilogues, 256 exponentials a lane, run with the matrix cores idle.  One block a CU going on to its next
// tile, whose first loads are under way meanwhile, was slower (26.0 ms in all, 25.8): its addresses do not fit the registers that the
// accumulators leave.
//
// Where there are few tokens or few tiles (large_tiles), tiles are 128 x 128, two blocks a CU: such a product is bound by the read of the
// weight, and twice as many blocks read it.  If even those are not more than the CUs, a block has its CU to itself, and eight stages: three pairs of
// them in flight in place of one (forward of 64 tokens, 32000 x 1024 bf16, 250 tiles: 22.5 us, with four stages 25.7; 512 tokens,
// 8192 x 2048: 27.3, 31.9; past that two blocks hide more, 64 tokens, 131072 x 1024, 1024 tiles: 65.4, 56.6).
constexpr int kTile = 256, kSmallTile = 128, kStep = 32, kStages = 4, kDeep = 8;
constexpr int kInner = 2 * kStep;  // what K has to be a multiple of where it is innermost
constexpr int stage_bytes(int tile) { return tile * kStep * 2; }  // of one operand

// One wave's loads of an operand: four (of a small tile two) a step with K outermost, twice as many every other step with K innermost.
template <bool K_OUTER, int TILE>
struct Loader {
    static constexpr int kLoads = K_OUTER ? TILE / 64 : TILE / 32, kRowLanes = TILE / 8, kSteps = K_OUTER ? 1 : 2, kStageBytes = stage_bytes(TILE);
    i32x4 from;         // the buffer of the next loads
    uint32_t advance_bytes;
    uint32_t records;   // bytes of a buffer: those the tile has from its first column on (K inner), or those of 32 rows (K outer)
    int32_t rows_left;  // (K outer)
    uint32_t ld_bytes, to;
    uint32_t lane_offset[K_OUTER ? 2 : 1];  // of this lane's chunks
    uint32_t row_offset[kLoads];

    // `n0`: the tile's first row (K inner) or column (K outer); `rows` of the operand in memory, `cols` elements each.
    __device__ __forceinline__ void init(uint32_t lds, uint32_t wave, uint64_t ld, uint32_t n0, uint32_t rows, uint32_t cols) {
        const uint32_t lane = threadIdx.x % 64;
        ld_bytes = (uint32_t)(ld * 2);
        to = lds + wave * (kLoads * 1024);
        if constexpr (K_OUTER) {
            advance_bytes = kStep * ld_bytes;
            records = advance_bytes - (ld_bytes - cols * 2) - n0 * 2;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t k = lane / kRowLanes + (TILE == 256 ? 2 * i : 0);  // (its lowest two bits)
                lane_offset[i] = (wave * 8 + lane / kRowLanes) * ld_bytes + ((lane % kRowLanes) ^ (k << 1) ^ ((wave & 1) << 3)) * 16;
            }
        } else {
            advance_bytes = 2 * kStep * 2;
            const uint32_t some = n0 >= rows ? 0 : rows - n0 < TILE ? rows - n0 : TILE;  // (none: a result is filled up to tiles of 256)
            records = some ? (some - 1) * ld_bytes + cols * 2 : 0;
            lane_offset[0] = (wave * (TILE / 4) + lane / 8) * ld_bytes + ((lane % 8) ^ (lane / 8)) * 16;
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) row_offset[i] = (K_OUTER ? 64 / kRowLanes * i : 8 * i) * ld_bytes;
    }
    // The steps from `step` on of a plane come next.
    __device__ __forceinline__ void start(const void* plane, uint32_t step, uint64_t ld, uint32_t n0, uint32_t rows) {
        const uint64_t at = (uint64_t)plane + (K_OUTER ? (uint64_t)n0 * 2 + (uint64_t)step * advance_bytes : (uint64_t)n0 * ld * 2 + step * (kStep * 2));
        const uint32_t gone = K_OUTER ? 0 : step * (kStep * 2);
        from = i32x4{__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32)),
                     __builtin_amdgcn_readfirstlane((int)(records > gone ? records - gone : 0)), 0x00027000};
        rows_left = K_OUTER ? (int32_t)(rows - step * kStep) : 0;
        if constexpr (K_OUTER) limit();
    }
    __device__ __forceinline__ void limit() {
        const int32_t some = rows_left < 0 ? 0 : rows_left < kStep ? rows_left : kStep;
        const int32_t n = (int32_t)records - (kStep - some) * (int32_t)ld_bytes;
        from[2] = __builtin_amdgcn_readfirstlane(n < 0 ? 0 : n);
    }
    // On to the next loads; `any` false: nothing of them is there.
    __device__ __forceinline__ void advance(bool any) {
        const uint64_t at = ((uint64_t)(uint32_t)from[1] << 32 | (uint32_t)from[0]) + advance_bytes;
        from[0] = (int)at;
        from[1] = (int)(at >> 32);
        if constexpr (K_OUTER) {
            rows_left -= kStep;
            rows_left = any ? rows_left : 0;
            limit();
        } else {
            from[2] = any && from[2] > (int32_t)advance_bytes ? from[2] - (int32_t)advance_bytes : 0;
        }
    }
    template <int STAGE, int I>
    __device__ __forceinline__ void load() const {  // load I of kLoads into a stage, or the pair of stages it belongs to
        load_to_lds<STAGE / kSteps * kSteps * kStageBytes + I * 1024>(to, lane_offset[K_OUTER ? I & 1 : 0], from, row_offset[I]);
    }
};

template <bool K_OUTER, int TILE>
struct Reader {
    static constexpr int kStageBytes = stage_bytes(TILE);
    static constexpr int kFrags = TILE / 32;
    uint32_t at[K_OUTER ? kFrags : 2];
    __device__ __forceinline__ void init(uint32_t lds, int part) {  // which half of the tile
        const int lane = threadIdx.x % 64;
        if constexpr (K_OUTER) {
            const int h = ((lane >> 2) & 3) | (((lane >> 4) & 1) << 2);
            const int k = (lane / 16) * 8 + (lane % 16) / 4;
#pragma unroll
            for (int f = 0; f < kFrags; ++f) at[f] = lds + k * (TILE * 2) + ((part * kFrags + f) ^ h) * 32 + (lane % 4) * 8;
        } else {
#pragma unroll
            for (int s = 0; s < 2; ++s) at[s] = lds + (part * (TILE / 2) + lane % 16) * 128 + (((s * 4 + lane / 16) ^ (lane & 7)) * 16);
        }
    }
    template <int STAGE>
    __device__ __forceinline__ i16x8 read(int i) const {
        if constexpr (K_OUTER) {
            MCCLX_LDS i16x4* const p = (MCCLX_LDS i16x4*)(uintptr_t)at[i] + STAGE * kStageBytes / 8;
            const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p + 4 * (TILE * 2) / 8);
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *((const MCCLX_LDS i16x8*)(uintptr_t)at[STAGE % 2] + (STAGE / 2 * 2 * kStageBytes + i * 16 * 128) / 16);
        }
    }
};

struct Operand {
    const void* plane[kMostPlanes];
    uint64_t ld;          // elements
    uint32_t rows, cols;  // in memory
};
struct GemmArgs {
    Operand p, q;
    uint32_t k;                // of one plane; a multiple of kInner where an operand has K inner
    uint32_t rows_out;         // q of the result (kStore, kPartial)
    uint32_t tiles_p, tiles_q;
    uint32_t splits;           // shares of K, each a number of whole steps
    // epilogues
    float *max_sum, *target_logit;  // [tiles_p][tokens][2], [tokens]
    const int64_t* target;
    const float *lse, *row_scale, *scales;  // scales: see Scale
    void* out[kMostPlanes];
    uint64_t out_ld;
    uint32_t first;         // vocabulary entry of p = 0 (logits)
    uint32_t vocab, tokens;
    int32_t add;            // partial sums: add to what is there
};
// Device floats behind `scales`.
enum Scale { kInverseHidden = 0, kInverseWeight = 1, kGradient = 2, kScales = 4 };

enum Epilogue { kLse, kDz, kStore, kPartial };

constexpr float kLog2e = 1.44269504f;
// e^(z - away), with `minus` = -away log2(e).  For 16-bit matrices one fused step, off by 2^-24 of the exponent, next to results of 8
// or 11 bits; for fp32 the exponent is carried in two parts.
template <class E>
__device__ __forceinline__ float exp_from(float z, float away, float minus) {
    if constexpr (E::kPlanes == 1) return __builtin_amdgcn_exp2f(__builtin_fmaf(z, kLog2e, minus));
    const float d = z - away, t = d * kLog2e;
    const float rest = __builtin_fmaf(d, 1.92596299e-8f, __builtin_fmaf(d, kLog2e, -t));  // log2(e) - kLog2e
    const float e = __builtin_amdgcn_exp2f(t);
    return d > -104.f ? __builtin_fmaf(e, rest * 0.693147181f, e) : e;  // (below e^-104 there is nothing to correct, and a -inf has no rest)
}
// The larger of two rows of 16 lanes' values, and of two halves', in both; their sums.
__device__ __forceinline__ float max_of_rows(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float sum_of_rows(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// A lane's four 16-bit values of two neighbouring fragments, lanes 16 apart holding the next four, become eight of one: lanes
// 0 .. 15 and 16 .. 31 get the first fragment's lower and upper half, the others the second one's.
template <class T4>
__device__ __forceinline__ i32x4 eight_of(const T4& first, const T4& second) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 a = __builtin_bit_cast(u32x2, first), b = __builtin_bit_cast(u32x2, second);
    i32x4 v;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const auto halves = __builtin_amdgcn_permlane32_swap(a[w], b[w], false, false);
        const auto rows = __builtin_amdgcn_permlane16_swap(halves[0], halves[1], false, false);
        v[w] = (int)rows[0];
        v[w + 2] = (int)rows[1];
    }
    return v;
}

template <class E, bool P_OUTER, bool Q_OUTER, Epilogue EPI, int TILE = kTile, int STAGES = kStages>
__global__ void __launch_bounds__(256, TILE == kTile || STAGES > kStages ? 1 : 2) gemm_kernel(GemmArgs a) {
    static_assert((TILE == kTile || P_OUTER == Q_OUTER) && (STAGES == kStages || !P_OUTER));
    constexpr int kStageBytes = stage_bytes(TILE), kWaveTile = TILE / 2, kFrags = kWaveTile / 16;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGES * kStageBytes];
    const uint32_t lds_p = (uint32_t)(uintptr_t)(MCCLX_LDS char*)lds, lds_q = lds_p + STAGES * kStageBytes;
    // Blocks go to the XCDs in turn: each XCD gets a run of tiles, eight tiles of q at a time, whose operands meet in its L2.
    const uint32_t tiles = a.tiles_p * a.tiles_q, split = blockIdx.x / tiles;
    uint32_t id = blockIdx.x - split * tiles;
    {
        const uint32_t xcd = id % 8, each = tiles / 8, more = tiles % 8;
        id = id / 8 + xcd * each + (xcd < more ? xcd : more);
    }
    const uint32_t group = id / (8 * a.tiles_p), in_group = id - group * 8 * a.tiles_p;
    const uint32_t rows = a.tiles_q - group * 8 < 8 ? a.tiles_q - group * 8 : 8;
    const uint32_t q0 = (group * 8 + in_group % rows) * TILE, p0 = in_group / rows * TILE;

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64, wave_p = wave % 2, wave_q = wave / 2;
    const uint32_t all = (a.k + kStep - 1) / kStep, share = ((all + a.splits - 1) / a.splits + STAGES - 1) / STAGES * STAGES;
    const uint32_t begin = split * share < all ? split * share : all, count = all - begin < share ? all - begin : share;
    constexpr bool kSplit = E::kPlanes > 1;
    constexpr uint32_t kTurns = kSplit ? kPasses : 1;
    constexpr int kPair = 2 * TILE / 32;              // loads of two stages, where both operands lie alike

    Loader<P_OUTER, TILE> load_p;
    Loader<Q_OUTER, TILE> load_q;
    load_p.init(lds_p, wave, a.p.ld, p0, a.p.rows, a.p.cols);
    load_q.init(lds_q, wave, a.q.ld, q0, a.q.rows, a.q.cols);
    Reader<P_OUTER, TILE> read_p;
    Reader<Q_OUTER, TILE> read_q;
    read_p.init(lds_p, wave_p);
    read_q.init(lds_q, wave_q);

    // Steps go by rounds, one a stage; those past the last are zeros.
    const uint32_t rounds = (count + STAGES - 1) / STAGES;
    uint32_t load_step = 0, load_pass = 0;  // the next step to load
    auto start = [&] {
        auto plane = [](const Operand& o, uint32_t n) { return !kSplit || n == 0 ? o.plane[0] : n == 1 ? o.plane[1] : o.plane[2]; };
        load_p.start(plane(a.p, plane_of_p(load_pass)), begin, a.p.ld, p0, a.p.rows);
        load_q.start(plane(a.q, plane_of_q(load_pass)), begin, a.q.ld, q0, a.q.rows);
    };
    auto advance = [&](int stage) {  // past the loads of a stage
        ++load_step;
        if (P_OUTER || stage % 2) load_p.advance(load_step < count);
        if (Q_OUTER || stage % 2) load_q.advance(load_step < count);
        if (kSplit && load_step == rounds * STAGES && load_pass + 1 < kTurns) {
            load_step = 0;
            ++load_pass;
            start();
        }
    };

    f32x4 acc[kFrags][kFrags];  // [p][q]
#pragma unroll
    for (int i = 0; i < kFrags; ++i)
#pragma unroll
        for (int j = 0; j < kFrags; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Between products and any other use of the accumulators: the wait that the matrix cores need, and no way round it.
    auto settle = [&] {
        asm volatile("s_nop 15\n\ts_nop 15");
#pragma unroll
        for (int i = 0; i < kFrags; ++i)
#pragma unroll
            for (int j = 0; j < kFrags; ++j) asm volatile("" : "+a"(acc[i][j]));
        asm volatile("s_nop 15");
    };

    i16x8 fp[2][kFrags], fq[2][kFrags];
    // In front of a step: what this wave has read is in registers, and of its loads those that the next step reads have
    // landed; then everybody's.  An operand with K innermost is loaded in every other step, in odd stages, once both
    // stages of a pair have been read, and with two of them nothing changes in front of even ones.
    auto arrive = [&](auto stage) {
        if constexpr (P_OUTER && Q_OUTER) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kPair) : "memory");
        else if constexpr (P_OUTER || Q_OUTER) {
            if constexpr (stage % 2) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        } else if constexpr (stage % 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((STAGES / 2 - 2) * kPair) : "memory");
    };

    if (count) {
        start();
        each<STAGES>([&](auto stage) {  // (a pair's loads in front of those of its second stage)
            if constexpr (!P_OUTER && stage % 2 == 0) each<load_p.kLoads>([&](auto i) { load_p.template load<stage, i>(); });
            if constexpr (!Q_OUTER && stage % 2 == 0) each<load_q.kLoads>([&](auto i) { load_q.template load<stage, i>(); });
            if constexpr (P_OUTER) each<load_p.kLoads>([&](auto i) { load_p.template load<stage, i>(); });
            if constexpr (Q_OUTER) each<load_q.kLoads>([&](auto i) { load_q.template load<stage, i>(); });
            advance(stage);
        });
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(P_OUTER != Q_OUTER ? 16 : (STAGES / 2 - 1) * kPair) : "memory");
#pragma unroll
        for (int i = 0; i < kFrags; ++i) {
            fp[0][i] = read_p.template read<0>(i);
            fq[0][i] = read_q.template read<0>(i);
        }
        settle();
        // The step in a stage, from one half of the registers; into the other, the next step; into LDS, in the place of what
        // every wave has read, the fourth step on.  Between two products a wave can issue three other instructions while the
        // first of them runs: the reads go behind every third product, the loads at even distances.
        auto step = [&](auto stage) {
            constexpr int kStage = stage, kNow = kStage % 2, kNext = (kStage + 1) % STAGES;
            constexpr int kLoadsP = P_OUTER || kStage % 2 ? load_p.kLoads : 0, kLoadsQ = Q_OUTER || kStage % 2 ? load_q.kLoads : 0;
            constexpr int kProducts = kFrags * kFrags, kReadEvery = kProducts * 3 / 4 / (2 * kFrags);
            arrive(stage);
            each<kProducts>([&](auto product) {
                constexpr int m = product, i = m % kFrags, j = m / kFrags;
                mfma<E>(fp[kNow][i], fq[kNow][j], acc[i][j]);
                constexpr int read = m / kReadEvery;
                if constexpr (m % kReadEvery == 0 && read < 2 * kFrags) {
                    if constexpr (read % 2 == 0) fp[kNow ^ 1][read / 2] = read_p.template read<kNext>(read / 2);
                    else fq[kNow ^ 1][read / 2] = read_q.template read<kNext>(read / 2);
                }
                if constexpr (kLoadsP + kLoadsQ > 0) {
                    constexpr int kEvery = kProducts * 3 / 4 / (kLoadsP + kLoadsQ), n = m / kEvery;
                    if constexpr (m % kEvery == (kEvery > 1) && n < kLoadsP + kLoadsQ) {
                        if constexpr (n < kLoadsP) load_p.template load<kStage, n>();
                        else load_q.template load<kStage, n - kLoadsP>();
                    }
                }
            });
            advance(stage);
        };
        for (uint32_t t = 0; t < rounds * kTurns; ++t) each<STAGES>(step);
        settle();
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // LDS is free

    // Lane: p = p_lane + 16 i + r, q = q_lane + 16 j.
    const uint32_t p_lane = p0 + wave_p * kWaveTile + lane / 16 * 4, q_lane = q0 + wave_q * kWaveTile + lane % 16;
    const uint32_t p_pair = p0 + wave_p * kWaveTile + lane / 32 * 16 + lane / 16 % 2 * 8;  // of eight_of's values
    if constexpr (EPI == kLse || EPI == kDz) {
        if constexpr (kSplit) {
            // (the product of both inverses may overflow where a logit does not)
            const float unit_h = a.scales[kInverseHidden], unit_w = a.scales[kInverseWeight], unit = unit_h * unit_w;
            const bool one = unit > 1e-36f && unit < 1e36f;
#pragma unroll
            for (int i = 0; i < kFrags; ++i)
#pragma unroll
                for (int j = 0; j < kFrags; ++j) acc[i][j] = one ? acc[i][j] * unit : acc[i][j] * unit_h * unit_w;
        }
        if (a.first + p0 + TILE > a.vocab) {  // entries past the end of the vocabulary count as -inf
#pragma unroll
            for (int i = 0; i < kFrags; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool in = a.first + p_lane + 16 * i + r < a.vocab;
#pragma unroll
                    for (int j = 0; j < kFrags; ++j) acc[i][j][r] = in ? acc[i][j][r] : -__builtin_inff();
                }
        }
    }
    // Which of this lane's 128 entries p_lane .. is the target of its row, -1: none.
    auto place_of = [&](int64_t target) {
        const int64_t past = target - (int64_t)(a.first + p_lane);
        return past >= 0 && past < kWaveTile && target < (int64_t)a.vocab && (past & 15) < 4 ? (int)past : -1;
    };
    if constexpr (EPI == kLse) {
        float* both = reinterpret_cast<float*>(lds);  // [TILE][2] of the waves with the upper half of p
        float top[kFrags], sum[kFrags];
#pragma unroll
        for (int j = 0; j < kFrags; ++j) {
            const uint32_t q = q_lane + 16 * j;
            const int place = place_of(q < a.tokens ? a.target[q] : -1);
            if (__any(place >= 0)) {  // (few tiles hold a token's target)
                float z = 0.f;
#pragma unroll
                for (int i = 0; i < kFrags; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) z = place == 16 * i + r ? acc[i][j][r] : z;
                if (place >= 0) a.target_logit[q] = z;
            }
            float m = -__builtin_inff();  // (a NaN shows in the sum)
#pragma unroll
            for (int i = 0; i < kFrags; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) m = __builtin_fmaxf(m, acc[i][j][r]);
            m = max_of_rows(m);
            const float away = m == -__builtin_inff() ? 0.f : m, minus = -away * kLog2e;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < kFrags; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += exp_from<E>(acc[i][j][r], away, minus);
            top[j] = m;
            sum[j] = sum_of_rows(s);
        }
        if (wave_p == 1 && lane < 16)
#pragma unroll
            for (int j = 0; j < kFrags; ++j) {
                const int at = (wave_q * kWaveTile + 16 * j + lane) * 2;
                both[at] = top[j];
                both[at + 1] = sum[j];
            }
        __syncthreads();
        if (wave_p == 0 && lane < 16)
#pragma unroll
            for (int j = 0; j < kFrags; ++j) {
                const int at = (wave_q * kWaveTile + 16 * j + lane) * 2;
                const float om = both[at], os = both[at + 1];
                const float m = __builtin_fmaxf(om, top[j]), away = m == -__builtin_inff() ? 0.f : m;
                const uint32_t q = q_lane + 16 * j;
                if (q < a.tokens) {
                    float* to = a.max_sum + ((uint64_t)(p0 / TILE) * a.tokens + q) * 2;
                    to[0] = m;
                    to[1] = sum[j] * expf(top[j] - away) + os * expf(om - away);
                }
            }
    } else if constexpr (EPI == kDz) {
        // For 16-bit matrices dz is rounded to their type: a product takes two operands of one type, and a second plane of dz would double
        // dw's and dh's time (12 ms of the 26 of 8192 tokens, 131072 x 4096).  Its price: gradients of 2047 tokens, 50001 x 1000 bf16 differ from those
        // of a 32-bit dz by 7e-4 and 5e-4 of their norm, where their own rounding to bf16 is 1.7e-3 of it.
#pragma unroll
        for (int j = 0; j < kFrags; ++j) {
            const uint32_t q = q_lane + 16 * j;
            const bool in = q < a.tokens;
            const float lse = in ? a.lse[q] : 0.f, scale = in ? a.row_scale[q] * E::kDzScale : 0.f, minus = -lse * kLog2e;
#pragma unroll
            for (int i = 0; i < kFrags; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = exp_from<E>(acc[i][j][r], lse, minus);
            const int place = place_of(in ? a.target[q] : -1);
            if (__any(place >= 0))  // (few tiles hold a token's target)
#pragma unroll
                for (int i = 0; i < kFrags; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[i][j][r] -= place == 16 * i + r ? 1.f : 0.f;
            // (where nothing flows, in padding too, the logits do not matter, NaN or not)
#pragma unroll
            for (int i = 0; i < kFrags; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = scale != 0.f ? acc[i][j][r] * scale : 0.f;
#pragma unroll
            for (int i = 0; i < kFrags; i += 2) {
                const uint64_t at = (uint64_t)q * a.out_ld + p_pair + 16 * i;
                f32x4 rest[2] = {acc[i][j], acc[i + 1][j]};
#pragma unroll
                for (int plane = 0; plane < E::kPlanes; ++plane) {
                    typename E::T4 part[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        part[k] = __builtin_convertvector(rest[k], typename E::T4);
                        rest[k] -= __builtin_convertvector(part[k], f32x4);
                    }
                    *reinterpret_cast<i32x4*>(static_cast<typename E::T*>(a.out[plane]) + at) = eight_of(part[0], part[1]);
                }
            }
        }
    } else if constexpr (EPI == kStore) {
        const float gradient = a.scales[kGradient], unit = kSplit ? a.scales[kInverseHidden] : 1.f;
        // (dz's power of two first, then the matrix's: the sum in the numbers it stands for, which fp32 holds)
        auto result = [&](const f32x4& v) { return v * (1.f / E::kDzScale) * unit * gradient; };
#pragma unroll
        for (int j = 0; j < kFrags; ++j) {
            const uint32_t q = q_lane + 16 * j;
            const bool in = q < a.rows_out;
            if constexpr (kSplit) {
                typedef f32x4 Loose __attribute__((aligned(4)));
                float* row = static_cast<float*>(a.out[0]) + (uint64_t)q * a.out_ld;
#pragma unroll
                for (int i = 0; i < kFrags; ++i) {
                    const uint32_t p = p_lane + 16 * i;
                    const f32x4 v = result(acc[i][j]);
                    if (in && p + 4 <= a.out_ld) {
                        *reinterpret_cast<Loose*>(row + p) = v;
                    } else if (in) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (p + r < a.out_ld) row[p + r] = v[r];
                    }
                }
            } else {
                typedef typename E::T T;
                typedef i32x4 Loose __attribute__((aligned(2)));
                T* row = static_cast<T*>(a.out[0]) + (uint64_t)q * a.out_ld;
#pragma unroll
                for (int i = 0; i < kFrags; i += 2) {
                    const uint32_t p = p_pair + 16 * i;
                    const i32x4 v = eight_of(__builtin_convertvector(result(acc[i][j]), typename E::T4),
                                             __builtin_convertvector(result(acc[i + 1][j]), typename E::T4));
                    if (in && p + 8 <= a.out_ld) {
                        *reinterpret_cast<Loose*>(row + p) = v;
                    } else if (in) {
                        const typename E::T8 each8 = __builtin_bit_cast(typename E::T8, v);
#pragma unroll
                        for (int r = 0; r < 8; ++r)
                            if (p + r < a.out_ld) row[p + r] = each8[r];
                    }
                }
            }
        }
    } else {
        float* sums = static_cast<float*>(a.out[0]) + (uint64_t)split * a.tiles_q * kTile * a.out_ld;  // rows padded to whole tiles
#pragma unroll
        for (int j = 0; j < kFrags; ++j) {
            const uint32_t q = q_lane + 16 * j;
            if (q >= a.rows_out) continue;
#pragma unroll
            for (int i = 0; i < kFrags; ++i) {
                f32x4* to = reinterpret_cast<f32x4*>(sums + (uint64_t)q * a.out_ld + p_lane + 16 * i);
                *to = a.add ? *to + acc[i][j] : acc[i][j];
            }
        }
    }
}

// ---- small kernels around it ---------------------------------------------------------------

// The sum of a value over a block of 1024 lanes, in each of them.
__device__ __forceinline__ float block_sum(float v, float* scratch) {
    for (int x = 32; x; x >>= 1) v += __shfl_xor(v, x);
    if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < 16; ++i) v += scratch[i];
    __syncthreads();
    return v;
}

struct JoinArgs {
    const float *max_sum, *target_logit;
    const int64_t* target;
    int64_t ignore;
    uint32_t parts, tokens, vocab;
    int mean;
    float *lse, *losses, *loss;
    uint32_t each;  // tokens a block
    bool whole;     // one block sees all of them, and makes the loss
};
// lse and loss of a block's `each` tokens, 16 or 64, from the tiles' parts: neighbouring lanes have neighbouring tokens, so that reads take
// whole lines, the other lanes and sixteen waves take the parts in turn, eight loads under way at a time (8192 tokens of 512 parts 10.5 us; a
// wave to a token, whose reads are eight bytes of a line, 32).  A target outside the vocabulary has no logit, and its loss is NaN.
__global__ void __launch_bounds__(1024) join_lse_kernel(JoinArgs a) {
    __shared__ float2 waves[16][64];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, q = blockIdx.x * a.each + lane % a.each;
    const bool mine = q < a.tokens && threadIdx.x < a.each;  // this lane ends with its token's lse
    const int64_t target = mine ? a.target[q] : a.ignore;
    const float logit = mine ? a.target_logit[q] : 0.f;      // (anything, where no tile holds the target)
    float m = -__builtin_inff(), s = 0.f;
    auto join = [&](const auto& parts) {  // (one maximum first, and the exponentials do not wait for each other)
        float top = m;
        for (const float2& p : parts) top = !(p.x <= top) ? p.x : top;
        const float away = top == -__builtin_inff() ? 0.f : top;
        s *= expf(m - away);
        for (const float2& p : parts) s += p.y * expf(p.x - away);
        m = top;
    };
    if (q < a.tokens)
        for (uint32_t i = threadIdx.x / a.each, step = 1024 / a.each; i < a.parts; i += 8 * step) {
            float2 parts[8];
#pragma unroll
            for (int k = 0; k < 8; ++k)
                parts[k] = i + k * step < a.parts ? reinterpret_cast<const float2*>(a.max_sum)[(uint64_t)(i + k * step) * a.tokens + q]
                                                  : make_float2(-__builtin_inff(), 0.f);
            join(parts);
        }
    for (uint32_t x = a.each; x < 64; x <<= 1) {
        const float2 other[1] = {make_float2(__shfl_xor(m, x), __shfl_xor(s, x))};
        join(other);
    }
    waves[wave][lane] = make_float2(m, s);
    __syncthreads();
    if (wave) return;
    float2 others[15];
#pragma unroll
    for (int w = 1; w < 16; ++w) others[w - 1] = waves[w][lane];
    join(others);
    float loss = 0.f;
    if (mine) {
        const float lse = m + logf(s);
        if (target != a.ignore) loss = target >= 0 && target < (int64_t)a.vocab ? lse - logit : __builtin_nanf("");
        a.lse[q] = lse;
        a.losses[q] = loss;
    }
    if (!a.whole) return;
    float count = target != a.ignore ? 1.f : 0.f;
    for (int x = 32; x; x >>= 1) {
        loss += __shfl_xor(loss, x);
        count += __shfl_xor(count, x);
    }
    if (lane == 0) *a.loss = a.mean ? loss / count : loss;
}
// The loss of all tokens, in one order (one block, 8192 tokens 4.8 us).
__global__ void __launch_bounds__(1024) reduce_loss_kernel(JoinArgs a) {
    __shared__ float scratch[16];
    float sum = 0.f, count = 0.f;  // (fewer than 2^24 tokens: the count is exact)
    for (uint32_t i = threadIdx.x; i < a.tokens; i += 1024) {
        sum += a.losses[i];
        count += a.target[i] == a.ignore ? 0.f : 1.f;
    }
    sum = block_sum(sum, scratch);
    count = block_sum(count, scratch);
    if (threadIdx.x == 0) *a.loss = a.mean ? sum / count : sum;
}

// What each row's dz is multiplied by, in -1 .. 1 (NaN where its target does not exist, as its loss is), and the factor
// that the gradients then lack (one block).  With a gradient a token, the factor is the largest finite one's size, and a row whose own is
// no number, or infinite, takes that as it is: it reaches that row of dhidden, and dweight, to which every row adds.
__global__ void __launch_bounds__(1024) row_scale_kernel(const float* grad, int reduction, const int64_t* target, int64_t ignore, uint32_t tokens,
                                                         uint32_t vocab, float* row_scale, float* scales) {
    __shared__ float scratch[16];
    auto there = [&](uint32_t i) { return target[i] >= 0 && target[i] < (int64_t)vocab ? 1.f : __builtin_nanf(""); };
    float factor;
    if (reduction == MCCLX_LOSS_NONE) {
        float top = 0.f;
        for (uint32_t i = threadIdx.x; i < tokens; i += 1024) {
            const float g = __builtin_fabsf(grad[i]);
            top = target[i] != ignore && __builtin_isfinite(g) ? __builtin_fmaxf(top, g) : top;
        }
        for (int x = 32; x; x >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, x));
        if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = top;
        __syncthreads();
        for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, scratch[i]);
        factor = top == 0.f ? 1.f : top;
        for (uint32_t i = threadIdx.x; i < tokens; i += 1024) {
            const float g = grad[i];
            row_scale[i] = target[i] == ignore ? 0.f : (__builtin_isfinite(g) ? g / factor : g) * there(i);
        }
    } else {
        float count = 0.f;
        for (uint32_t i = threadIdx.x; i < tokens; i += 1024) {
            const bool valid = target[i] != ignore;
            row_scale[i] = valid ? there(i) : 0.f;
            count += valid ? 1.f : 0.f;
        }
        count = block_sum(count, scratch);
        factor = reduction == MCCLX_LOSS_SUM ? *grad : count == 0.f ? 0.f : *grad / count;
    }
    if (threadIdx.x == 0) scales[kGradient] = factor;
}

// The lanes of a block over a matrix: 2^shift to a row, for rows of `packets` packets.
struct Spread {
    uint32_t shift, lane, row, rows;  // this lane's place in its row, its first row, rows from turn to turn
    __device__ __forceinline__ explicit Spread(uint32_t packets) {
        shift = packets > 1 ? 32 - __builtin_clz(packets - 1) : 0;
        shift = shift < 8 ? shift : 8;
        lane = threadIdx.x & ((1u << shift) - 1);
        row = blockIdx.x * (256u >> shift) + (threadIdx.x >> shift);
        rows = gridDim.x * (256u >> shift);
    }
};

// The matrices of a call that are copied for its products, `cols` of `wide` columns: hidden, weight or both in one launch, by blockIdx.y.
struct Copies {
    const void* from[2];
    uint64_t ld[2];
    uint32_t rows[2];
    void* to[2];              // (fp32: the planes, one behind the other)
    uint32_t inverse[2];      // fp32: which of `scales`
    uint32_t cols, wide;
    uint32_t* bits;           // fp32: kLargest floats' a matrix
    float* scales;
};
// A matrix whose rows the product can read: 16-byte aligned, padded with zeros (50001 x 1000 bf16 34 us, 5.9 TB/s).
template <class T>
__global__ void __launch_bounds__(256) pack_kernel(Copies a) {
    const T* const from = static_cast<const T*>(a.from[blockIdx.y]);
    T* const to = static_cast<T*>(a.to[blockIdx.y]);
    const uint64_t ld = a.ld[blockIdx.y];
    const uint32_t rows = a.rows[blockIdx.y], cols = a.cols, wide = a.wide;
    typedef T T8 __attribute__((ext_vector_type(8)));
    typedef T8 Loose __attribute__((aligned(sizeof(T))));
    const Spread at(wide / 8);
    for (uint64_t row = at.row; row < rows; row += at.rows)
        for (uint32_t c = at.lane; c < wide / 8; c += 1u << at.shift) {
            const T* p = from + row * ld + c * 8;
            T8 v = {};
            if (c * 8 + 8 <= cols) {
                v = *reinterpret_cast<const Loose*>(p);
            } else {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (c * 8 + r < cols) v[r] = p[r];
            }
            *reinterpret_cast<T8*>(to + row * wide + c * 8) = v;
        }
}

// Blocks that look for the largest value of a matrix: four a CU (32000 x 768 f32 25 us, 3.9 TB/s).
constexpr int kLargest = 1024;
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t largest_of_block(uint32_t v) {  // of 256 lanes
    __shared__ uint32_t waves[4];
    for (int x = 32; x; x >>= 1) v = larger(v, __shfl_xor(v, x));
    if (threadIdx.x % 64 == 0) waves[threadIdx.x / 64] = v;
    __syncthreads();
    return larger(larger(waves[0], waves[1]), larger(waves[2], waves[3]));
}
// The largest finite magnitude of a block's share of a matrix, as the bits of a float (which order as numbers do).
__global__ void __launch_bounds__(256) largest_kernel(Copies a) {
    const float* const from = static_cast<const float*>(a.from[blockIdx.y]);
    const uint64_t ld = a.ld[blockIdx.y];
    const uint32_t rows = a.rows[blockIdx.y], cols = a.cols;
    typedef f32x4 Loose __attribute__((aligned(4)));
    const Spread at((cols + 3) / 4);
    uint32_t top = 0;
    auto look = [&](float v) {
        const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
        top = b < 0x7F800000u ? larger(top, b) : top;
    };
    for (uint64_t row = at.row; row < rows; row += at.rows)
        for (uint32_t c = at.lane * 4; c < cols; c += 4u << at.shift) {
            const float* p = from + row * ld + c;
            if (c + 4 <= cols) {
                const f32x4 v = *reinterpret_cast<const Loose*>(p);
#pragma unroll
                for (int r = 0; r < 4; ++r) look(v[r]);
            } else {
                for (uint32_t r = 0; c + r < cols; ++r) look(p[r]);
            }
        }
    top = largest_of_block(top);
    if (threadIdx.x == 0) a.bits[blockIdx.y * kLargest + blockIdx.x] = top;
}
// The three bf16 planes of an fp32 matrix, and the inverse of its scale.
__global__ void __launch_bounds__(256) split_kernel(Copies a) {
    const float* const from = static_cast<const float*>(a.from[blockIdx.y]);
    __bf16* const to = static_cast<__bf16*>(a.to[blockIdx.y]);
    const uint64_t ld = a.ld[blockIdx.y];
    const uint32_t rows = a.rows[blockIdx.y], cols = a.cols, wide = a.wide;
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kLargest; i += 256) most = larger(most, a.bits[blockIdx.y * kLargest + i + threadIdx.x]);
    // 2^e with the largest value below 2^51 after it (a sum of 2^24 products of two such values stays below 2^126); 0 and the smallest
    // numbers get the largest e
    int e = 50 - ((int)(largest_of_block(most) >> 23) - 127);
    e = e > 126 ? 126 : e;
    const float s = __builtin_ldexpf(1.f, e);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.scales[a.inverse[blockIdx.y]] = __builtin_ldexpf(1.f, -e);
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    typedef f32x8 Loose __attribute__((aligned(4)));
    const Spread at(wide / 8);
    for (uint64_t row = at.row; row < rows; row += at.rows)
        for (uint32_t c = at.lane; c < wide / 8; c += 1u << at.shift) {
            const float* p = from + row * ld + c * 8;
            f32x8 v = {};
            if (c * 8 + 8 <= cols) {
                v = *reinterpret_cast<const Loose*>(p);
            } else {
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (c * 8 + r < cols) v[r] = p[r];
            }
            v *= s;
#pragma unroll
            for (int plane = 0; plane < Split::kPlanes; ++plane) {
                const bf16x8 part = __builtin_convertvector(v, bf16x8);
                *reinterpret_cast<bf16x8*>(to + ((uint64_t)plane * rows + row) * wide + c * 8) = part;
                const f32x8 rest = v - __builtin_convertvector(part, f32x8);
#pragma unroll
                for (int r = 0; r < 8; ++r) v[r] = __builtin_isfinite(v[r]) ? rest[r] : 0.f;  // (an infinity or a NaN is all in its first plane)
            }
        }
}

// dh from its partial sums, four columns a lane, eight loads under way at a time.
template <class E, class T>
__global__ void __launch_bounds__(256) join_hidden_kernel(const float* sums, uint32_t splits, uint64_t split_stride, uint32_t wide, uint32_t tokens,
                                                          uint32_t width, const float* scales, T* out) {
    const float gradient = scales[kGradient], unit = E::kPlanes > 1 ? scales[kInverseWeight] : 1.f;
    const Spread at((width + 3) / 4);
    for (uint64_t row = at.row; row < tokens; row += at.rows)
        for (uint32_t c = at.lane * 4; c < width; c += 4u << at.shift) {
            const float* from = sums + row * wide + c;  // (rows are whole tiles wide)
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            uint32_t s = 0;
            for (; s + 8 <= splits; s += 8) {
                f32x4 part[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) part[k] = *reinterpret_cast<const f32x4*>(from + (s + k) * split_stride);
#pragma unroll
                for (int k = 0; k < 8; ++k) v += part[k];
            }
            for (; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(from + s * split_stride);
            v = v * (1.f / E::kDzScale) * unit * gradient;
            T* to = out + row * width + c;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (c + r < width) to[r] = (T)v[r];
        }
}

uint32_t blocks_for(uint64_t items) {
    const uint64_t n = (items + 255) / 256;
    return (uint32_t)(n < 8192 ? n ? n : 1 : 8192);
}
uint64_t up(uint64_t n, uint64_t to) { return (n + to - 1) / to * to; }

// Where everything lies in the workspace of a call.
struct Plan {
    bool split, pack_h, pack_w;
    uint32_t wide;                    // columns of a packed operand
    uint32_t tiles_tokens, tiles_vocab;  // of 256
    uint32_t tile, cus;                  // of the logits' products; of the device
    uint64_t h, w;                    // packed operands (all planes), bytes from the start
    uint64_t scales, bits, row_scale, target_logit, losses, max_sum, dz, sums;
    uint32_t piece, splits, sum_wide; // vocabulary entries of a piece
    uint64_t bytes;
};
// Can the products read a matrix where it lies?  Rows of whole 128-byte lines, or they are copied to such rows, with zeros behind a width
// that is no multiple of kInner.  (The 50001 x 1000 bf16 weight could be read in place: each of its two products then takes 45 us
// more, and the copy takes 34.)
bool readable(const void* p, uint64_t ld, uint32_t width) {
    return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && width % kInner == 0 && ld < (1u << 20);
}
// How many of `tiles` columns of 256 x 256 tiles, `others` tiles each, are left so large.  A last round of them that keeps at most half of
// the CUs busy goes in small tiles instead, and so does an only one.  bf16, width 1024, forward: 200 tokens, vocabulary 32000 (125 tiles)
// 28 us, all of them large 35; 512, 19200 (150) 38, 38; 512, 32000 (250) 45, 40; 1024, 16400 (260) 52, 63; 1024, 24500 (384) 60, 65;
// 2047, 50001 (1568) 206, 215.  The weight's gradient of 1024, 16400: backward 154, 162.
uint32_t large_tiles(uint32_t tiles, uint32_t others, uint32_t cus) {
    const uint64_t all = (uint64_t)tiles * others, rounds = all / cus;
    const uint32_t large = (uint32_t)(rounds * cus / others);
    return (uint64_t)(tiles - large) * others * 2 <= cus ? large : tiles;
}
uint32_t large_logits(const Plan& l, uint32_t tiles) { return l.tile == kTile ? large_tiles(tiles, l.tiles_tokens, l.cus) : 0; }
// Tiles of the forward pass along the vocabulary.
uint32_t lse_parts(const Plan& l, uint32_t vocab) {
    const uint32_t large = large_logits(l, l.tiles_vocab);
    return large + (vocab > large * kTile ? (vocab - large * kTile + kSmallTile - 1) / kSmallTile : 0);
}
Plan plan_for(const LossArgs& a, bool backward, int cus) {
    Plan l = {};
    if (a.tokens == 0) return l;
    l.split = a.dtype == MCCLX_F32;
    l.cus = (uint32_t)cus;
    l.wide = (uint32_t)up(a.width, kInner);
    l.pack_h = l.split || !readable(a.hidden, a.hidden_ld, a.width);
    l.pack_w = l.split || !readable(a.weight, a.weight_ld, a.width);
    l.tiles_tokens = (uint32_t)up(a.tokens, kTile) / kTile;
    l.tiles_vocab = (uint32_t)up(a.vocab, kTile) / kTile;
    // (128 tokens, 131072 x 1024 bf16 forward: 60 us, in large tiles 75)
    l.tile = a.tokens <= kSmallTile || large_tiles(l.tiles_vocab, l.tiles_tokens, l.cus) == 0 ? kSmallTile : kTile;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        const uint64_t was = at;
        at += up(bytes, 256);
        return was;
    };
    const uint64_t planes = l.split ? Split::kPlanes : 1;
    l.scales = take(kScales * 4);
    if (l.split) l.bits = take(2 * kLargest * 4);
    if (l.pack_h) l.h = take(planes * a.tokens * l.wide * 2);
    if (l.pack_w) l.w = take(planes * a.vocab * l.wide * 2);
    if (!backward) {
        l.target_logit = take((uint64_t)a.tokens * 4);
        l.losses = take((uint64_t)a.tokens * 4);
        l.max_sum = take((uint64_t)lse_parts(l, a.vocab) * a.tokens * 8);
    } else {
        l.row_scale = take((uint64_t)a.tokens * 4);
        // dz of a piece: 512 MB, and at least 16 tiles.  (Backward of 4096 tokens, 50257 x 768 f32: 5.67 ms at 256 MB, which the last
        // cache holds, 4.91 at 512, 4.84 at 1024; of 8192, 131072 x 4096 bf16: 19.4, 19.4, 19.2.)
        const uint64_t rows = up(a.tokens, l.tile);
        uint64_t tiles = (512ull << 20) / (rows * kTile * 2 * planes);
        tiles = tiles < 16 ? 16 : tiles;
        tiles = tiles < l.tiles_vocab ? tiles : l.tiles_vocab;
        const uint64_t pieces = (l.tiles_vocab + tiles - 1) / tiles;
        l.piece = (uint32_t)((l.tiles_vocab + pieces - 1) / pieces) * kTile;
        l.dz = take(planes * rows * l.piece * 2);
        l.sum_wide = (uint32_t)up(a.width, kTile);
        const uint32_t tiles_h = l.tiles_tokens * (l.sum_wide / kTile);
        // dh has few tiles and a long sum: shares of it, as many as CUs go round, of at least eight steps (backward of 512 tokens,
        // 32000 x 1024 bf16, 155 us, unsplit 600; of 2047, 50001, 624, 1285)
        uint32_t splits = (uint32_t)cus / tiles_h;
        const uint32_t most = l.piece / kStep / 8;
        l.splits = splits < 1 ? 1 : splits < most ? splits : most ? most : 1;
        l.sums = take((uint64_t)l.splits * l.tiles_tokens * kTile * l.sum_wide * 4);
    }
    l.bytes = at;
    return l;
}

struct Run {
    hipStream_t st;
    hipError_t e = hipSuccess;
    int n = 0;
    void done() {
        ++n;
        const hipError_t now = hipGetLastError();
        if (e == hipSuccess) e = now;
    }
};

__global__ void __launch_bounds__(256) clear_kernel(uint16_t* p, uint64_t n) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256) p[i] = 0;
}
void clear(Run& r, void* p, uint64_t bytes) {
    clear_kernel<<<dim3(blocks_for(bytes / 2)), dim3(256), 0, r.st>>>(static_cast<uint16_t*>(p), bytes / 2);
    r.done();
}

// The operands as the products read them.
template <class E>
void operands(Run& r, const LossArgs& a, const Plan& l, char* work, Operand* h, Operand* w) {
    *h = {{a.hidden}, a.hidden_ld, a.tokens, a.width};
    *w = {{a.weight}, a.weight_ld, a.vocab, a.width};
    Copies c = {};
    c.cols = a.width;
    c.wide = l.wide;
    c.bits = reinterpret_cast<uint32_t*>(work + l.bits);
    c.scales = reinterpret_cast<float*>(work + l.scales);
    uint32_t n = 0;
    auto copy = [&](uint64_t at, int inverse, Operand* o) {
        c.from[n] = o->plane[0];
        c.ld[n] = o->ld;
        c.rows[n] = o->rows;
        c.to[n] = work + at;
        c.inverse[n] = inverse;
        for (int i = 0; i < E::kPlanes; ++i) o->plane[i] = work + at + (uint64_t)i * o->rows * l.wide * 2;
        o->ld = o->cols = l.wide;
        ++n;
    };
    if (l.pack_h) copy(l.h, kInverseHidden, h);
    if (l.pack_w) copy(l.w, kInverseWeight, w);
    if (n == 0) return;
    if constexpr (E::kPlanes > 1) {
        largest_kernel<<<dim3(kLargest, n), dim3(256), 0, r.st>>>(c);
        r.done();
        split_kernel<<<dim3(2048, n), dim3(256), 0, r.st>>>(c);
    } else {
        pack_kernel<typename E::T><<<dim3(2048, n), dim3(256), 0, r.st>>>(c);
    }
    r.done();
}

// The logits' product for `columns` vocabulary entries (a multiple of 128, or those that are left) and `rows` tokens: large tiles for the
// first `large` x 256 entries, small ones for the others, of which a CU holds two, or, where it gets one at most, one with loads further
// ahead.
template <class E, Epilogue EPI>
void logits(Run& r, GemmArgs g, const Plan& l, uint32_t large, uint64_t columns, uint64_t rows) {
    const dim3 block(256);
    if (large) {
        g.tiles_p = large;
        g.tiles_q = l.tiles_tokens;
        gemm_kernel<E, false, false, EPI><<<dim3(g.tiles_p * g.tiles_q), block, 0, r.st>>>(g);
        r.done();
    }
    const uint32_t done = large * kTile;
    if (columns <= done) return;
    for (int i = 0; i < E::kPlanes; ++i) {
        g.p.plane[i] = static_cast<const char*>(g.p.plane[i]) + (uint64_t)done * g.p.ld * 2;
        if (EPI == kDz) g.out[i] = static_cast<char*>(g.out[i]) + (uint64_t)done * 2;
    }
    g.p.rows = g.p.rows > done ? g.p.rows - done : 0;
    g.first += done;
    if (EPI == kLse) g.max_sum += (uint64_t)large * g.tokens * 2;
    g.tiles_p = (uint32_t)(up(columns - done, kSmallTile) / kSmallTile);
    g.tiles_q = (uint32_t)(up(rows, kSmallTile) / kSmallTile);
    const dim3 grid(g.tiles_p * g.tiles_q);
    if (grid.x <= l.cus) gemm_kernel<E, false, false, EPI, kSmallTile, kDeep><<<grid, block, 0, r.st>>>(g);
    else gemm_kernel<E, false, false, EPI, kSmallTile><<<grid, block, 0, r.st>>>(g);
    r.done();
}

template <class E>
void forward(Run& r, const LossArgs& a, const Plan& l) {
    char* work = static_cast<char*>(a.workspace);
    Operand h, w;
    operands<E>(r, a, l, work, &h, &w);
    GemmArgs g = {};
    g.p = w;
    g.q = h;
    g.k = l.wide;
    g.splits = 1;
    g.max_sum = reinterpret_cast<float*>(work + l.max_sum);
    g.target_logit = reinterpret_cast<float*>(work + l.target_logit);
    g.target = a.target;
    g.scales = reinterpret_cast<const float*>(work + l.scales);
    g.vocab = a.vocab;
    g.tokens = a.tokens;
    logits<E, kLse>(r, g, l, large_logits(l, l.tiles_vocab), a.vocab, a.tokens);
    // (more tokens a block where that makes one of it and saves a launch, unless it would have too much to read: forward of 64 tokens,
    // 32000 x 1024 bf16, 250 parts, 22.1, 22.6; 131072 x 1024, 1024 parts, stays at two)
    const uint32_t parts = lse_parts(l, a.vocab), each = a.tokens > 16 && a.tokens <= 64 && parts <= 512 ? 64 : 16;
    const JoinArgs join = {g.max_sum, g.target_logit, a.target, a.ignore_index, parts, a.tokens, a.vocab, a.reduction == MCCLX_LOSS_MEAN, a.lse,
                           a.reduction == MCCLX_LOSS_NONE ? a.loss : reinterpret_cast<float*>(work + l.losses), a.loss, each,
                           a.reduction != MCCLX_LOSS_NONE && a.tokens <= each};
    join_lse_kernel<<<dim3((a.tokens + each - 1) / each), dim3(1024), 0, r.st>>>(join);
    r.done();
    if (a.reduction != MCCLX_LOSS_NONE && !join.whole) {
        reduce_loss_kernel<<<dim3(1), dim3(1024), 0, r.st>>>(join);
        r.done();
    }
}

template <class E>
void backward(Run& r, const LossArgs& a, const Plan& l) {
    typedef typename E::T T;
    typedef std::conditional_t<(E::kPlanes > 1), float, T> Out;
    char* work = static_cast<char*>(a.workspace);
    Operand h, w;
    operands<E>(r, a, l, work, &h, &w);
    float* scales = reinterpret_cast<float*>(work + l.scales);
    float* row_scale = reinterpret_cast<float*>(work + l.row_scale);
    row_scale_kernel<<<dim3(1), dim3(1024), 0, r.st>>>(a.grad, a.reduction, a.target, a.ignore_index, a.tokens, a.vocab, row_scale, scales);
    r.done();
    const uint64_t rows = up(a.tokens, l.tile);
    Operand dz = {{}, l.piece, (uint32_t)rows, l.piece};
    for (int i = 0; i < E::kPlanes; ++i) dz.plane[i] = work + l.dz + i * rows * l.piece * 2;
    for (uint32_t first = 0; first < a.vocab; first += l.piece) {
        const uint32_t some = a.vocab - first < l.piece ? a.vocab - first : l.piece;
        Operand wp = w;
        wp.rows = some;
        for (int i = 0; i < E::kPlanes; ++i) wp.plane[i] = static_cast<const char*>(w.plane[i]) + (uint64_t)first * w.ld * 2;
        GemmArgs g = {};
        g.p = wp;
        g.q = h;
        g.k = l.wide;
        g.splits = 1;
        g.target = a.target;
        g.lse = a.lse_in;
        g.row_scale = row_scale;
        g.scales = scales;
        for (int i = 0; i < E::kPlanes; ++i) g.out[i] = const_cast<void*>(dz.plane[i]);
        g.out_ld = l.piece;
        g.first = first;
        g.vocab = a.vocab;
        g.tokens = a.tokens;
        logits<E, kDz>(r, g, l, large_logits(l, (uint32_t)(up(some, kTile) / kTile)), up(some, kTile), rows);
        if (a.dweight) {
            GemmArgs d = {};
            d.p = h;
            d.q = dz;
            d.k = a.tokens;
            d.rows_out = some;
            d.splits = 1;
            d.scales = scales;
            d.out[0] = static_cast<Out*>(a.dweight) + (uint64_t)first * a.width;
            d.out_ld = a.width;
            const uint32_t wide = (a.width + kTile - 1) / kTile, tiles = (uint32_t)(up(some, kTile) / kTile), large = large_tiles(tiles, wide, l.cus);
            if (large) {
                d.tiles_p = wide;
                d.tiles_q = large;
                gemm_kernel<E, true, true, kStore><<<dim3(d.tiles_p * d.tiles_q), dim3(256), 0, r.st>>>(d);
                r.done();
            }
            if (large < tiles) {
                const uint32_t done = large * kTile;
                for (int i = 0; i < E::kPlanes; ++i) d.q.plane[i] = static_cast<const char*>(dz.plane[i]) + (uint64_t)done * 2;
                d.q.cols -= done;
                d.rows_out -= done;
                d.out[0] = static_cast<Out*>(d.out[0]) + (uint64_t)done * a.width;
                d.tiles_p = (a.width + kSmallTile - 1) / kSmallTile;
                d.tiles_q = (d.rows_out + kSmallTile - 1) / kSmallTile;
                gemm_kernel<E, true, true, kStore, kSmallTile><<<dim3(d.tiles_p * d.tiles_q), dim3(256), 0, r.st>>>(d);
                r.done();
            }
        }
        if (a.dhidden) {
            GemmArgs d = {};
            d.p = wp;
            d.q = dz;
            d.k = (uint32_t)up(some, kInner);
            d.rows_out = a.tokens;
            d.tiles_p = l.sum_wide / kTile;
            d.tiles_q = l.tiles_tokens;
            d.splits = l.splits;
            d.out[0] = work + l.sums;
            d.out_ld = l.sum_wide;
            d.add = first > 0;
            gemm_kernel<E, true, false, kPartial><<<dim3(d.tiles_p * d.tiles_q * d.splits), dim3(256), 0, r.st>>>(d);
            r.done();
        }
    }
    if (a.dhidden) {
        join_hidden_kernel<E, Out><<<dim3(a.tokens < 4096 ? a.tokens : 4096), dim3(256), 0, r.st>>>(
            reinterpret_cast<const float*>(work + l.sums), l.splits, (uint64_t)l.tiles_tokens * kTile * l.sum_wide, l.sum_wide, a.tokens, a.width, scales,
            static_cast<Out*>(a.dhidden));
        r.done();
    }
}

}  // namespace

uint64_t loss_workspace_bytes(const LossArgs& a, bool backward, int cus) { return plan_for(a, backward, cus).bytes; }

int launch_loss(hipStream_t st, const LossArgs& a, bool back, int cus, hipError_t* error) {
    const Plan l = plan_for(a, back, cus);
    Run r{st};
    if (a.tokens == 0) {  // the loss of nothing, and a weight that nothing reaches
        if (back && a.dweight) clear(r, a.dweight, (uint64_t)a.vocab * a.width * (a.dtype == MCCLX_F32 ? 4 : 2));
        if (!back && a.reduction != MCCLX_LOSS_NONE) {
            JoinArgs none = {};
            none.mean = a.reduction == MCCLX_LOSS_MEAN;
            none.loss = a.loss;
            reduce_loss_kernel<<<dim3(1), dim3(1024), 0, st>>>(none);
            r.done();
        }
        *error = r.e;
        return r.e == hipSuccess ? r.n : -1;
    }
    if (a.dtype == MCCLX_BF16) back ? backward<Bf16>(r, a, l) : forward<Bf16>(r, a, l);
    else if (a.dtype == MCCLX_F16) back ? backward<F16>(r, a, l) : forward<F16>(r, a, l);
    else back ? backward<Split>(r, a, l) : forward<Split>(r, a, l);
    *error = r.e;
    return r.e == hipSuccess ? r.n : -1;
}

}  // namespace mcclx
