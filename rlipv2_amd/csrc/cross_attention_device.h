// cross_attention_device.h -- what the forward and backward kernels of cross attention share (gfx950, wave64).
//
// Every product is one shape: a STREAMED side, tiles of rows in LDS, against 32 RESIDENT rows per wave in registers.  With the
// streamed rows as operand A and the resident ones as operand B of the 32x32 matrix instructions, the result has one resident
// row per lane (lane & 31) and 16 streamed rows in its registers.  That result, rounded to the operands' type, IS an operand B
// again: the contraction over the streamed rows may run in any order, and the order the registers have is taken (slot e of
// half h = lane >> 5 and step u is streamed row 16 u + (e & 3) + 8 (e >> 2) + 4 h).  So the probabilities never leave the
// registers, the sums and maxima of a softmax row are sums over a lane's registers plus one exchange between the two halves,
// and the second product only needs the streamed tile transposed, which ds_read_b64_tr_b16 does on the way out of LDS.
//
// LDS tile: row-major, 16-byte chunks, chunk c of row r in slot c ^ swizzle(r).  The swizzle separates both access patterns over
// the banks: the operand-A reads (8 consecutive rows, one chunk each: 8 different bank groups) and the transposing reads
// (4 rows, two neighbouring chunks each: 8 different bank groups).  Global memory is copied in by LDS-DMA, which puts lane i's
// 16 bytes at base + 16 i; the swizzle is therefore applied to the lane's SOURCE address.  The lanes of rows that must not count
// (padding, behind the end) write zeros instead: a NaN or infinity in a masked row reaches no product.
//
// float32 runs the same code on v_mfma_f32_32x32x2_f32: eight of them contract what one 32x32x16 does, element e of both halves
// at a time.
#pragma once
#include <hip/hip_runtime.h>
#ifdef MSDA_EMU
#include <vector>
#endif
#include <stdint.h>

#include "../../include/rlipv2_attention.h"
#include "../../include/rlipv2_msda.h"
#include "msda_device.h"
#include "once_per_device.h"

// (tools/emu/ compiles the kernel files for the CPU against a lane-level model of the workgroup and defines these itself)
#ifndef MSDA_DYNAMIC_LDS
#define MSDA_DYNAMIC_LDS(type, name) extern __shared__ __attribute__((aligned(16))) type name[]
#endif

namespace xattn {

using namespace msda;

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) __bf16 bf16x4;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr float kInf = __builtin_inff();

#ifdef MSDA_EMU
inline float exp2_fast(float x) { return exp2f(x); }
inline float log2_fast(float x) { return log2f(x); }
#else
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }      // v_exp_f32
__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }       // v_log_f32: base 2
#endif

// two floats -> packed bfloat16 pair, round to nearest even (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack2(float a, float b)
{
#ifdef MSDA_EMU
    return pack_bf16x2(a, b);
#else
    const f32x2 f = {a, b};
    const bf16x2 h = __builtin_convertvector(f, bf16x2);
    uint32_t u;
    __builtin_memcpy(&u, &h, 4);
    return u;
#endif
}

// streamed row -> XOR of its chunk slots (CPR: chunks per row)
template <int CPR> __device__ __forceinline__ int swizzle(int row)
{
    return CPR >= 8 ? (((row & 3) << 1) | ((row >> 2) & 1)) : ((row & 2) | ((row >> 2) & 1));
}

// ---- 8 consecutive contraction elements of one row per lane -------------------------------------------------------------
template <typename T> struct Frag;
template <> struct Frag<bf16_t> { union { uint4 u; uint32_t w[4]; uint2 half[2]; bf16x8 v; }; };
template <> struct Frag<float> { union { float4 u[2]; float f[8]; }; };

__device__ __forceinline__ void mma(const Frag<bf16_t> &a, const Frag<bf16_t> &b, f32x16 &c)
{
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
__device__ __forceinline__ void mma(const Frag<float> &a, const Frag<float> &b, f32x16 &c)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.f[e], b.f[e], c, 0, 0, 0);
}

// registers 8u .. 8u + 7 of a result as an operand
__device__ __forceinline__ void to_operand(const float (&p)[8], Frag<bf16_t> &f)
{
#pragma unroll
    for (int e = 0; e < 4; ++e) f.w[e] = pack2(p[2 * e], p[2 * e + 1]);
}
__device__ __forceinline__ void to_operand(const float (&p)[8], Frag<float> &f)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) f.f[e] = p[e];
}
// what the rounding took: a second operand, whose product brings the first one's to float32's precision but for 2^-17
__device__ __forceinline__ void rest_operand(const float (&p)[8], const Frag<bf16_t> &f, Frag<bf16_t> &rest)
{
#pragma unroll
    for (int e = 0; e < 4; ++e) rest.w[e] = pack2(p[2 * e] - bf16_lo(f.w[e]), p[2 * e + 1] - bf16_hi(f.w[e]));
}
__device__ __forceinline__ void rest_operand(const float (&)[8], const Frag<float> &, Frag<float> &) {}

// Before a loop: the compiler waits for these registers' loads HERE.  Left to itself it puts the wait in front of the first use,
// inside the loop, where it would wait for the copies of the next tile in every iteration.
#ifdef MSDA_EMU
template <typename F> inline void settle(F &) {}
#define XATTN_SCHED_GROUP(mask, size) do { } while (0)
#else
__device__ __forceinline__ void settle(Frag<bf16_t> &f) { asm volatile("" : "+v"(f.v)); }
__device__ __forceinline__ void settle(Frag<float> &f)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) asm volatile("" : "+v"(f.f[e]));
}
// the next `size` instructions of a kind in the schedule (0x8: matrix instructions, 0x100: LDS reads)
#define XATTN_SCHED_GROUP(mask, size) __builtin_amdgcn_sched_group_barrier(mask, size, 0)
#endif
// Schedule of a run of N operand reads (R LDS reads each) and the MM matrix instructions that take each of them: the reads stay up to
// DEPTH operands ahead.  Left to itself the compiler reads one operand, waits, multiplies.
template <bool ON, int N, int R, int MM> __device__ __forceinline__ void ahead()
{
    if constexpr (ON) {
        constexpr int MOST = MM <= 2 ? 4 : 2, DEPTH = N < MOST ? N : MOST;
        XATTN_SCHED_GROUP(0x100, DEPTH * R);
#pragma unroll
        for (int i = 0; i < N - DEPTH; ++i) {
            XATTN_SCHED_GROUP(0x8, MM);
            XATTN_SCHED_GROUP(0x100, R);
        }
        XATTN_SCHED_GROUP(0x8, DEPTH * MM);
    }
}

// operand from global memory: 8 elements at `d0`, zeros where !ok or behind the head size.  `row` can be read in either case: the load
// is not behind a branch, so that all of a row's loads are on their way together.
__device__ __forceinline__ void load_operand(const bf16_t *row, int d0, int D, bool ok, Frag<bf16_t> &f)
{
    const uint4 x = *reinterpret_cast<const uint4 *>(row + min(d0, D - 8));
    const uint32_t keep = ok && d0 < D ? ~0u : 0u;
    f.u = make_uint4(x.x & keep, x.y & keep, x.z & keep, x.w & keep);
}
__device__ __forceinline__ void load_operand(const float *row, int d0, int D, bool ok, Frag<float> &f)
{
    const float *p = row + min(d0, D - 8);
    f.u[0] = *reinterpret_cast<const float4 *>(p);
    f.u[1] = *reinterpret_cast<const float4 *>(p + 4);
    const bool in = ok && d0 < D;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.f[e] = in ? f.f[e] : 0.f;
}
__device__ __forceinline__ float dot8(const Frag<bf16_t> &a, const Frag<bf16_t> &b)
{
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) s = fmaf(bf16_lo(a.w[e]), bf16_lo(b.w[e]), fmaf(bf16_hi(a.w[e]), bf16_hi(b.w[e]), s));
    return s;
}
__device__ __forceinline__ float dot8(const Frag<float> &a, const Frag<float> &b)
{
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(a.f[e], b.f[e], s);
    return s;
}

// ---- LDS tiles ------------------------------------------------------------------------------------------------------------
template <typename T, int DP> struct Tile {
    static constexpr int EPC = 16 / (int)sizeof(T);        // elements per chunk
    static constexpr int CPR = DP / EPC;                   // chunks per row
    static constexpr int ROW = DP * (int)sizeof(T);        // bytes per row
};

// (The swizzle changes a chunk's low three bits only: what the loop counters add above them is written as a constant byte offset,
// which the read instruction takes, instead of one address register per read.)
// operand A = streamed row `row` of the tile, contraction elements 16 s + 8 (lane >> 5) ..
template <int DP> __device__ __forceinline__ void read_rows(const char *tile, int row, int s, int half, Frag<bf16_t> &f)
{
    constexpr int CPR = Tile<bf16_t, DP>::CPR;
    const char *p = tile + row * Tile<bf16_t, DP>::ROW + ((2 * (s & 3) + half) ^ swizzle<CPR>(row)) * 16;
    f.u = *reinterpret_cast<const uint4 *>(p + (s >> 2) * 128);
}
template <int DP> __device__ __forceinline__ void read_rows(const char *tile, int row, int s, int half, Frag<float> &f)
{
    constexpr int CPR = Tile<float, DP>::CPR;
    const int c = 4 * (s & 1) + 2 * half, x = swizzle<CPR>(row);
    const char *p = tile + row * Tile<float, DP>::ROW + (s >> 1) * 128;
    f.u[0] = *reinterpret_cast<const float4 *>(p + (c ^ x) * 16);
    f.u[1] = *reinterpret_cast<const float4 *>(p + ((c + 1) ^ x) * 16);
}

#ifdef MSDA_EMU
inline uint2 read_tr(const char *p)
{
    const emu_s16x4 v = emu_tr_read(MSDA_LDS_BYTE_ADDR(p), 0);
    uint2 u;
    std::memcpy(&u, &v, 8);
    return u;
}
#else
__device__ __forceinline__ uint2 read_tr(const char *p)
{
    typedef __attribute__((ext_vector_type(4))) short s16x4;
    typedef __attribute__((address_space(3))) s16x4 *lds_p;
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(p));
    uint2 u;
    __builtin_memcpy(&u, &v, 8);
    return u;
}
#endif

// operand A = the TRANSPOSED tile: lane -> head element 32 dt + (lane & 31), contraction over the streamed rows
// base + 16 u + (e & 3) + 8 (e >> 2) + 4 (lane >> 5)
template <int DP> __device__ __forceinline__ void read_columns(const char *tile, int base, int dt, int lane, Frag<bf16_t> &f)
{
    constexpr int CPR = Tile<bf16_t, DP>::CPR, ROW = Tile<bf16_t, DP>::ROW;
    const int row = 4 * (lane >> 5) + ((lane & 15) >> 2);               // (base: a multiple of 16, the same swizzle)
    const int chunk = (dt & 1) * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    const char *p = tile + row * ROW + ((chunk ^ swizzle<CPR>(row)) * 16) + (lane & 1) * 8 + base * ROW + (dt >> 1) * 128;
    f.half[0] = read_tr(p);
    f.half[1] = read_tr(p + 8 * ROW);                                   // (row + 8: the same swizzle)
}
template <int DP> __device__ __forceinline__ void read_columns(const char *tile, int base, int dt, int lane, Frag<float> &f)
{
    constexpr int CPR = Tile<float, DP>::CPR, ROW = Tile<float, DP>::ROW;
    const int d = lane & 31;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int row = (e & 3) + 4 * (lane >> 5);                      // (8 and base rows further: the same swizzle)
        const char *p = tile + row * ROW + (((d >> 2) ^ swizzle<CPR>(row)) * 16) + (d & 3) * 4;
        f.f[e] = *reinterpret_cast<const float *>(p + (base + 8 * (e >> 2)) * ROW + dt * 128);
    }
}

// rows of a query-side operand: the G heads that share a key head follow each other, row r = head g = r / Lq, token r - g Lq
struct Rows {
    int Lq, heads_per_kv, count;          // count = G * Lq
    __device__ __forceinline__ void split(int r, int &g, int &q) const
    {
        if (heads_per_kv == 1) { g = 0; q = r; }
        else { g = r / Lq; q = r - g * Lq; }
    }
};

// One LDS-DMA instruction: lane i copies 16 bytes from base (the same for the whole wave) + its offset to lds_base + 16 i; lanes
// that are switched off leave their 16 bytes alone.  Written as inline assembly (it has no register output): behind the builtin the
// compiler waits for EVERY outstanding copy before the next LDS read, which would end the overlap of a tile's copy with the tile
// before.  copies_done() is the wait.
#ifdef MSDA_EMU
// (nothing arrives before it has been waited for: a wait that is missing shows)
struct Copy { const char *from; char *to; };
inline std::vector<Copy> &copies_under_way() { thread_local std::vector<Copy> list; return list; }
inline void copy16(const char *base, uint32_t offset, char *lds_base) { copies_under_way().push_back({base + offset, lds_base}); }
inline void copies_done()
{
    for (const Copy &c : copies_under_way()) MSDA_GLOBAL_LOAD_LDS16(c.from, c.to);
    copies_under_way().clear();
}
#else
// (M0 is written here and by nothing that would expect it back: the compiler sets it right before an instruction that reads it)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy16(const char *base, uint32_t offset, char *lds_base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(__builtin_amdgcn_readfirstlane((int)MSDA_LDS_BYTE_ADDR(lds_base))), "v"(offset), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void copies_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
#endif

// Copies tiles of ROWS rows of a [*, D] operand into LDS (not waited for).  A thread's offsets inside a tile are the same for every
// tile (the C entry checks that 64 rows span less than 4 GB); the tile's base is a scalar.
template <typename T, int DP, int ROWS, int THREADS> struct Stager {
    static constexpr int CPR = Tile<T, DP>::CPR, EPC = Tile<T, DP>::EPC, TOTAL = ROWS * CPR, ITERATIONS = TOTAL / THREADS;
    static constexpr int RPI = THREADS / CPR;                         // rows per iteration
    static constexpr int NV = RPI >= 8 ? 1 : 8 / RPI < ITERATIONS ? 8 / RPI : ITERATIONS;      // the swizzle repeats every 8 rows
    static constexpr unsigned long long ALL = ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1;
    static_assert(TOTAL % THREADS == 0 && THREADS % CPR == 0, "whole rows");
    int64_t step;                                                     // bytes from one iteration's rows to the next's
    uint32_t offset[NV];
    int row0, slot, tid;
    bool whole_head;
    int D;
    __device__ __forceinline__ void init(int64_t row_stride, int tid_, int D_)
    {
        const uint32_t row_bytes = (uint32_t)(row_stride * (int64_t)sizeof(T));
        tid = tid_;
        D = D_;
        whole_head = D == DP;
        row0 = tid / CPR;
        slot = tid % CPR;
        step = (int64_t)RPI * row_bytes;
#pragma unroll
        for (int j = 0; j < NV; ++j) offset[j] = (uint32_t)row0 * row_bytes + (uint32_t)((slot ^ swizzle<CPR>(row0 + j * RPI)) * 16);
    }
    // `first`: the tile's first row; bit i of `word`: row i counts (the others become zeros, as does what is behind the head size)
    __device__ __forceinline__ void copy(char *tile, const T *first, unsigned long long word) const
    {
        char *wave_base = tile + (tid & ~63) * 16;
        const char *base = reinterpret_cast<const char *>(first);
        if (word == ALL && whole_head) {
#pragma unroll
            for (int it = 0; it < ITERATIONS; ++it, base += step) copy16(base, offset[it % NV], wave_base + it * THREADS * 16);
        } else {
#pragma unroll
            for (int it = 0; it < ITERATIONS; ++it, base += step) {
                const int row = row0 + it * RPI, chunk = slot ^ swizzle<CPR>(row);
                if (((word >> row) & 1) && chunk * EPC < D) copy16(base, offset[it % NV], wave_base + it * THREADS * 16);
                else *reinterpret_cast<uint4 *>(tile + (it * THREADS + tid) * 16) = make_uint4(0, 0, 0, 0);
            }
        }
    }
};

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// Workgroups are dealt to the 8 dies round-robin; give every die a contiguous range of tasks, so that the workgroups that read
// the same keys (or rows) share its L2.
__device__ __forceinline__ int task_of(int id, int total)
{
    const int die = id & 7, slot = id >> 3, per = total >> 3, rest = total & 7;
    return die * per + min(die, rest) + slot;
}

// ---- keys that count -----------------------------------------------------------------------------------------------------
struct KeyMask {
    const uint8_t *padding;               // this sequence's row, or null
    int length;                           // keys [0, length)
    __device__ __forceinline__ void init(const cross_attention_args &a, int b)
    {
        padding = a.padding ? static_cast<const uint8_t *>(a.padding) + (int64_t)b * a.padding_stride : nullptr;
        length = a.lengths ? max(0, min(a.Lk, static_cast<const int *>(a.lengths)[b])) : a.Lk;
    }
    // A softmax over one key does not depend on the query: dS is 0, where P (dP - delta) is what the two sums' orders leave.
    __device__ __forceinline__ bool one() const { return length == 1; }
    // (the byte is loaded a tile ahead of the ballot that needs it)
    __device__ __forceinline__ int load(int key) const { return key < length ? (padding ? (int)padding[key] : 0) : 1; }
};

template <typename T> __device__ __forceinline__ void store4(T *p, float a, float b, float c, float d);
template <> __device__ __forceinline__ void store4<bf16_t>(bf16_t *p, float a, float b, float c, float d)
{
    *reinterpret_cast<uint2 *>(p) = make_uint2(pack2(a, b), pack2(c, d));
}
template <> __device__ __forceinline__ void store4<float>(float *p, float a, float b, float c, float d)
{
    *reinterpret_cast<float4 *>(p) = make_float4(a, b, c, d);
}

// the 16 streamed rows of a result's registers, from a float per row (p: row 4 (lane >> 5) of the 32)
__device__ __forceinline__ void load_quads(const float *p, f32x16 &v)
{
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const float4 x = *reinterpret_cast<const float4 *>(p + 8 * g);
        v[4 * g] = x.x; v[4 * g + 1] = x.y; v[4 * g + 2] = x.z; v[4 * g + 3] = x.w;
    }
}

// x - bf16(x), exact in float32
__device__ __forceinline__ void rounded_off(float (&x)[4])
{
    const uint32_t a = pack2(x[0], x[1]), b = pack2(x[2], x[3]);
    x[0] -= bf16_lo(a); x[1] -= bf16_hi(a); x[2] -= bf16_lo(b); x[3] -= bf16_hi(b);
}

template <int N> __device__ __forceinline__ void clear(f32x16 (&a)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) a[i][r] = 0.f;
}

template <int N> __device__ __forceinline__ void zero_unless(bool keep, f32x16 (&a)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) a[i][r] = keep ? a[i][r] : 0.f;
}

// The result's 32 rows (lane = resident row, registers = head elements) times `f` to global memory, through LDS: a register holds 8 or
// 16 bytes of 32 different rows, whole rows go out 16 bytes a lane.  `region`: BYTES of LDS of this wave; `dense`: the lane's own row
// as an element offset from `out`, -1 for a row that is not there.  A wave writes and reads its own region only.
// LOW: what rounding takes from those values instead.
template <typename OutT, int DP, int BYTES, bool LOW = false>
__device__ __forceinline__ void put_rows(const f32x16 (&acc)[DP / 32], float f, char *region, OutT *out, int64_t dense, int D, int lane)
{
    constexpr int FIT = BYTES / 32 / (int)sizeof(OutT), W = FIT < DP ? FIT : DP;       // columns per pass
    static_assert(W % 32 == 0 && DP % W == 0, "whole accumulator tiles");
    constexpr int CPR = Tile<OutT, W>::CPR, ROW = Tile<OutT, W>::ROW, EPC = Tile<OutT, W>::EPC;
    const int half = lane >> 5, row = lane & 31;
    const int lo = (int)(uint32_t)(dense & 0xffffffff), hi = (int)(dense >> 32);
#pragma unroll
    for (int c0 = 0; c0 < DP; c0 += W) {
#pragma unroll
        for (int dt = 0; dt < W / 32; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = dt * 32 + 8 * g + 4 * half;
                char *p = region + row * ROW + ((d / EPC) ^ swizzle<CPR>(row)) * 16 + (d % EPC) * (int)sizeof(OutT);
                const f32x16 &v = acc[c0 / 32 + dt];
                float x[4] = {v[4 * g] * f, v[4 * g + 1] * f, v[4 * g + 2] * f, v[4 * g + 3] * f};
                if (LOW) rounded_off(x);
                store4<OutT>(reinterpret_cast<OutT *>(p), x[0], x[1], x[2], x[3]);
            }
        MSDA_WAVE_LDS_SYNC();
        constexpr int ITERATIONS = CPR / 2, BATCH = ITERATIONS < 4 ? ITERATIONS : 4;
#pragma unroll
        for (int it0 = 0; it0 < ITERATIONS; it0 += BATCH) {
            uint4 v[BATCH];
            int64_t at[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int pos = (it0 + j) * 64 + lane, r = pos / CPR, chunk = pos % CPR;
                v[j] = *reinterpret_cast<const uint4 *>(region + r * ROW + (chunk ^ swizzle<CPR>(r)) * 16);
                at[j] = ((int64_t)__shfl(hi, r, 64) << 32) | (uint32_t)__shfl(lo, r, 64);
            }
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int d = c0 + (((it0 + j) * 64 + lane) % CPR) * EPC;
                if (at[j] >= 0 && d < D) *reinterpret_cast<uint4 *>(out + at[j] + d) = v[j];
            }
        }
        MSDA_WAVE_LDS_SYNC();
    }
}

// A float32 accumulator takes at most 2048 streamed rows in sequence, because its rounding error grows with their number.  A split with
// more is cut into stretches, a launch each (2048 rows of a full card are long enough for one): all but the last leave their float32 sums,
// not scaled, where the result or the split's partial result goes, and a launch adds what the one before left.  Memory for the
// stretches themselves would grow with the product of the lengths; adding up inside the loop cost the registers of the heads of 256 (5000
// rows over 5000 keys, 16 heads: 23 -> 36 ms).
constexpr int kStretch = 2048;
struct Stretch { int index, count; };

// tiles [t0, t1) of this stretch of a split's
template <typename T, int ROWS> __device__ __forceinline__ void take_stretch(const Stretch &s, int &t0, int &t1)
{
    if (sizeof(T) == 2) return;
    t0 = min(t0 + s.index * (kStretch / ROWS), t1);
    t1 = min(t0 + kStretch / ROWS, t1);
}

// acc += f times this lane's row (lane & 31) in memory
template <int N> __device__ __forceinline__ void add_row(f32x16 (&acc)[N], const float *row, float f, int D, int half)
{
#pragma unroll
    for (int dt = 0; dt < N; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = dt * 32 + 8 * g + 4 * half;
            if (d < D) {
                const float4 v = *reinterpret_cast<const float4 *>(row + d);
                acc[dt][4 * g] = fmaf(v.x, f, acc[dt][4 * g]);
                acc[dt][4 * g + 1] = fmaf(v.y, f, acc[dt][4 * g + 1]);
                acc[dt][4 * g + 2] = fmaf(v.z, f, acc[dt][4 * g + 2]);
                acc[dt][4 * g + 3] = fmaf(v.w, f, acc[dt][4 * g + 3]);
            }
        }
}

// ---- host: how a call is cut --------------------------------------------------------------------------------------------------
struct Plan { int waves, tiles, splits; };

// `resident` rows of each of `groups` (batch, key head) pairs are held 32 per wave, one, two or four waves a workgroup.  Where that does
// not fill the card the streamed tiles are cut into splits: as many as all fit on the 256 compute units at once, by LDS and by the
// waves a SIMD holds, with at least `least` tiles each.  Measured (bf16): twice as many cost the partial results' traffic -- 64 rows of
// heads of 256 over 22 223 keys 147 us with one round, 163 with two, 193 with four; four shared heads of 128 129 / 134 / 145 us.
inline Plan plan_for(int64_t resident, int64_t streamed_tiles, int64_t groups, int lds, int waves_per_simd, int least)
{
    Plan p;
    int64_t most = streamed_tiles / least > 1 ? streamed_tiles / least : 1;
    p.waves = resident <= 32 ? 1 : resident <= 64 ? 2 : 4;
    p.tiles = (int)((resident + 32 * p.waves - 1) / (32 * p.waves));
    const int by_lds = 160 * 1024 / lds, by_simd = waves_per_simd * 4 / p.waves, fit = by_lds < by_simd ? by_lds : by_simd;
    const int64_t have = p.tiles * groups;
    // (half of the compute units have work already: joining pays from 16 tiles a split on -- 2331 rows of heads of 64 over 1091 keys
    // 24.6 us with one split, 30.5 with three)
    if (have >= 128 && least == 4) most = streamed_tiles / 16 > 1 ? streamed_tiles / 16 : 1;
    const int64_t split = have ? 256 * (int64_t)fit / have : 1;
    p.splits = (int)(split < 1 ? 1 : split > most ? most : split);
    return p;
}

inline int padded_size(const cross_attention_args &a) { return a.D <= 32 ? 32 : a.D <= 64 ? 64 : a.D <= 128 ? 128 : 256; }
inline int row_bytes(const cross_attention_args &a) { return padded_size(a) * (a.dtype == MSDA_BF16 ? 2 : 4); }
// streamed rows per tile: the two buffers of both operands stay within 64 KB where two workgroups share a compute unit
inline constexpr int rows_per_tile(int row_bytes) { return row_bytes >= 512 ? 32 : 64; }
inline int tile_lds(const cross_attention_args &a) { return rows_per_tile(row_bytes(a)) * (4 * row_bytes(a) + 16); }
// float32 tiles hold eight times the matrix instructions: worth a split of their own
inline int least_tiles(const cross_attention_args &a) { return a.dtype == MSDA_BF16 ? 4 : 1; }

// bf16 backward: the products with P and dS also take what the rounding of the two left out (rest_operand).  Without it the gradients'
// errors are 1.42 times those of rounded exact gradients, at every size (300 rows over 300 keys to 2048 over 4096: 1.41 to 1.48; with it
// 1.00 to 1.04): the two roundings weigh as much as the result's own.  It costs matrix instructions only, which calls of few probabilities do
// not wait for -- step without / with: 300 rows over 300 keys, 8 heads of 64, batch 16 73 / 73 us; 777 over 1091, 8 heads of 128 86 / 91;
// 1500 over 1500, 8 heads of 64 88 / 85 -- and large ones do: 512 over 512, 16 heads of 128, batch 64 881 / 1077; 2048 over 4096, 16 heads of
// 128, batch 4 1228 / 1617.  So the rule is the call's whole number of probabilities, batch and heads included: a sequence can get the
// one or the other with its batch, as it gets other splits.  Not with a dropout mask: dropping with probability 0.1 gives every term of
// the sums a relative deviation of sqrt(0.1 / 0.9) = 0.33, 170 times a rounding's 2^-9.
inline bool few_probabilities(const cross_attention_args &a)
{
    return a.dtype == MSDA_BF16 && !a.keep && (double)a.B * a.heads * a.Lq * a.Lk <= 1 << 24;
}

// stretches (add_row) of a split of `tiles` tiles
inline int stretches_of(const cross_attention_args &a, int64_t tiles, const Plan &p)
{
    const int64_t per = (tiles + p.splits - 1) / p.splits, most = kStretch / rows_per_tile(row_bytes(a));
    return a.dtype == MSDA_BF16 || per <= most ? 1 : (int)((per + most - 1) / most);
}

}  // namespace xattn
