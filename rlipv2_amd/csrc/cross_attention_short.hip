// cross_attention_short.hip -- backward pass where one side of the attention is short: at most 64 keys (every pixel reads the label
// texts) or at most 64 query rows (the label texts read every pixel).  bf16, heads of 65 to 256 elements.
//
// Such a call is bound by the long side's memory traffic.  The two passes of cross_attention_backward.hip read the long side twice;
// here one pass does all five products.  A workgroup keeps the short side in REGISTERS, streams the long side through LDS in tiles
// of 32 rows and keeps the short side's gradient as accumulators; its long gradients leave tile by tile.
//
//   X1, X2 = K, V (few keys) or Q, dO (few rows)        the short side, 64 rows
//   Y1, Y2 = Q, dO           or K, V                    a tile of the long side, 32 rows
//   phase 1   S = X1 Y1^T, dP = X2 Y2^T on 16x16x32 tiles: wave = (16 or 32 short rows, 16 long rows); P and dS go to LDS [long][short]
//   phase 2   wave = 32 of the head elements:  long gradient 1 = dS X1,  few rows also long gradient 2 = P X2;
//             short sum 1 += dS Y1,  few keys also short sum 2 += P Y2
//
// Few keys: a row's delta = sum_j P dP is complete in one tile, so it is computed here in float32 (not from the rounded result).
// Few rows: delta comes from the result and its rounding residual, once per workgroup.  The long gradients of tile t are stored
// during tile t + 1, beside the copy of tile t + 1's successor.  Heads of 256: one workgroup of eight waves per compute unit (LDS),
// the long side is cut among them; partial sums of the short gradients are float32, joined by the reduce kernel in the order of the splits.
//
// Measured (heads of 256, 8 heads, batch 4; averages of 20 calls in a kernel trace): 22 223 rows over 64 keys 260 us (1.09 GB: 4.2 TB/s; the two
// passes 541 + 378 us), 64 rows over 22 223 keys 310 us (1.32 GB: 4.3 TB/s; the two passes 187 + 470 us): HBM.  With four waves and twice the registers per wave 497 and 317 us.
#include "cross_attention_device.h"

namespace xattn {

typedef __attribute__((ext_vector_type(4))) float f32x4;

// operand A = the transposed tile with the rows in their natural order: lane -> head element 32 dt + (lane & 31), contraction over
// rows 16 u + 8 (lane >> 5) + e
template <int DP> __device__ __forceinline__ void read_columns_in_order(const char *tile, int u, int dt, int lane, Frag<bf16_t> &f)
{
    constexpr int CPR = Tile<bf16_t, DP>::CPR, ROW = Tile<bf16_t, DP>::ROW;
    const int chunk = dt * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = 16 * u + 8 * (lane >> 5) + 4 * j + ((lane & 15) >> 2);
        f.half[j] = read_tr(tile + row * ROW + ((chunk ^ swizzle<CPR>(row)) * 16) + (lane & 1) * 8);
    }
}

template <int DP, bool FEW_KEYS, bool KEEP, bool FINE>
__global__ __launch_bounds__(2 * DP, 2) void short_kernel(cross_attention_args a, int splits, float c)
{
    typedef bf16_t T;
    constexpr int WAVES = DP / 32, THREADS = 64 * WAVES, GROUPS = WAVES / 2, NI = 4 / GROUPS;       // phase 1: 16 NI short rows per wave
    constexpr int ROW = Tile<T, DP>::ROW, CPR = Tile<T, DP>::CPR, TILE = 32 * ROW, BUF = 2 * TILE, KS = DP / 32;
    constexpr int XROW = 128, XBUF = 32 * XROW, OUTS = FEW_KEYS ? 1 : 2, REGION = 32 * 32 * (int)sizeof(T);
    MSDA_DYNAMIC_LDS(char, lds);
    // P and dS [32 long][64 short], what their rounding took (FINE); long gradients
    char *pbuf = lds + 2 * BUF, *dsbuf = pbuf + XBUF, *prest = dsbuf + (FINE ? XBUF : 0), *dsrest = prest + (FINE ? XBUF : 0), *regions = dsrest + XBUF;
    float *part = reinterpret_cast<float *>(regions + WAVES * OUTS * REGION);       // few keys: delta [GROUPS][32]; few rows: -L / c, -delta [2][64]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int task = task_of(blockIdx.x, gridDim.x), sp = task % splits, bh = task / splits;
    const int b = bh / a.kv_heads, hk = bh - b * a.kv_heads, G = a.heads / a.kv_heads;
    const int64_t row0 = ((int64_t)b * a.heads + hk * G) * a.Lq;                     // (stats and keep: row r = g Lq + q of the key head)
    const Rows rows = {a.Lq, G, G * a.Lq};
    KeyMask mask;
    mask.init(a, b);
    const T *kbase = static_cast<const T *>(a.key) + (int64_t)b * a.key_stride[0] + (int64_t)hk * a.key_stride[2];
    const T *vbase = static_cast<const T *>(a.value) + (int64_t)b * a.value_stride[0] + (int64_t)hk * a.value_stride[2];
    const T *qbase = static_cast<const T *>(a.query) + (int64_t)b * a.query_stride[0];
    const T *gbase = static_cast<const T *>(a.grad_out) + (int64_t)b * a.grad_out_stride[0];
    const unsigned long long keys = __builtin_amdgcn_ballot_w64(mask.load(lane) == 0);          // (few keys)

    // ---- the short side: through LDS into registers ----
    for (int pos = tid; pos < 64 * CPR; pos += THREADS) {
        const int r = pos / CPR, chunk = pos % CPR;
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (chunk * 8 < a.D) {
            if (FEW_KEYS) {
                if ((keys >> r) & 1) {
                    x = *reinterpret_cast<const uint4 *>(kbase + r * a.key_stride[1] + chunk * 8);
                    y = *reinterpret_cast<const uint4 *>(vbase + r * a.value_stride[1] + chunk * 8);
                }
            } else if (r < rows.count) {
                int g, q;
                rows.split(r, g, q);
                x = *reinterpret_cast<const uint4 *>(qbase + q * a.query_stride[1] + (hk * G + g) * a.query_stride[2] + chunk * 8);
                y = *reinterpret_cast<const uint4 *>(gbase + q * a.grad_out_stride[1] + (hk * G + g) * a.grad_out_stride[2] + chunk * 8);
            }
        }
        const int at = r * ROW + (chunk ^ swizzle<CPR>(r)) * 16;
        *reinterpret_cast<uint4 *>(lds + at) = x;
        *reinterpret_cast<uint4 *>(lds + 64 * ROW + at) = y;
    }
    __syncthreads();
    const int group = wave % GROUPS, rh = wave / GROUPS, short0 = group * 16 * NI;
    Frag<T> x1[NI][KS], x2[NI][KS], x1t[4], x2t[4];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int r = short0 + i * 16 + (lane & 15), at = r * ROW + ((4 * s + (lane >> 4)) ^ swizzle<CPR>(r)) * 16;
            x1[i][s].u = *reinterpret_cast<const uint4 *>(lds + at);
            x2[i][s].u = *reinterpret_cast<const uint4 *>(lds + 64 * ROW + at);
        }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        read_columns_in_order<DP>(lds, u, wave, lane, x1t[u]);
        if (!FEW_KEYS) read_columns_in_order<DP>(lds + 64 * ROW, u, wave, lane, x2t[u]);
    }
    f32x4 s0[NI], dp0[NI];                       // what the accumulators of phase 1 start from
    if (FEW_KEYS) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s0[i][e] = (keys >> (short0 + i * 16 + 4 * (lane >> 4) + e)) & 1 ? 0.f : -kInf;
                dp0[i][e] = 0.f;
            }
    } else {
        // four threads per row: delta = rowsum(dO O)
        const int r = tid >> 2;
        float d = 0.f;
        int g = 0, q = 0;
        if (r < rows.count) {
            rows.split(r, g, q);
            const int64_t dense = (((int64_t)b * a.Lq + q) * a.heads + hk * G + g) * a.D;
            for (int chunk = tid & 3; chunk * 8 < a.D; chunk += 4) {
                Frag<T> o, w;
                w.u = *reinterpret_cast<const uint4 *>(gbase + q * a.grad_out_stride[1] + (hk * G + g) * a.grad_out_stride[2] + chunk * 8);
                o.u = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.out) + dense + chunk * 8);
                d += dot8(o, w);
                if (a.out_low) {
                    o.u = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.out_low) + dense + chunk * 8);
                    d += dot8(o, w);
                }
            }
        }
        d += __shfl_xor(d, 1, 64);
        d += __shfl_xor(d, 2, 64);
        if ((tid & 3) == 0 && r < 64) {
            part[r] = r < rows.count ? static_cast<const float *>(a.stats)[row0 + r] * (-1.f / c) : -kInf;
            part[64 + r] = -d;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = short0 + i * 16 + 4 * (lane >> 4) + e;
                s0[i][e] = part[at];
                dp0[i][e] = part[64 + at];
            }
    }
    __syncthreads();                           // the short side's LDS becomes the tile buffers

    // ---- the long side ----
    const int head_tiles = (a.Lq + 31) / 32, tiles = FEW_KEYS ? G * head_tiles : (a.Lk + 31) / 32, per = (tiles + splits - 1) / splits;
    const int t0 = min(sp * per, tiles), t1 = min(tiles, t0 + per);
    Stager<T, DP, 32, THREADS> stage1, stage2;
    stage1.init(FEW_KEYS ? a.query_stride[1] : a.key_stride[1], tid, a.D);
    stage2.init(FEW_KEYS ? a.grad_out_stride[1] : a.value_stride[1], tid, a.D);
    const auto place = [&](int t, int &g, int &first) {
        g = FEW_KEYS ? t / head_tiles : 0;
        first = (t - g * head_tiles * (FEW_KEYS ? 1 : 0)) * 32;
    };
    const auto fill = [&](int t, uint32_t word) {
        char *tile = lds + (t & 1) * BUF;
        int g, first;
        place(t, g, first);
        const int head = hk * G + g;
        stage1.copy(tile, FEW_KEYS ? qbase + (int64_t)first * a.query_stride[1] + (int64_t)head * a.query_stride[2]
                                   : kbase + (int64_t)first * a.key_stride[1], word);
        stage2.copy(tile + TILE, FEW_KEYS ? gbase + (int64_t)first * a.grad_out_stride[1] + (int64_t)head * a.grad_out_stride[2]
                                          : vbase + (int64_t)first * a.value_stride[1], word);
    };
    // which rows of tile t count; few rows: from the mask bytes that were loaded a tile ahead
    int byte = 1;
    const auto word_of = [&](int t) -> uint32_t {
        if (!FEW_KEYS) return (uint32_t)__builtin_amdgcn_ballot_w64(byte == 0);
        if (!keys) return 0;                   // (no key at all: no gradient, whatever grad_out holds)
        int g, first;
        place(t, g, first);
        const int n = a.Lq - first;
        return n >= 32 ? ~0u : (1u << n) - 1;
    };
    const auto load_log = [&](int t) {         // few keys: the statistics of this lane's long row
        int g, first;
        place(t, g, first);
        const int q = first + rh * 16 + (lane & 15);
        return q < a.Lq ? static_cast<const float *>(a.stats)[row0 + (int64_t)g * a.Lq + q] : kInf;
    };
    char *region = regions + wave * OUTS * REGION;
    // a long gradient's columns of this wave, from the wave's region to global memory (32 rows span less than 4 GB: short_side)
    constexpr int WCPR = 4;
    const int leave_row = lane / WCPR, d0 = __builtin_amdgcn_readfirstlane(wave) * 32;
    const uint32_t stride = (uint32_t)(FEW_KEYS ? a.heads : a.kv_heads) * a.D;
    const uint32_t leave_at = leave_row * stride + (lane % WCPR) * 8;
    const bool leave_in = d0 + (lane % WCPR) * 8 < a.D;
    const auto leave = [&](int t) {
        int g, first;
        place(t, g, first);
        const int n = (FEW_KEYS ? a.Lq : a.Lk) - first;
        const int64_t at = FEW_KEYS ? (((int64_t)b * a.Lq + first) * a.heads + hk * G + g) * a.D : (((int64_t)b * a.Lk + first) * a.kv_heads + hk) * a.D;
#pragma unroll
        for (int o = 0; o < OUTS; ++o) {
            T *out = static_cast<T *>(FEW_KEYS ? a.grad_query : o ? a.grad_value : a.grad_key) + at + d0;
#pragma unroll
            for (int it = 0; it < WCPR / 2; ++it, out += (64 / WCPR) * stride) {
                const int r = it * (64 / WCPR) + leave_row, chunk = lane % WCPR;
                const uint4 v = *reinterpret_cast<const uint4 *>(region + o * REGION + r * (WCPR * 16) + (chunk ^ swizzle<WCPR>(r)) * 16);
                if (r < n && leave_in) *reinterpret_cast<uint4 *>(out + leave_at) = v;
            }
        }
    };

    // operand A of the short sums: this wave's 32 head elements of a tile, transposed (the wave's part of the address is not a constant)
    const int column_row = 4 * half + ((lane & 15) >> 2);
    const int column_at = column_row * ROW + (((wave * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ swizzle<CPR>(column_row)) * 16) + (lane & 1) * 8;
    const auto read_wave_columns = [&](const char *tile, int u, Frag<T> &f) {
        f.half[0] = read_tr(tile + column_at + 16 * u * ROW);
        f.half[1] = read_tr(tile + column_at + (16 * u + 8) * ROW);
    };
    f32x16 sum1[2], sum2[2];
    clear(sum1);
    clear(sum2);
    uint32_t word = 0, next = 0;
    float log_sum = kInf, next_log = kInf;
    if (t0 < t1) {
        if (!FEW_KEYS) byte = mask.load(t0 * 32 + (lane & 31));
        next = word_of(t0);
        if (next) fill(t0, next);
        if (FEW_KEYS) next_log = load_log(t0);
        else byte = mask.load((t0 + 1) * 32 + (lane & 31));
    }
    for (int t = t0; t < t1; ++t) {
        copies_done();
        __syncthreads();                       // tile t has arrived, everybody is done with the other buffer
        word = next;
        log_sum = next_log;
        if (t + 1 < t1) {
            next = word_of(t + 1);
            if (next) fill(t + 1, next);
            if (FEW_KEYS) next_log = load_log(t + 1);
            else byte = mask.load((t + 2) * 32 + (lane & 31));
        }
        if (t > t0) leave(t - 1);
        const char *y1 = lds + (t & 1) * BUF, *y2 = y1 + TILE;
        f32x16 long1[1], long2[1];
        clear(long1);
        clear(long2);
        if (word) {                            // (a tile whose keys all do not count: zeros)
            const int row = rh * 16 + (lane & 15);
            f32x4 s[NI], dp[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[i][e] = s0[i][e];
                    dp[i][e] = KEEP ? 0.f : dp0[i][e];
                }
            const int low = (lane >> 4), x = swizzle<CPR>(row);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                Frag<T> f1, f2;
                const int at = row * ROW + ((4 * (k & 1) + low) ^ x) * 16 + (k >> 1) * 128;
                f1.u = *reinterpret_cast<const uint4 *>(y1 + at);
                f2.u = *reinterpret_cast<const uint4 *>(y2 + at);
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x1[i][k].v, f1.v, s[i], 0, 0, 0);
                    dp[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x2[i][k].v, f2.v, dp[i], 0, 0, 0);
                }
            }
            // (the reads run ahead of the matrix instructions)
            if (!KEEP) {
                XATTN_SCHED_GROUP(0x100, 6);
#pragma unroll
                for (int k = 3; k < KS; ++k) {
                    XATTN_SCHED_GROUP(0x8, 2 * NI);
                    XATTN_SCHED_GROUP(0x100, 2);
                }
                XATTN_SCHED_GROUP(0x8, 6 * NI);
            }
            const bool counts = FEW_KEYS || ((word >> row) & 1);
            float p[NI][4], pd[NI][4], d = 0.f;  // probabilities, the dropped ones, this lane's part of delta
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[i][e] = FEW_KEYS ? exp2_fast(fmaf(s[i][e], c, -log_sum)) : counts ? exp2_fast(s[i][e] * c) : 0.f;
                    float factor = 1.f;
                    if (KEEP) {
                        const int shrt = short0 + i * 16 + 4 * (lane >> 4) + e;
                        int g, first;
                        place(t, g, first);
                        const int64_t r = FEW_KEYS ? (int64_t)g * a.Lq + min(first + row, a.Lq - 1) : min(shrt, rows.count - 1);
                        const int key = FEW_KEYS ? min(shrt, a.Lk - 1) : min(first + row, a.Lk - 1);
                        factor = static_cast<const uint8_t *>(a.keep)[(row0 + r) * a.Lk + key] ? a.keep_scale : 0.f;
                    }
                    pd[i][e] = p[i][e] * factor;
                    if (KEEP) dp[i][e] *= factor;
                    if (FEW_KEYS) d = fmaf(p[i][e], dp[i][e], d);
                }
            float delta = 0.f;
            if (FEW_KEYS) {
                d += __shfl_xor(d, 16, 64);
                d += __shfl_xor(d, 32, 64);
                if (lane < 16) part[group * 32 + row] = d;
                __syncthreads();
                delta = part[row] + part[32 + row];
                if (GROUPS == 4) delta += part[64 + row] + part[96 + row];
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                float ds[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) ds[e] = p[i][e] * (FEW_KEYS ? dp[i][e] - delta : KEEP ? dp[i][e] + dp0[i][e] : dp[i][e]);
                const int at = row * XROW + (((short0 >> 3) + i * 2 + (lane >> 5)) ^ swizzle<8>(row)) * 16 + ((lane >> 4) & 1) * 8;
                store4<T>(reinterpret_cast<T *>(dsbuf + at), ds[0], ds[1], ds[2], ds[3]);
                store4<T>(reinterpret_cast<T *>(pbuf + at), pd[i][0], pd[i][1], pd[i][2], pd[i][3]);
                if constexpr (FINE) {
                    rounded_off(ds);
                    rounded_off(pd[i]);
                    store4<T>(reinterpret_cast<T *>(dsrest + at), ds[0], ds[1], ds[2], ds[3]);
                    store4<T>(reinterpret_cast<T *>(prest + at), pd[i][0], pd[i][1], pd[i][2], pd[i][3]);
                }
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                Frag<T> f, h;
                read_rows<64>(dsbuf, lane & 31, u, half, f);
                if (!FEW_KEYS) read_rows<64>(pbuf, lane & 31, u, half, h);
                mma(x1t[u], f, long1[0]);
                if (!FEW_KEYS) mma(x2t[u], h, long2[0]);
                if (FINE) {
                    read_rows<64>(dsrest, lane & 31, u, half, f);
                    mma(x1t[u], f, long1[0]);
                    if (!FEW_KEYS) {
                        read_rows<64>(prest, lane & 31, u, half, h);
                        mma(x2t[u], h, long2[0]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                Frag<T> ds[2], pp[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    read_columns<64>(dsbuf, 16 * u, i, lane, ds[i]);
                    if (FEW_KEYS) read_columns<64>(pbuf, 16 * u, i, lane, pp[i]);
                }
                Frag<T> f, h;
                read_wave_columns(y1, u, f);
                if (FEW_KEYS) read_wave_columns(y2, u, h);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    mma(f, ds[i], sum1[i]);
                    if (FEW_KEYS) mma(h, pp[i], sum2[i]);
                    if (FINE) {
                        read_columns<64>(dsrest, 16 * u, i, lane, ds[i]);
                        mma(f, ds[i], sum1[i]);
                        if (FEW_KEYS) {
                            read_columns<64>(prest, 16 * u, i, lane, pp[i]);
                            mma(h, pp[i], sum2[i]);
                        }
                    }
                }
            }
            if (!KEEP && !FINE) {
                // reads of the long gradients; matrix instructions with the reads of the sums between them; the last ones
                constexpr int R1 = FEW_KEYS ? 4 : 8, R2 = FEW_KEYS ? 24 : 12, M = 12;
                constexpr int PER = FEW_KEYS ? 3 : 2, STEPS = (R2 + PER - 1) / PER;
                static_assert(STEPS <= M, "reads fit between");
                XATTN_SCHED_GROUP(0x100, R1);
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    XATTN_SCHED_GROUP(0x8, 1);
                    XATTN_SCHED_GROUP(0x100, PER);
                }
                XATTN_SCHED_GROUP(0x8, M - STEPS);
            }
        }
        if (mask.one()) clear(long1);
        if (!FEW_KEYS && word != ~0u) {        // (keys that do not count: 0 times an infinite or NaN grad_out is NaN)
            zero_unless((word >> (lane & 31)) & 1, long1);
            zero_unless((word >> (lane & 31)) & 1, long2);
        }
        // (few keys: grad_query; few rows: grad_key, grad_value)
        MSDA_WAVE_LDS_SYNC();
#pragma unroll
        for (int o = 0; o < OUTS; ++o)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int r = lane & 31;
                const float f = o ? 1.f : a.scale;
                const f32x16 &v = o ? long2[0] : long1[0];
                char *at = region + o * REGION + r * (WCPR * 16) + (g ^ swizzle<WCPR>(r)) * 16 + half * 8;
                store4<T>(reinterpret_cast<T *>(at), v[4 * g] * f, v[4 * g + 1] * f, v[4 * g + 2] * f, v[4 * g + 3] * f);
            }
        MSDA_WAVE_LDS_SYNC();
    }
    if (t0 < t1) leave(t1 - 1);
    if (FEW_KEYS && !a.grad_key) return;
    __syncthreads();                           // everybody is done with the tiles: their memory carries the short gradients out

    constexpr int OUT_REGION = 2 * BUF / WAVES;
    char *mine = lds + wave * OUT_REGION;
    const int64_t all = FEW_KEYS ? (int64_t)a.B * a.Lk * a.kv_heads * a.D : (int64_t)a.B * a.Lq * a.heads * a.D;
    float *partial = static_cast<float *>(a.workspace) + (int64_t)sp * (FEW_KEYS ? 2 : 1) * all + d0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = i * 32 + (lane & 31);
        int64_t dense = -1;
        if (FEW_KEYS) {
            if (r < a.Lk) dense = (((int64_t)b * a.Lk + r) * a.kv_heads + hk) * a.D;
        } else if (r < rows.count) {
            int g, q;
            rows.split(r, g, q);
            dense = (((int64_t)b * a.Lq + q) * a.heads + hk * G + g) * a.D;
        }
        f32x16 v[1] = {sum1[i]};
        zero_unless(!mask.one() && (!FEW_KEYS || ((keys >> r) & 1)), v);
        T *first = static_cast<T *>(FEW_KEYS ? a.grad_key : a.grad_query) + d0;
        if (splits == 1) put_rows<T, 32, OUT_REGION>(v, a.scale, mine, first, dense, a.D - d0, lane);
        else put_rows<float, 32, OUT_REGION>(v, 1.f, mine, partial, dense, a.D - d0, lane);
        if constexpr (FEW_KEYS) {
            v[0] = sum2[i];
            zero_unless((keys >> r) & 1, v);
            if (splits == 1) put_rows<T, 32, OUT_REGION>(v, 1.f, mine, static_cast<T *>(a.grad_value) + d0, dense, a.D - d0, lane);
            else put_rows<float, 32, OUT_REGION>(v, 1.f, mine, partial + all, dense, a.D - d0, lane);
        }
    }
}

// Which of the two kernels a call takes: 1 few keys (also for the query's gradient alone: the forward call, which does not know what will
// be asked for, leaves out out_low), 2 few rows, 0 neither.
int short_side(const cross_attention_args &a)
{
    if (a.dtype != MSDA_BF16 || a.D <= 64 || a.Lq == 0 || a.Lk == 0 || a.heads > (1 << 16)) return 0;
    return a.Lk <= 64 ? 1 : a.grad_key && (int64_t)(a.heads / a.kv_heads) * a.Lq <= 64 ? 2 : 0;
}

int short_splits(const cross_attention_args &a)
{
    const int64_t tiles = a.Lk <= 64 ? (int64_t)(a.heads / a.kv_heads) * ((a.Lq + 31) / 32) : (a.Lk + 31) / 32;
    const int64_t groups = (int64_t)a.B * a.kv_heads, most = tiles / 4 > 1 ? tiles / 4 : 1, want = a.D > 128 ? 256 : 512;
    const int64_t s = (want + groups - 1) / groups;
    return (int)(s > most ? most : s);
}

template <int DP, bool FEW_KEYS, bool KEEP, bool FINE> void launch_short_kernel(const cross_attention_args &a, int splits, hipStream_t stream)
{
    constexpr int LDS = 4 * 32 * DP * 2 + (FINE ? 4 : 2) * 4096 + DP / 32 * (FEW_KEYS ? 1 : 2) * 2048 + 512;
    const auto kernel = short_kernel<DP, FEW_KEYS, KEEP, FINE>;
    RLIPV2_ONCE_PER_DEVICE((void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
    hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)splits * a.B * a.kv_heads)), dim3(2 * DP), LDS, stream, a, splits,
                       a.scale * 1.4426950408889634f);
}

template <int DP, bool FEW_KEYS> void short_by_mask(const cross_attention_args &a, int splits, hipStream_t stream)
{
    if (few_probabilities(a)) launch_short_kernel<DP, FEW_KEYS, false, true>(a, splits, stream);
    else if (a.keep) launch_short_kernel<DP, FEW_KEYS, true, false>(a, splits, stream);
    else launch_short_kernel<DP, FEW_KEYS, false, false>(a, splits, stream);
}

template <bool FEW_KEYS> void short_by_size(const cross_attention_args &a, int splits, hipStream_t stream)
{
    a.D <= 128 ? short_by_mask<128, FEW_KEYS>(a, splits, stream) : short_by_mask<256, FEW_KEYS>(a, splits, stream);
}

void launch_short(const cross_attention_args &a, int splits, hipStream_t stream)
{
    if (short_side(a) == 1) short_by_size<true>(a, splits, stream);
    else short_by_size<false>(a, splits, stream);
}

}  // namespace xattn
