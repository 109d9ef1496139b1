// cross_attention_backward.hip -- gradients of softmax(scale q k^T) v (include/rlipv2_attention.h; the layout of the products:
// cross_attention_device.h).  The probabilities are recomputed from the logits and the forward pass's logarithms of the row sums:
//
//   P = 2^(c S - L),  dP = keep keep_scale (dO V^T),  dS = P (dP - delta),  delta = rowsum(dO O)
//   dQ = scale dS K      query_kernel: 32 query rows per wave, the keys are streamed (and delta is computed and stored)
//   dV = P~^T dO, dK = scale dS^T Q      key_kernel: 32 keys per wave, the rows of ALL heads that share the key head are streamed
//
// Two passes instead of one with atomics: nothing is added up in an order that can change.  Where one side is short, the streamed
// side is cut into splits that write float32 partial sums; reduce_kernel adds them in the order of the splits.  P and dS are
// rounded to the operands' type for the products (relative 2^-9 in bf16), everything else is float32.  delta is taken from out and what
// its rounding took (out_low): with the rounded out alone the errors of dQ and dK grow from 2.4e-3 to 2.7e-3 over 64 keys.
//
// What bounds it, measured (bf16; averages of 20 calls in a kernel trace, profiles/operators_kernel_stats.csv, and the last of them, the
// clock settled): 2048 rows over 4096 keys, 16 heads of 128, batch 4: query_kernel 425 us (406: 1015 TFLOP/s), key_kernel 606 us (561: 980
// TFLOP/s): matrix instructions and the vector work between them, two waves per SIMD; the key pass holds 192 registers of operands
// and sums.  Read ahead of the matrix instructions: key pass 1107 -> 920 us, row statistics as the accumulators' start values and no
// dropout code: -> 610.  777 rows of 12 heads of 64 over 1091 keys, batch 3: 30 + 34 us, short loops between prologue and epilogue.
// float32, the same 2048 rows: 127 TFLOP/s; heads of 256, 5000 rows over 5000 keys: 87, with the logits a second time for the keys'
// gradient (registers).
#include "cross_attention_device.h"

namespace {

using namespace msda;
using namespace xattn;

// KEEP: with a dropout mask
template <typename T, int DP, int NW, int BN, int OCC, bool KEEP, bool FINE>
__global__ __launch_bounds__(64 * NW, OCC) void query_kernel(cross_attention_args a, int row_tiles, int splits, Stretch stretch, float c)
{
    constexpr int THREADS = 64 * NW, NSUB = BN / 32, KB = BN * Tile<T, DP>::ROW, BUF = 2 * KB;
    constexpr bool AHEAD = sizeof(T) == 2 && !KEEP;      // (float32: eight matrix instructions per operand; the schedule takes minutes to compile)
    constexpr int ROW_READS = sizeof(T) == 2 ? 1 : 2, COLUMN_READS = sizeof(T) == 2 ? 2 : 8, MMAS = sizeof(T) == 2 ? 1 : 8;
    MSDA_DYNAMIC_LDS(char, lds);
    float *bias = reinterpret_cast<float *>(lds + 2 * BUF);              // [2 buffers][BN]: 0, or -infinity for keys that do not count
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int task = task_of(blockIdx.x, gridDim.x);
    const int rt = task % row_tiles, sp = (task / row_tiles) % splits, bh = task / (row_tiles * splits);
    const int b = bh / a.kv_heads, hk = bh - b * a.kv_heads, G = a.heads / a.kv_heads;
    const Rows rows = {a.Lq, G, G * a.Lq};
    const int r = (rt * NW + wave) * 32 + (lane & 31);
    const bool ok = r < rows.count;
    int g, q;
    rows.split(ok ? r : 0, g, q);
    const int head = hk * G + g;
    const int64_t stat = ((int64_t)b * a.heads + head) * a.Lq + q, dense = (((int64_t)b * a.Lq + q) * a.heads + head) * a.D;

    // float32 heads of 256: the registers hold the queries and the sums; grad_out comes from the cache once per tile
    constexpr bool AGAIN = DP * sizeof(T) > 512;
    Frag<T> qf[DP / 16], gf[AGAIN ? 1 : DP / 16];
    float delta = 0.f;
    const T *grow = static_cast<const T *>(a.grad_out) + (int64_t)b * a.grad_out_stride[0] + (int64_t)q * a.grad_out_stride[1] +
                    (int64_t)head * a.grad_out_stride[2];
    {
        const T *row = static_cast<const T *>(a.query) + (int64_t)b * a.query_stride[0] + (int64_t)q * a.query_stride[1] +
                       (int64_t)head * a.query_stride[2];
        const T *orow = static_cast<const T *>(a.out) + dense;
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            Frag<T> of;
            load_operand(row, 16 * s + 8 * half, a.D, ok, qf[s]);
            Frag<T> &g_ = gf[AGAIN ? 0 : s];
            load_operand(grow, 16 * s + 8 * half, a.D, ok, g_);
            load_operand(orow, 16 * s + 8 * half, a.D, ok, of);
            delta += dot8(g_, of);
            if (sizeof(T) == 2 && a.out_low) {
                load_operand(static_cast<const T *>(a.out_low) + dense, 16 * s + 8 * half, a.D, ok, of);
                delta += dot8(g_, of);
            }
        }
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            settle(qf[s]);
            if (!AGAIN) settle(gf[s]);
        }
        delta += other_half(delta);
    }
    float log_sum = ok ? static_cast<const float *>(a.stats)[stat] : kInf;
    MSDA_ASM_OPAQUE(log_sum);
    if (ok && sp == 0 && half == 0) static_cast<float *>(a.delta)[stat] = delta;
    const T *kbase = static_cast<const T *>(a.key) + (int64_t)b * a.key_stride[0] + (int64_t)hk * a.key_stride[2];
    const T *vbase = static_cast<const T *>(a.value) + (int64_t)b * a.value_stride[0] + (int64_t)hk * a.value_stride[2];
    const uint8_t *keep = static_cast<const uint8_t *>(a.keep) + stat * a.Lk;

    KeyMask mask;
    mask.init(a, b);
    const int tiles = (mask.length + BN - 1) / BN, per = (tiles + splits - 1) / splits;
    int t0 = min(sp * per, tiles), t1 = min(tiles, t0 + per);
    take_stretch<T, BN>(stretch, t0, t1);
    const int my_key = lane & (BN - 1);
    Stager<T, DP, BN, THREADS> kstage, vstage;
    kstage.init(a.key_stride[1], tid, a.D);
    vstage.init(a.value_stride[1], tid, a.D);
    const auto fill = [&](int t, unsigned long long word_) {
        char *tile = lds + (t & 1) * BUF;
        kstage.copy(tile, kbase + (int64_t)t * BN * a.key_stride[1], word_);
        vstage.copy(tile + KB, vbase + (int64_t)t * BN * a.value_stride[1], word_);
        if (tid < BN) bias[(t & 1) * BN + tid] = (word_ >> tid) & 1 ? 0.f : -kInf;
    };

    f32x16 acc[DP / 32];
    clear(acc);
    unsigned long long word = 0, next = 0;
    int byte = 1;
    constexpr unsigned long long ALL = BN == 64 ? ~0ull : 0xffffffffull;
    if (t0 < t1) {
        next = __builtin_amdgcn_ballot_w64(mask.load(t0 * BN + my_key) == 0) & ALL;
        byte = mask.load((t0 + 1) * BN + my_key);
        if (next) fill(t0, next);
    }
    for (int t = t0; t < t1; ++t) {
        copies_done();
        __syncthreads();                      // tile t has arrived, everybody is done with the other buffer
        word = next;
        if (t + 1 < t1) {
            next = __builtin_amdgcn_ballot_w64(byte == 0) & ALL;
            if (next) fill(t + 1, next);
            byte = mask.load((t + 2) * BN + my_key);
        }
        if (!word) continue;
        const char *kt = lds + (t & 1) * BUF, *vt = kt + KB;
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub) {
            f32x16 s[1], dp[1];
            load_quads(bias + (t & 1) * BN + sub * 32 + 4 * half, s[0]);       // (the mask: see the forward kernel)
            clear(dp);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                Frag<T> f;
                read_rows<DP>(kt, sub * 32 + (lane & 31), k, half, f);
                mma(f, qf[k], s[0]);
                read_rows<DP>(vt, sub * 32 + (lane & 31), k, half, f);
                if (AGAIN) load_operand(grow, 16 * k + 8 * half, a.D, ok, gf[0]);
                mma(f, gf[AGAIN ? 0 : k], dp[0]);
            }
            if (AHEAD) XATTN_SCHED_GROUP(0x100, 4);
            ahead<AHEAD, 2 * DP / 16, ROW_READS, MMAS>();
            Frag<T> df[2], df_rest[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float ds[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = 8 * u + e;
                    float d = dp[0][i];
                    if (KEEP) {
                        const int key = t * BN + sub * 32 + (i & 3) + 8 * (i >> 2) + 4 * half;
                        d *= keep[min(key, a.Lk - 1)] ? a.keep_scale : 0.f;
                    }
                    const float p = exp2_fast(fmaf(s[0][i], c, -log_sum));
                    ds[e] = p * (d - delta);
                }
                to_operand(ds, df[u]);
                if (FINE) rest_operand(ds, df[u], df_rest[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) {
                    Frag<T> f;
                    read_columns<DP>(kt, sub * 32 + 16 * u, dt, lane, f);
                    mma(f, df[u], acc[dt]);
                    if (FINE) mma(f, df_rest[u], acc[dt]);
                }
            ahead<AHEAD, 2 * DP / 32, COLUMN_READS, FINE ? 2 : MMAS>();
        }
    }
    float *part = static_cast<float *>(a.workspace) + (int64_t)sp * a.B * a.Lq * a.heads * a.D;
    if (sizeof(T) == 4 && stretch.index > 0 && ok) add_row(acc, (splits == 1 ? static_cast<const float *>(a.grad_query) : part) + dense, 1.f, a.D, half);
    const float factor = sizeof(T) == 4 && stretch.index + 1 < stretch.count ? 1.f : a.scale;
    zero_unless(!mask.one(), acc);
    __syncthreads();                          // everybody is done with the tiles: their memory carries the results out
    constexpr int REGION = 2 * BUF / NW;
    char *region = lds + wave * REGION;
    if (splits == 1) put_rows<T, DP, REGION>(acc, factor, region, static_cast<T *>(a.grad_query), ok ? dense : -1, a.D, lane);
    else put_rows<float, DP, REGION>(acc, 1.f, region, part, ok ? dense : -1, a.D, lane);
}

// DV / DK: which of the two gradients this launch computes (float32 heads of 256: one at a time, the registers do not hold both)
template <typename T, int DP, int NW, int BM, int OCC, bool DV, bool DK, bool KEEP, bool FINE>
__global__ __launch_bounds__(64 * NW, OCC) void key_kernel(cross_attention_args a, int key_tiles, int splits, Stretch stretch, float c)
{
    constexpr int THREADS = 64 * NW, NSUB = BM / 32, QB = BM * Tile<T, DP>::ROW, BUF = 2 * QB;
    constexpr bool AHEAD = sizeof(T) == 2 && !KEEP;      // (float32: eight matrix instructions per operand; the schedule takes minutes to compile)
    constexpr int ROW_READS = sizeof(T) == 2 ? 1 : 2, COLUMN_READS = sizeof(T) == 2 ? 2 : 8, MMAS = sizeof(T) == 2 ? 1 : 8;
    MSDA_DYNAMIC_LDS(char, lds);
    float *stat_lds = reinterpret_cast<float *>(lds + 2 * BUF);          // [2 buffers][log sums BM | deltas BM]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int task = task_of(blockIdx.x, gridDim.x);
    const int kt_ = task % key_tiles, sp = (task / key_tiles) % splits, bh = task / (key_tiles * splits);
    const int b = bh / a.kv_heads, hk = bh - b * a.kv_heads, G = a.heads / a.kv_heads;
    const int key = (kt_ * NW + wave) * 32 + (lane & 31);
    KeyMask mask;
    mask.init(a, b);
    const bool counts = mask.load(key) == 0;

    Frag<T> kf[DP / 16], vf[DK ? DP / 16 : 1];
    {
        const int64_t at = counts ? key : 0;
        const T *krow = static_cast<const T *>(a.key) + (int64_t)b * a.key_stride[0] + at * a.key_stride[1] + (int64_t)hk * a.key_stride[2];
        const T *vrow = static_cast<const T *>(a.value) + (int64_t)b * a.value_stride[0] + at * a.value_stride[1] + (int64_t)hk * a.value_stride[2];
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            load_operand(krow, 16 * s + 8 * half, a.D, counts, kf[s]);
            if (DK) load_operand(vrow, 16 * s + 8 * half, a.D, counts, vf[s]);
        }
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            settle(kf[s]);
            if (DK) settle(vf[s]);
        }
    }
    // a tile of rows belongs to one query head: tile t is head g = t / head_tiles of those that share the key head
    const int head_tiles = (a.Lq + BM - 1) / BM, tiles = G * head_tiles, per = (tiles + splits - 1) / splits;
    int t0 = min(sp * per, tiles), t1 = __builtin_amdgcn_ballot_w64(counts) || NW > 1 ? min(tiles, t0 + per) : t0;
    take_stretch<T, BM>(stretch, t0, t1);
    Stager<T, DP, BM, THREADS> qstage, gstage;
    qstage.init(a.query_stride[1], tid, a.D);
    gstage.init(a.grad_out_stride[1], tid, a.D);
    const auto fill = [&](int t) {
        char *tile = lds + (t & 1) * BUF;
        const int g = t / head_tiles, q0 = (t - g * head_tiles) * BM, n = a.Lq - q0, head = hk * G + g;
        const unsigned long long word = n >= 64 ? ~0ull : (1ull << n) - 1;
        qstage.copy(tile, static_cast<const T *>(a.query) + (int64_t)b * a.query_stride[0] + (int64_t)q0 * a.query_stride[1] +
                              (int64_t)head * a.query_stride[2], BM == 64 ? word : word & 0xffffffffull);
        gstage.copy(tile + QB, static_cast<const T *>(a.grad_out) + (int64_t)b * a.grad_out_stride[0] +
                                   (int64_t)q0 * a.grad_out_stride[1] + (int64_t)head * a.grad_out_stride[2],
                    BM == 64 ? word : word & 0xffffffffull);
    };
    const int64_t head0 = (int64_t)b * a.heads + hk * G;
    constexpr int NSTAT = (2 * BM + THREADS - 1) / THREADS;
    static_assert(NSTAT <= 2, "one or two row statistics per thread");
    float next_stat[NSTAT];
    constexpr bool FOLD = sizeof(T) == 2;
    const float log_factor = FOLD ? -1.f / c : 1.f;                      // statistics as the loop wants them: -L / c and -delta, or both as they are
    const auto load_stats = [&](int t) {
        const int g = t / head_tiles, q0 = (t - g * head_tiles) * BM;
        const float *logs = static_cast<const float *>(a.stats) + (head0 + g) * a.Lq;
        const float *deltas = static_cast<const float *>(a.delta) + (head0 + g) * a.Lq;
#pragma unroll
        for (int j = 0; j < NSTAT; ++j) {
            const int i = j * THREADS + tid, q = q0 + (i & (BM - 1));
            const float v = q >= a.Lq ? (i < BM ? kInf : 0.f) : (i < BM ? logs[q] : deltas[q]);
            next_stat[j] = i < BM ? v * log_factor : FOLD ? -v : v;
        }
    };
    f32x16 dv[DV ? DP / 32 : 1], dk[DK ? DP / 32 : 1];
    clear(dv);
    clear(dk);
    if (t0 < t1) {
        fill(t0);
        load_stats(t0);
    }
    for (int t = t0; t < t1; ++t) {
        copies_done();                        // (waves without row statistics have nothing else to wait for)
        float *st = stat_lds + (t & 1) * 2 * BM;
#pragma unroll
        for (int j = 0; j < NSTAT; ++j)
            if (j * THREADS + tid < 2 * BM) st[j * THREADS + tid] = next_stat[j];
        __syncthreads();                      // tile t and its statistics are there, everybody is done with the other buffer
        if (t + 1 < t1) {
            fill(t + 1);
            load_stats(t + 1);
        }
        const char *qt = lds + (t & 1) * BUF, *gt = qt + QB;
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub) {
            // bf16: the accumulators start from -L / c and (without dropout) from -delta, which saves the registers for both; the
            // logits' rounding steps grow to those of |L / c|, far below the operands' own.  float32 subtracts at the end.
            f32x16 s[1], dp[1], row_log[1], row_delta[1];
            const float *stp = st + sub * 32 + 4 * half;
            if (FOLD) {
                load_quads(stp, s[0]);
                if (!KEEP) load_quads(stp + BM, dp[0]);
                else clear(dp);
            } else {
                load_quads(stp, row_log[0]);
                load_quads(stp + BM, row_delta[0]);
                clear(s);
                clear(dp);
            }
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                Frag<T> f;
                read_rows<DP>(qt, sub * 32 + (lane & 31), k, half, f);
                mma(f, kf[k], s[0]);
                if (DK) {
                    read_rows<DP>(gt, sub * 32 + (lane & 31), k, half, f);
                    mma(f, vf[k], dp[0]);
                }
            }
            if (AHEAD) XATTN_SCHED_GROUP(0x100, DK ? 8 : 4);
            ahead<AHEAD, (DK ? 2 : 1) * DP / 16, ROW_READS, MMAS>();
            Frag<T> pf[2], df[2], pf_rest[2], df_rest[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float p[8], ds[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int i = 8 * u + e;
                    float factor = 1.f;
                    if (KEEP) {
                        const int at = sub * 32 + (i & 3) + 8 * (i >> 2) + 4 * half;
                        const int g = t / head_tiles, q = min((t - g * head_tiles) * BM + at, a.Lq - 1);
                        factor = static_cast<const uint8_t *>(a.keep)[((head0 + g) * a.Lq + q) * a.Lk + min(key, a.Lk - 1)] ? a.keep_scale : 0.f;
                    }
                    float d = dp[0][i];
                    if (KEEP || !FOLD) d = fmaf(d, factor, FOLD ? stp[BM + (i & 3) + 8 * (i >> 2)] : -row_delta[0][i]);
                    const float x = counts ? exp2_fast(FOLD ? s[0][i] * c : fmaf(s[0][i], c, -row_log[0][i])) : 0.f;
                    p[e] = x * factor;
                    ds[e] = DK ? x * d : 0.f;
                }
                to_operand(p, pf[u]);
                if (FINE) rest_operand(p, pf[u], pf_rest[u]);
                to_operand(ds, df[u]);
                if (FINE) rest_operand(ds, df[u], df_rest[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) {
                    Frag<T> f;
                    if (DV) {
                        read_columns<DP>(gt, sub * 32 + 16 * u, dt, lane, f);
                        mma(f, pf[u], dv[dt]);
                        if (FINE) mma(f, pf_rest[u], dv[dt]);
                    }
                    if (DK) {
                        read_columns<DP>(qt, sub * 32 + 16 * u, dt, lane, f);
                        mma(f, df[u], dk[dt]);
                        if (FINE) mma(f, df_rest[u], dk[dt]);
                    }
                }
            ahead<AHEAD, 2 * (DV && DK ? 2 : 1) * DP / 32, COLUMN_READS, FINE ? 2 : MMAS>();
        }
    }
    const int64_t dense = key < a.Lk ? (((int64_t)b * a.Lk + key) * a.kv_heads + hk) * a.D : -1, all = (int64_t)a.B * a.Lk * a.kv_heads * a.D;
    float *part = static_cast<float *>(a.workspace) + (int64_t)sp * 2 * all;
    if (sizeof(T) == 4 && stretch.index > 0 && dense >= 0) {
        if constexpr (DV) add_row(dv, (splits == 1 ? static_cast<const float *>(a.grad_value) : part) + dense, 1.f, a.D, half);
        if constexpr (DK) add_row(dk, (splits == 1 ? static_cast<const float *>(a.grad_key) : part + all) + dense, 1.f, a.D, half);
    }
    const float factor = sizeof(T) == 4 && stretch.index + 1 < stretch.count ? 1.f : a.scale;
    // (a key that does not count has P = 0, but 0 times an infinite or NaN grad_out is NaN)
    if constexpr (DV) zero_unless(counts, dv);
    if constexpr (DK) zero_unless(counts && !mask.one(), dk);
    __syncthreads();                          // everybody is done with the tiles: their memory carries the results out
    constexpr int REGION = 2 * BUF / NW;
    char *region = lds + wave * REGION;
    if constexpr (DV) {
        if (splits == 1) put_rows<T, DP, REGION>(dv, 1.f, region, static_cast<T *>(a.grad_value), dense, a.D, lane);
        else put_rows<float, DP, REGION>(dv, 1.f, region, part, dense, a.D, lane);
    }
    if constexpr (DK) {
        if (splits == 1) put_rows<T, DP, REGION>(dk, factor, region, static_cast<T *>(a.grad_key), dense, a.D, lane);
        else put_rows<float, DP, REGION>(dk, 1.f, region, part + all, dense, a.D, lane);
    }
}

// out[i] = factor * sum over splits of part[s * stride + i], four elements a thread; elements n .. 2 n - 1 (if any) belong to out2
template <typename T>
__global__ __launch_bounds__(256) void reduce_kernel(const float *__restrict__ part, int splits, int64_t stride, int64_t n, float factor,
                                                     T *__restrict__ out, float factor2, T *__restrict__ out2)
{
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= stride) return;
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
        const float4 v = *reinterpret_cast<const float4 *>(part + s * stride + i);
        o[0] += v.x; o[1] += v.y; o[2] += v.z; o[3] += v.w;
    }
    const float f = i < n ? factor : factor2;
    store4<T>(i < n ? out + i : out2 + (i - n), o[0] * f, o[1] * f, o[2] * f, o[3] * f);
}

// (`n`: elements of an output, a multiple of 8)
template <typename T>
void reduce(const cross_attention_args &a, int splits, int64_t n, float factor, void *out, float factor2, void *out2, hipStream_t stream)
{
    const int64_t stride = out2 ? 2 * n : n;
    hipLaunchKernelGGL(reduce_kernel<T>, dim3((unsigned)((stride / 4 + 255) / 256)), dim3(256), 0, stream,
                       static_cast<const float *>(a.workspace), splits, stride, n, factor, static_cast<T *>(out), factor2, static_cast<T *>(out2));
}

Plan query_plan(const cross_attention_args &a)
{
    const int bytes = row_bytes(a), n = rows_per_tile(bytes);
    return plan_for((int64_t)(a.heads / a.kv_heads) * a.Lq, (a.Lk + n - 1) / n, (int64_t)a.B * a.kv_heads, tile_lds(a),
                    bytes <= 64 ? 4 : bytes <= 128 ? 3 : bytes <= 256 ? 2 : 1, least_tiles(a));
}
Plan key_plan(const cross_attention_args &a)
{
    const int bytes = row_bytes(a), n = rows_per_tile(bytes);
    return plan_for(a.Lk, (int64_t)(a.heads / a.kv_heads) * ((a.Lq + n - 1) / n), (int64_t)a.B * a.kv_heads, tile_lds(a),
                    bytes <= 64 ? 3 : bytes <= 256 ? 2 : 1, least_tiles(a));
}

template <typename T, int DP, int NW, bool KEEP, bool FINE> void launch_query(const cross_attention_args &a, const Plan &p, float c, hipStream_t stream)
{
    constexpr int BN = rows_per_tile(Tile<T, DP>::ROW), LDS = 4 * BN * Tile<T, DP>::ROW + 2 * BN * 4, OCC = DP * (int)sizeof(T) >= 512 ? 1 : 2;
    const auto kernel = query_kernel<T, DP, NW, BN, OCC, KEEP, FINE>;
    RLIPV2_ONCE_PER_DEVICE((void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
    const int stretches = stretches_of(a, (a.Lk + BN - 1) / BN, p);
    for (int i = 0; i < stretches; ++i)
        hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)p.tiles * p.splits * a.B * a.kv_heads)), dim3(64 * NW), LDS, stream, a, p.tiles,
                           p.splits, Stretch{i, stretches}, c);
    if (p.splits > 1) {
        const int64_t n = (int64_t)a.B * a.Lq * a.heads * a.D;
        reduce<T>(a, p.splits, n, a.scale, a.grad_query, 0.f, nullptr, stream);
    }
}

template <typename T, int DP, int NW, bool DV, bool DK, bool KEEP, bool FINE> void launch_key_part(const cross_attention_args &a, const Plan &p, float c, hipStream_t stream)
{
    constexpr int BM = rows_per_tile(Tile<T, DP>::ROW), LDS = 4 * BM * Tile<T, DP>::ROW + 4 * BM * 4, OCC = DP * (int)sizeof(T) >= 512 ? 1 : 2;
    const auto kernel = key_kernel<T, DP, NW, BM, OCC, DV, DK, KEEP, FINE>;
    RLIPV2_ONCE_PER_DEVICE((void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
    const int stretches = stretches_of(a, (int64_t)(a.heads / a.kv_heads) * ((a.Lq + BM - 1) / BM), p);
    for (int i = 0; i < stretches; ++i)
        hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)p.tiles * p.splits * a.B * a.kv_heads)), dim3(64 * NW), LDS, stream, a, p.tiles,
                           p.splits, Stretch{i, stretches}, c);
}

template <typename T, int DP, int NW, bool KEEP, bool FINE> void launch_key(const cross_attention_args &a, const Plan &p, float c, hipStream_t stream)
{
    if constexpr (DP * sizeof(T) > 512) {
        launch_key_part<T, DP, NW, true, false, KEEP, FINE>(a, p, c, stream);
        launch_key_part<T, DP, NW, false, true, KEEP, FINE>(a, p, c, stream);
    } else {
        launch_key_part<T, DP, NW, true, true, KEEP, FINE>(a, p, c, stream);
    }
    if (p.splits > 1) {
        const int64_t n = (int64_t)a.B * a.Lk * a.kv_heads * a.D;
        reduce<T>(a, p.splits, n, 1.f, a.grad_value, a.scale, a.grad_key, stream);
    }
}

template <typename T, int DP, bool KEEP, bool FINE> int run(const cross_attention_args &a, hipStream_t stream)
{
    const float c = a.scale * 1.4426950408889634f;
    const Plan pq = query_plan(a), pk = key_plan(a);
    // (small heads: dS adds up to nothing over a row but its rounding errors do not, and the smaller the head, the more of what cancels)
    constexpr bool FQ = FINE || (sizeof(T) == 2 && DP == 32 && !KEEP);
    if (a.Lq > 0)
        pq.waves == 1 ? launch_query<T, DP, 1, KEEP, FQ>(a, pq, c, stream) : pq.waves == 2 ? launch_query<T, DP, 2, KEEP, FQ>(a, pq, c, stream)
                                                                                           : launch_query<T, DP, 4, KEEP, FQ>(a, pq, c, stream);
    if (!a.grad_key || a.Lk == 0) return hipGetLastError() == hipSuccess ? MSDA_OK : MSDA_ERR_LAUNCH;
    pk.waves == 1 ? launch_key<T, DP, 1, KEEP, FINE>(a, pk, c, stream) : pk.waves == 2 ? launch_key<T, DP, 2, KEEP, FINE>(a, pk, c, stream)
                                                                                       : launch_key<T, DP, 4, KEEP, FINE>(a, pk, c, stream);
    return hipGetLastError() == hipSuccess ? MSDA_OK : MSDA_ERR_LAUNCH;
}

template <typename T, bool KEEP, bool FINE> int by_size(const cross_attention_args &a, hipStream_t stream)
{
    return a.D <= 32 ? run<T, 32, KEEP, FINE>(a, stream) : a.D <= 64 ? run<T, 64, KEEP, FINE>(a, stream)
         : a.D <= 128 ? run<T, 128, KEEP, FINE>(a, stream) : run<T, 256, KEEP, FINE>(a, stream);
}

template <typename T> int by_mask(const cross_attention_args &a, hipStream_t stream)
{
    if constexpr (sizeof(T) == 2)
        if (few_probabilities(a)) return by_size<T, false, true>(a, stream);
    return a.keep ? by_size<T, true, false>(a, stream) : by_size<T, false, false>(a, stream);
}

}  // namespace

namespace xattn {

int short_side(const cross_attention_args &a);
int short_splits(const cross_attention_args &a);
void launch_short(const cross_attention_args &a, int splits, hipStream_t stream);
size_t forward_workspace(const cross_attention_args &a);
int forward(const cross_attention_args &a, hipStream_t stream);

// (the two passes run one after the other on the same workspace)
size_t backward_workspace(const cross_attention_args &a)
{
    if (const int side = short_side(a)) {
        const int splits = short_splits(a);
        return splits == 1 || !a.grad_key ? 0 : (size_t)splits * (side == 1 ? 2 * (size_t)a.Lk * a.kv_heads : (size_t)a.Lq * a.heads) * a.B * a.D * sizeof(float);
    }
    const Plan pq = query_plan(a), pk = a.grad_key ? key_plan(a) : Plan{1, 1, 1};
    const size_t q = pq.splits == 1 ? 0 : (size_t)pq.splits * a.B * a.Lq * a.heads * a.D * sizeof(float);
    const size_t k = pk.splits == 1 ? 0 : (size_t)pk.splits * 2 * a.B * a.Lk * a.kv_heads * a.D * sizeof(float);
    return q > k ? q : k;
}

int backward(const cross_attention_args &a, hipStream_t stream)
{
    if (const int side = short_side(a)) {
        const int splits = short_splits(a);
        launch_short(a, splits, stream);
        if (splits > 1 && side == 1 && a.grad_key)
            reduce<bf16_t>(a, splits, (int64_t)a.B * a.Lk * a.kv_heads * a.D, a.scale, a.grad_key, 1.f, a.grad_value, stream);
        else if (splits > 1 && side == 2)
            reduce<bf16_t>(a, splits, (int64_t)a.B * a.Lq * a.heads * a.D, a.scale, a.grad_query, 0.f, nullptr, stream);
        return hipGetLastError() == hipSuccess ? MSDA_OK : MSDA_ERR_LAUNCH;
    }
    return a.dtype == MSDA_BF16 ? by_mask<bf16_t>(a, stream) : by_mask<float>(a, stream);
}

bool sizes_ok(const cross_attention_args &a)
{
    if (a.B < 0 || a.Lq < 0 || a.Lk < 0 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads) return false;
    if (a.D < 8 || a.D > 256 || a.D % 8) return false;
    // Rows of a key head are counted in 32 bits, and so are the threads of a launch: 256 per 128 rows of a key head's longer side, 512 per
    // key head where a side is short.  (Splits add at most 2304 workgroups: nine fit on each of 256 compute units.)
    const int64_t rows = (int64_t)(a.heads / a.kv_heads) * a.Lq, side = rows > a.Lk ? rows : a.Lk, groups = (int64_t)a.B * a.kv_heads;
    const int64_t limit = ((int64_t)1 << 32) / 512 - 4096;
    return side <= (int64_t)1 << 30 && groups <= limit && (side + 127) / 128 <= 2 * limit / (groups > 0 ? groups : 1);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// (1 / (scale log2 e) times a row's logarithm stays finite: the key pass starts its logits from there)
bool scale_ok(const cross_attention_args &a) { return a.scale >= 0.99e-30f && a.scale < kInf; }

int check(const cross_attention_args *a, bool backward)
{
    if (!a) return MSDA_ERR_NULL_POINTER;
    if (a->dtype != MSDA_BF16 && a->dtype != MSDA_F32) return MSDA_ERR_BAD_DTYPE;
    if (!sizes_ok(*a) || !scale_ok(*a)) return MSDA_ERR_BAD_SHAPE;
    if (a->B == 0 || (a->Lq == 0 && (!backward || a->Lk == 0))) return MSDA_OK;
    const void *need[] = {a->query, a->out};
    if (a->Lq > 0)
        for (const void *p : need)
            if (!p) return MSDA_ERR_NULL_POINTER;
    if (a->Lk > 0 && (!a->key || !a->value)) return MSDA_ERR_NULL_POINTER;
    const int per16 = a->dtype == MSDA_BF16 ? 8 : 4;
    for (int i = 0; i < 3; ++i)
        if (a->query_stride[i] % per16 || a->key_stride[i] % per16 || a->value_stride[i] % per16) return MSDA_ERR_ALIGNMENT;
    // (a thread's offset inside a tile of 64 rows is 32 bits)
    const int64_t far = ((int64_t)1 << 32) / 64 / (a->dtype == MSDA_BF16 ? 2 : 4);
    for (const int64_t s : {a->query_stride[1], a->key_stride[1], a->value_stride[1], backward ? a->grad_out_stride[1] : 0})
        if (s < 0 || s >= far) return MSDA_ERR_BAD_SHAPE;
    const void *operands[] = {a->query, a->key, a->value, a->out, a->out_low};
    for (const void *p : operands)
        if (!aligned16(p)) return MSDA_ERR_ALIGNMENT;
    if (backward) {
        if (a->Lq > 0 && (!a->grad_out || !a->grad_query || !a->stats || !a->delta)) return MSDA_ERR_NULL_POINTER;
        if (!a->grad_key != !a->grad_value) return MSDA_ERR_NULL_POINTER;
        for (int i = 0; i < 3; ++i)
            if (a->grad_out_stride[i] % per16) return MSDA_ERR_ALIGNMENT;
        const void *grads[] = {a->grad_out, a->grad_query, a->grad_key, a->grad_value};
        for (const void *p : grads)
            if (!aligned16(p)) return MSDA_ERR_ALIGNMENT;
    }
    const size_t need_bytes = backward ? backward_workspace(*a) : forward_workspace(*a);
    if (need_bytes && (!a->workspace || a->workspace_bytes < need_bytes)) return MSDA_ERR_NULL_POINTER;
    return aligned16(a->workspace) ? MSDA_OK : MSDA_ERR_ALIGNMENT;
}

}  // namespace xattn

extern "C" size_t cross_attention_args_bytes(void) { return sizeof(cross_attention_args); }

extern "C" int cross_attention_supported(const cross_attention_args *a)
{
    return a && (a->dtype == MSDA_BF16 || a->dtype == MSDA_F32) && xattn::sizes_ok(*a) && xattn::scale_ok(*a);
}

extern "C" int cross_attention_short_keys(const cross_attention_args *a) { return cross_attention_supported(a) && xattn::short_side(*a) == 1; }

extern "C" size_t cross_attention_workspace_bytes(const cross_attention_args *a, int backward)
{
    if (!cross_attention_supported(a) || a->B == 0 || (a->Lq == 0 && (!backward || a->Lk == 0))) return 0;
    return backward ? xattn::backward_workspace(*a) : xattn::forward_workspace(*a);
}

extern "C" int cross_attention_forward(const cross_attention_args *a, void *stream)
{
    if (const int st = xattn::check(a, false)) return st;
    if (a->B == 0 || a->Lq == 0) return MSDA_OK;
    (void)hipGetLastError();                  // (an error that an earlier call left is not this one's)
    return xattn::forward(*a, static_cast<hipStream_t>(stream));
}

extern "C" int cross_attention_backward(const cross_attention_args *a, void *stream)
{
    if (const int st = xattn::check(a, true)) return st;
    if (a->B == 0 || (a->Lq == 0 && a->Lk == 0)) return MSDA_OK;
    (void)hipGetLastError();                  // (an error that an earlier call left is not this one's)
    return xattn::backward(*a, static_cast<hipStream_t>(stream));
}
