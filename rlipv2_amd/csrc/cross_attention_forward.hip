// cross_attention_forward.hip -- softmax(scale q k^T) v over states of another length, one pass over the keys
// (include/rlipv2_attention.h; the layout of the products: cross_attention_device.h).
//
// A wave holds 32 query rows (the rows of the heads that share a key head follow each other), a workgroup of 1, 2 or 4 waves
// walks over the keys in tiles of BN.  Two LDS buffers: the copy of tile t + 1 is issued before tile t is computed, one barrier
// per tile.  Per tile: S^T = K Q^T, the row's running maximum m and sum l, O^T = O^T 2^(m_old - m_new) + V^T P^T.  The
// exponentials are base 2 with scale * log2(e) folded into one multiply-add.  P is rounded to the operands' type for the second
// product (values in [0, 1], relative 2^-9 in bf16); sums, maxima and the accumulators are float32.
//
// The accumulators of S^T start from the mask (0 or -infinity per key, from LDS), so masking costs no instruction per logit.  The rescaling
// is skipped where no row of the wave got a new maximum.
//
// Few query rows: the keys are cut into splits (plan_for), each writes its normalised float32 result and its logarithm of the sum, and
// combine_kernel joins them in the order of the splits.
//
// What bounds it, measured (bf16; this kernel's averages of 20 calls in a kernel trace, profiles/operators_kernel_stats.csv; under long
// matrix work the clock settles, the last calls are 7 % faster): one token of eight requests, four heads of 128 per key head, 22 223 keys
// 131 us (569 MB: 4.3 TB/s, HBM); 64 rows of 8 heads of 256 over 22 223 keys, batch 4, 166 us (590 MB: 3.6 TB/s); 22 223 rows over 64 keys,
// heads of 256, 187 us (728 MB: 3.9 TB/s, HBM); 300 rows over 22 223 keys, heads of 32, 87 us (32 exponentials, 96 other vector and 8
// matrix instructions per wave and tile: vector issue; 384 rows for 300, two of a last workgroup's four waves without any); 2048 rows over 4096 keys, 16
// heads of 128, batch 4, 327 us (840 TFLOP/s; 304 us, 905 in the last calls; a large library product reaches 1210 on this card): matrix and
// vector instructions of two waves per SIMD in turn.
// The copies' wait in front of the loop instead of inside it: single tokens 683 -> 144 us; reads ahead of the matrix instructions and
// copies with scalar bases: the 2048 rows 451 -> 350 us; variants without the dropout mask: -> 302 us (timed without the trace).  float32 at the
// same size 2114 us, 130 TFLOP/s (library product 154); heads of 256, 5000 rows over 5000 keys: 92.
#include "cross_attention_device.h"

namespace {

using namespace msda;
using namespace xattn;

// KEEP: with a dropout mask
template <typename T, int DP, int NW, int BN, int OCC, bool KEEP>
__global__ __launch_bounds__(64 * NW, OCC) void forward_kernel(cross_attention_args a, int row_tiles, int splits, Stretch stretch, float c)
{
    constexpr int THREADS = 64 * NW, NSUB = BN / 32, KB = BN * Tile<T, DP>::ROW, BUF = 2 * KB;
    constexpr bool AHEAD = !KEEP;
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

    Frag<T> qf[DP / 16];
    {
        const T *row = static_cast<const T *>(a.query) + (int64_t)b * a.query_stride[0] + (int64_t)q * a.query_stride[1] +
                       (int64_t)head * a.query_stride[2];
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) load_operand(row, 16 * s + 8 * half, a.D, ok, qf[s]);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) settle(qf[s]);
    }
    const T *kbase = static_cast<const T *>(a.key) + (int64_t)b * a.key_stride[0] + (int64_t)hk * a.key_stride[2];
    const T *vbase = static_cast<const T *>(a.value) + (int64_t)b * a.value_stride[0] + (int64_t)hk * a.value_stride[2];
    const uint8_t *keep = static_cast<const uint8_t *>(a.keep) + (((int64_t)b * a.heads + head) * a.Lq + q) * a.Lk;

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
    const int64_t at = ((int64_t)sp * a.B * a.kv_heads + bh) * rows.count + r, all = (int64_t)splits * a.B * a.kv_heads * rows.count;
    float *part = static_cast<float *>(a.workspace), *held = part + (splits == 1 ? 0 : all * (a.D + 1)) + 2 * at;
    float m = -kInf, scaled = -kInf, l = 0.f; // the maximum, c times it as the exponents subtract it; l: this half's keys only
    // (float32: held = the maximum and the sum that the stretches before left; the sum's halves meet at the end)
    const bool more = sizeof(T) == 4 && stretch.index > 0 && ok;
    if (more) {
        m = held[0];
        scaled = m * c;
    }
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

        // (the accumulators start from the mask: a key that does not count has a row of zeros in LDS and ends at -infinity)
        f32x16 s[NSUB];
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub) load_quads(bias + (t & 1) * BN + sub * 32 + 4 * half, s[sub]);
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                Frag<T> f;
                read_rows<DP>(kt, sub * 32 + (lane & 31), k, half, f);
                mma(f, qf[k], s[sub]);
            }
        if (AHEAD) XATTN_SCHED_GROUP(0x100, 4 * NSUB);
        ahead<AHEAD, NSUB * DP / 16, ROW_READS, MMAS>();
        float top = m;
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[sub][i]);
        top = fmaxf(top, other_half(top));
        // (from the rounded products: an unchanged maximum gives exactly 1, no drift over the tiles)
        const float base = top == -kInf ? 0.f : top * c, shrink = exp2_fast(scaled - base);      // (none before: 0)
        m = top;
        scaled = top * c;
        float sum = 0.f;
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[sub][i] = exp2_fast(fmaf(s[sub][i], c, -base));
                sum += s[sub][i];
            }
        l = fmaf(l, shrink, sum);
        if (__builtin_amdgcn_ballot_w64(shrink != 1.f)) {
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[dt][i] *= shrink;
        }
        if (KEEP) {
#pragma unroll
            for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int key = t * BN + sub * 32 + (i & 3) + 8 * (i >> 2) + 4 * half;
                    s[sub][i] *= keep[min(key, a.Lk - 1)] ? a.keep_scale : 0.f;
                }
        }
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = s[sub][8 * u + e];
                Frag<T> pf;
                to_operand(p, pf);
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) {
                    Frag<T> f;
                    read_columns<DP>(vt, sub * 32 + 16 * u, dt, lane, f);
                    mma(f, pf, acc[dt]);
                }
            }
        ahead<AHEAD, NSUB * 2 * DP / 32, COLUMN_READS, MMAS>();
    }

    const int64_t dense = (((int64_t)b * a.Lq + q) * a.heads + head) * a.D;
    if (more) {
        const float f = exp2_fast(held[0] * c - (scaled == -kInf ? 0.f : scaled));
        add_row(acc, splits == 1 ? static_cast<const float *>(a.out) + dense : part + at * a.D, f, a.D, half);
        if (half == 0) l = fmaf(held[1], f, l);
    }
    const float total = l + other_half(l);
    const float inv = total == 0.f ? 0.f : 1.f / total, log_sum = scaled + log2_fast(total);
    __syncthreads();                          // everybody is done with the tiles: their memory carries the results out
    constexpr int REGION = 2 * BUF / NW;
    char *region = lds + wave * REGION;
    if (sizeof(T) == 4 && stretch.index + 1 < stretch.count) {
        float *to = splits == 1 ? static_cast<float *>(a.out) : part;
        put_rows<float, DP, REGION>(acc, 1.f, region, to, !ok ? -1 : splits == 1 ? dense : at * a.D, a.D, lane);
        if (ok && half == 0) {
            held[0] = m;
            held[1] = total;
        }
        return;
    }
    if (splits == 1) {
        put_rows<T, DP, REGION>(acc, inv, region, static_cast<T *>(a.out), ok ? dense : -1, a.D, lane);
        if (sizeof(T) == 2 && a.out_low)
            put_rows<T, DP, REGION, true>(acc, inv, region, static_cast<T *>(a.out_low), ok ? dense : -1, a.D, lane);
        if (a.stats && ok && half == 0)
            static_cast<float *>(a.stats)[((int64_t)b * a.heads + head) * a.Lq + q] = total == 0.f ? kInf : log_sum;
    } else {
        put_rows<float, DP, REGION>(acc, inv, region, part, ok ? at * a.D : -1, a.D, lane);
        if (ok && half == 0) part[all * a.D + at] = total == 0.f ? -kInf : log_sum;
    }
}

// joins the splits of a row: out = sum_i 2^(L_i - L) out_i,  L = log2 sum_i 2^L_i.  A workgroup has 256 / (Q G) rows; a thread takes four
// elements (Q = a power of two >= D / 4) of every G-th split, the G partial results are joined through LDS in a fixed order.
template <typename T> __global__ __launch_bounds__(256) void combine_kernel(cross_attention_args a, int splits, int Q, int G_)
{
    __shared__ float lds_top[256], lds_sum[256];
    __shared__ float4 lds_o[256];
    const int tid = threadIdx.x, quad = tid & (Q - 1), sg = (tid / Q) & (G_ - 1);
    const int G = a.heads / a.kv_heads, rows_per_block = 256 / (Q * G_);
    const int64_t all = (int64_t)a.B * a.kv_heads * G * a.Lq;
    const int64_t row = (int64_t)blockIdx.x * rows_per_block + tid / (Q * G_);
    const int d = quad * 4;
    const bool in = row < all && d < a.D;
    const float *part = static_cast<const float *>(a.workspace), *logs = part + (int64_t)splits * all * a.D;
    float top = -kInf, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    if (in) {
        for (int s = sg; s < splits; s += G_) top = fmaxf(top, logs[s * all + row]);
        const float base = top == -kInf ? 0.f : top;
        for (int s = sg; s < splits; s += G_) {
            const float w = exp2_fast(logs[s * all + row] - base);
            const float4 v = *reinterpret_cast<const float4 *>(part + (s * all + row) * a.D + d);
            sum += w;
            o[0] = fmaf(w, v.x, o[0]); o[1] = fmaf(w, v.y, o[1]); o[2] = fmaf(w, v.z, o[2]); o[3] = fmaf(w, v.w, o[3]);
        }
    }
    lds_top[tid] = top;
    lds_sum[tid] = sum;
    lds_o[tid] = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    if (!in || sg != 0) return;
    for (int g = 1; g < G_; ++g) top = fmaxf(top, lds_top[tid + g * Q]);
    const float base = top == -kInf ? 0.f : top;
    sum = o[0] = o[1] = o[2] = o[3] = 0.f;
    for (int g = 0; g < G_; ++g) {
        const float w = exp2_fast(lds_top[tid + g * Q] - base);            // (a group without splits: top -inf, weight 0)
        const float4 v = lds_o[tid + g * Q];
        sum = fmaf(w, lds_sum[tid + g * Q], sum);
        o[0] = fmaf(w, v.x, o[0]); o[1] = fmaf(w, v.y, o[1]); o[2] = fmaf(w, v.z, o[2]); o[3] = fmaf(w, v.w, o[3]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t bh = row / ((int64_t)G * a.Lq);
    const int rr = (int)(row - bh * G * a.Lq), b = (int)(bh / a.kv_heads), g = rr / a.Lq, q = rr - g * a.Lq;
    const int head = (int)(bh - (int64_t)b * a.kv_heads) * G + g;
    const int64_t at = (((int64_t)b * a.Lq + q) * a.heads + head) * a.D + d;
    for (float &x : o) x *= inv;
    store4<T>(static_cast<T *>(a.out) + at, o[0], o[1], o[2], o[3]);
    if (sizeof(T) == 2 && a.out_low) {
        rounded_off(o);
        store4<T>(static_cast<T *>(a.out_low) + at, o[0], o[1], o[2], o[3]);
    }
    if (a.stats && d == 0)
        static_cast<float *>(a.stats)[((int64_t)b * a.heads + head) * a.Lq + q] = sum == 0.f ? kInf : base + log2_fast(sum);
}

Plan plan_of(const cross_attention_args &a)
{
    const int bytes = row_bytes(a), n = rows_per_tile(bytes);
    return plan_for((int64_t)(a.heads / a.kv_heads) * a.Lq, (a.Lk + n - 1) / n, (int64_t)a.B * a.kv_heads, tile_lds(a),
                    bytes <= 64 ? 4 : bytes <= 128 ? 3 : bytes <= 512 ? 2 : 1, least_tiles(a));
}

template <typename T, int DP, int NW, bool KEEP> int launch(const cross_attention_args &a, const Plan &p, hipStream_t stream)
{
    constexpr int BN = rows_per_tile(Tile<T, DP>::ROW), LDS = 4 * BN * Tile<T, DP>::ROW + 2 * BN * 4, OCC = DP * (int)sizeof(T) > 512 ? 1 : 2;
    const auto kernel = forward_kernel<T, DP, NW, BN, OCC, KEEP>;
    RLIPV2_ONCE_PER_DEVICE((void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
    const int64_t groups = (int64_t)p.tiles * p.splits * a.B * a.kv_heads;
    const int stretches = stretches_of(a, (a.Lk + BN - 1) / BN, p);
    for (int i = 0; i < stretches; ++i)
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(64 * NW), LDS, stream, a, p.tiles, p.splits, Stretch{i, stretches},
                           a.scale * 1.4426950408889634f);
    if (p.splits > 1) {
        int Q = 2, G = 1;
        while (Q < a.D / 4) Q *= 2;
        const int64_t n = (int64_t)a.B * a.heads * a.Lq;
        while (G < p.splits && 2 * G * Q <= 256 && n * G * Q < 256 * 1024) G *= 2;      // (until there are 1024 workgroups)
        const int64_t per = 256 / (Q * G);
        hipLaunchKernelGGL(combine_kernel<T>, dim3((unsigned)((n + per - 1) / per)), dim3(256), 0, stream, a, p.splits, Q, G);
    }
    return hipGetLastError() == hipSuccess ? MSDA_OK : MSDA_ERR_LAUNCH;
}

template <typename T, int DP> int by_waves(const cross_attention_args &a, const Plan &p, hipStream_t stream)
{
    if (a.keep)
        return p.waves == 1 ? launch<T, DP, 1, true>(a, p, stream) : p.waves == 2 ? launch<T, DP, 2, true>(a, p, stream)
                                                                                  : launch<T, DP, 4, true>(a, p, stream);
    return p.waves == 1 ? launch<T, DP, 1, false>(a, p, stream) : p.waves == 2 ? launch<T, DP, 2, false>(a, p, stream)
                                                                               : launch<T, DP, 4, false>(a, p, stream);
}

template <typename T> int by_size(const cross_attention_args &a, const Plan &p, hipStream_t stream)
{
    return a.D <= 32 ? by_waves<T, 32>(a, p, stream) : a.D <= 64 ? by_waves<T, 64>(a, p, stream)
         : a.D <= 128 ? by_waves<T, 128>(a, p, stream) : by_waves<T, 256>(a, p, stream);
}

}  // namespace

namespace xattn {

size_t forward_workspace(const cross_attention_args &a)
{
    const Plan p = plan_of(a);
    const int n = rows_per_tile(row_bytes(a));
    const size_t rows = (size_t)p.splits * a.B * a.heads * a.Lq, held = stretches_of(a, (a.Lk + n - 1) / n, p) > 1 ? 2 : 0;
    return rows * ((p.splits == 1 ? 0 : a.D + 1) + held) * sizeof(float);
}

int forward(const cross_attention_args &a, hipStream_t stream)
{
    const Plan p = plan_of(a);
    return a.dtype == MSDA_BF16 ? by_size<bf16_t>(a, p, stream) : by_size<float>(a, p, stream);
}

}  // namespace xattn
