// nl_experts.h -- kernels of the feed-forward of experts (include/nanollama_ops.h): choice of experts, grouping of tokens by expert, the
// experts' products, the close of a block.  Matrices and rows are plain row-major here, a product's operands are gathered as fragments
// (nl_frag.h) from where they lie: a token's row through its slot, an expert's matrix as the caller has it.
//
//   slot   t * k + j: the j-th choice of token t            place   its position among all slots ordered by (expert, slot)
#pragma once
#include "nl_frag.h"
#include "nl_ops.h"

namespace nl {

// ---------------------------------------------------------------- route ---

// largest value of the wavefront (as unsigned integers), in every lane
template <int CTRL> __device__ __forceinline__ unsigned dpp_umax(unsigned v) {
    return max(v, (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ unsigned wave_umax(unsigned v) {
    v = dpp_umax<0x140>(dpp_umax<0x141>(dpp_umax<0x4E>(dpp_umax<0xB1>(v))));
    return max(max((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 16)),
               max((unsigned)__builtin_amdgcn_readlane((int)v, 32), (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
}
// order-preserving image of a float, 1 at least for every number (0: out); -0 and +0 are one
__device__ __forceinline__ unsigned order_u32(float v) {
    const unsigned u = __float_as_uint(v + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_f32(unsigned u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

// A wavefront per token; expert e is element e / 64 of lane e % 64.
// With a bias the keys sigmoid(l) + b are 32-bit numbers within KEY_ERR (1 + |b|) of the exact ones: where two neighbours among the chosen ones and
// the best one left are nearer than twice that, the row's keys are computed again in 64 bits.
constexpr float KEY_ERR = 1e-6f;
template <int NE>
__global__ void __launch_bounds__(256) route_kernel(RouteParams P) {
    const int t = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= P.n) return;
    const float *row = P.logits + (long long)t * P.ld;
    float l[NE], b[NE];
    bool out[NE];
#pragma unroll
    for (int i = 0; i < NE; i++) {
        const int e = lane + 64 * i;
        l[i] = e < P.experts ? row[e] : -INFINITY;
        b[i] = P.bias && e < P.experts ? P.bias[e] : 0.f;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NE; i++) {
        out[i] = !(l[i] > -INFINITY) || !(b[i] > -INFINITY);       // (NaN too)
        if (out[i]) l[i] = -INFINITY;
        m = fmaxf(m, l[i]);
    }
    m = order_f32(wave_umax(order_u32(m)));
    unsigned key[NE];
    float off = 0.f;                                     // how far keys may be off, together
#pragma unroll
    for (int i = 0; i < NE; i++) {
        const float v = P.bias ? sigmoid_f32(l[i]) + b[i] : l[i];
        key[i] = out[i] ? 0 : order_u32(v);
        if (P.bias && !out[i]) off = fmaxf(off, 2.f * KEY_ERR * (1.f + fminf(fabsf(b[i]), 1e30f)));
    }
    int pick = -1;                                       // lane j: the j-th choice
    float score = 0.f;                                   // ... its logit
    {
        unsigned k[NE];
#pragma unroll
        for (int i = 0; i < NE; i++) k[i] = key[i];
        const float far = P.bias ? __uint_as_float(wave_umax(__float_as_uint(off))) : 0.f;
        float before = INFINITY;
        bool near = false;
        for (int j = 0; j <= P.k; j++) {                 // (one more than are chosen: the best that is left)
            if (j == P.k && !P.bias) break;
            unsigned mine = 0;
            int at = 0;
#pragma unroll
            for (int i = NE - 1; i >= 0; i--)
                if (k[i] >= mine) { mine = k[i]; at = i; }
            const unsigned best = wave_umax(mine);
            if (best == 0) break;
            if (P.bias) {
                const float v = order_f32(best);
                near |= !(before - v > far) && j > 0;
                before = v;
                if (j == P.k) break;
            }
            // equal ones: the lowest number
            unsigned e = mine == best ? (unsigned)(lane + 64 * at) : 0xffffffffu;
            const unsigned long long who = __ballot(mine == best);
            e = who & (who - 1) ? ~wave_umax(~e) : (unsigned)__builtin_amdgcn_readlane((int)e, __ffsll((long long)who) - 1);
            float le = 0.f;
#pragma unroll
            for (int i = 0; i < NE; i++) {
                if (i == (int)(e >> 6)) le = l[i];
                if (e == (unsigned)(lane + 64 * i)) k[i] = 0;
            }
            le = lane_value(le, e & 63);
            if (lane == j) { pick = (int)e; score = le; }
        }
        if (near) {                                      // (rare: the same in 64 bits)
            double kd[NE];
            unsigned gone = 0;
#pragma unroll
            for (int i = 0; i < NE; i++) {
                kd[i] = 1.0 / (1.0 + exp(-(double)l[i])) + (double)b[i];
                if (out[i]) gone |= 1u << i;
            }
            pick = -1;
            for (int j = 0; j < P.k; j++) {
                double mine = 0.0;
                int at = -1;
#pragma unroll
                for (int i = 0; i < NE; i++)
                    if (!(gone >> i & 1) && (at < 0 || kd[i] > mine)) { mine = kd[i]; at = i; }
                int e = at < 0 ? -1 : lane + 64 * at;
                for (int s = 1; s < 64; s <<= 1) {
                    const double ov = __shfl_xor(mine, s);
                    const int oe = __shfl_xor(e, s);
                    if (oe >= 0 && (e < 0 || ov > mine || (ov == mine && oe < e))) { mine = ov; e = oe; }
                }
                if (e < 0) break;
                float le = 0.f;
#pragma unroll
                for (int i = 0; i < NE; i++) {
                    if (i == e >> 6) le = l[i];
                    if (e == lane + 64 * i) gone |= 1u << i;
                }
                le = lane_value(le, e & 63);
                if (lane == j) { pick = e; score = le; }
            }
        }
    }
    float w = 0.f;
    if (pick >= 0 && !P.sigmoid) w = score == m ? 1.f : exp_f32(fmaxf(score - m, -1e4f));
    if (P.sigmoid) {
        // shares of sigmoids: e^(l - M) / (1 + e^l) with M the largest logit chosen, where that is negative (all may be 0 in 32 bits)
        float top = 0.f;
        if (P.renorm) top = fminf(order_f32(wave_umax(pick >= 0 ? order_u32(score) : 1u)), 0.f);
        if (pick >= 0) w = top < 0.f ? exp_f32(fmaxf(score - top, -1e4f)) * rcp_f32(1.f + exp_f32(fmaxf(score, -1e4f))) : sigmoid_f32(score);
    }
    float sum = 1.f;
    if (P.renorm) sum = wave_sum(w);
    else if (!P.sigmoid) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NE; i++) s += out[i] ? 0.f : l[i] == m ? 1.f : exp_f32(fmaxf(l[i] - m, -1e4f));
        sum = wave_sum(s);
    }
    if (lane < P.k) {
        P.ids[(long long)t * P.k + lane] = pick;
        P.weights[(long long)t * P.k + lane] = sum > 0.f ? w / sum * P.scale : 0.f;
    }
}

// ----------------------------------------------------------------- plan ---

// Workgroup e finds the places of expert e: how many slots go to lower experts, and its own slots in order.  Every workgroup reads all ids
// (L2), which saves a second launch for the sums over experts.  The last one leaves the end of the list too.
__global__ void __launch_bounds__(1024) plan_kernel(const int *ids, int nslots, int experts, int *offs, int *order) {
    __shared__ int less[16], mine[16];
    const int e = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int per = ((nslots + 15) / 16 + 63) & ~63, lo = min(w * per, nslots), hi = min(lo + per, nslots);      // this wavefront's slots
    int nl = 0, nm = 0;
    for (int s = lo; s < hi; s += 64) {
        const int id = s + lane < hi ? ids[s + lane] : -1;
        nl += __popcll(__ballot(id >= 0 && id < e));
        nm += __popcll(__ballot(id == e));
    }
    if (lane == 0) { less[w] = nl; mine[w] = nm; }
    __syncthreads();
    int at = 0, before = 0, all = 0;
    for (int i = 0; i < 16; i++) {
        at += less[i];
        if (i < w) before += mine[i];
        all += mine[i];
    }
    if (threadIdx.x == 0) {
        offs[e] = at;
        if (e == experts - 1) offs[experts] = at + all;
    }
    at += before;
    for (int s = lo; s < hi; s += 64) {
        const int id = s + lane < hi ? ids[s + lane] : -1;
        const unsigned long long m = __ballot(id == e);
        if (id == e) order[at + __popcll(m & ((1ull << lane) - 1))] = s + lane;
        at += __popcll(m);
    }
}

// tile number `tile` of the experts' places cut into tiles of BT: expert, first place, places; false: there are not that many.
// Every wavefront finds it by itself: a lane counts the tiles of a run of experts, a scan finds the lane.
template <int BT>
__device__ __forceinline__ bool find_tile(const int *offs, int experts, int tile, int &e, int &first, int &count) {
    const int lane = threadIdx.x & 63, per = (experts + 63) >> 6, e0 = lane * per;
    int mine = 0, lo = offs[min(e0, experts)];
    for (int i = 0, a = lo; i < per; i++) {
        const int b = offs[min(e0 + i + 1, experts)];
        mine += (b - a + BT - 1) / BT;
        a = b;
    }
    int upto = mine;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const int o = __shfl_up(upto, s);
        if (lane >= s) upto += o;
    }
    const unsigned long long who = __ballot(upto > tile);
    if (!who) return false;
    const int at = __ffsll((long long)who) - 1;
    int skip = tile - __builtin_amdgcn_readlane(upto - mine, at);
    e = at * per;
    int a = __builtin_amdgcn_readfirstlane(offs[e]);
    for (;; e++) {
        const int b = __builtin_amdgcn_readfirstlane(offs[e + 1]), n = (b - a + BT - 1) / BT;
        if (skip < n) { first = a + skip * BT; count = min(BT, b - first); return true; }
        skip -= n;
        a = b;
    }
}

// ------------------------------------------------------------- products ---

// a lane's run of 8 elements from k0 on of a row of K, zero behind its end.  VEC: 16-byte pieces, which lie within the row or behind it
template <bool VEC> __device__ __forceinline__ Frag<bf16> load_run(const bf16 *row, int k0, int K) {
    Frag<bf16> f;
    frag_zero(f);
    if constexpr (VEC) {
        if (k0 < K) f.v = *reinterpret_cast<const bf16x8 *>(row + k0);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (k0 + j < K) f.v[j] = row[k0 + j];
    }
    return f;
}
template <bool VEC> __device__ __forceinline__ Frag<float> load_run(const float *row, int k0, int K) {
    Frag<float> f;
    frag_zero(f);
    if constexpr (VEC) {
        if (k0 < K) f.a = *reinterpret_cast<const f32x4 *>(row + k0);
        if (k0 + 4 < K) f.b = *reinterpret_cast<const f32x4 *>(row + k0 + 4);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (k0 + j < K) frag_set(f, j, row[k0 + j]);
    }
    return f;
}
template <typename T> __device__ __forceinline__ void put_rows(T *p, int row, int rows, f32x4 v) {     // four consecutive ones, those that exist
    if (row + 3 < rows && (rows & 3) == 0) put4(p + row, v);
    else
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (row + i < rows) put(p + row + i, v[i]);
}
template <bool SILU> __device__ __forceinline__ f32x4 activate(f32x4 gate, f32x4 up) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = gate[i] * sigmoid_f32(SILU ? gate[i] : gelu_arg(gate[i])) * up[i];
    return v;
}

// 16 places x 16 R rows of one expert by a workgroup, K dealt to its four wavefronts, fragments straight to registers.  FIRST: gate and up rows of
// the tokens -> h; else rows of down of h -> part
// (32-bit: a third rounding to bfloat16, beside the activation's and the sum's, would make the error 1.2 times as large: 2.9e-3 instead of 2.4e-3).
template <typename T, bool FIRST, bool VEC, int R>
__global__ void __launch_bounds__(256) experts_few_kernel(ExpertsParams P) {
    constexpr int M = FIRST ? 2 : 1, N = R * M;
    __shared__ __align__(16) f32x4 red[4][N][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int rows = FIRST ? P.ff : P.dim, K = FIRST ? P.dim : P.ff, row0 = blockIdx.x * 16 * R;
    int e, first, count;
    if (!find_tile<16>(P.offs, P.experts, blockIdx.y, e, first, count)) return;
    const int place = first + min(c, count - 1), slot = P.order[place];
    const T *x = FIRST ? reinterpret_cast<const T *>(P.x) + (long long)(slot / P.k) * P.ldx : reinterpret_cast<const T *>(P.h) + (long long)place * P.ff;
    const T *a[N];
#pragma unroll
    for (int r = 0; r < N; r++) {
        const T *W = reinterpret_cast<const T *>(!FIRST ? P.down : r < R ? P.gate : P.up);
        a[r] = W + ((long long)e * rows + min(row0 + r % R * 16 + c, rows - 1)) * K;
    }
    f32x4 acc[N] = {};
#pragma unroll 4
    for (int k = w * 32; k < K; k += 128) {
        const Frag<T> b = load_run<VEC>(x, k + g * 8, K);
#pragma unroll
        for (int r = 0; r < N; r++) acc[r] = mma(load_run<VEC>(a[r], k + g * 8, K), b, acc[r]);
    }
#pragma unroll
    for (int r = 0; r < N; r++) red[w][r][lane] = acc[r];
    __syncthreads();
    if (c >= count) return;
    for (int r = w; r < R; r += 4) {
        f32x4 v[M];
#pragma unroll
        for (int i = 0; i < M; i++) v[i] = (red[0][r + i * R][lane] + red[1][r + i * R][lane]) + (red[2][r + i * R][lane] + red[3][r + i * R][lane]);
        const int row = row0 + r * 16 + 4 * g;
        if constexpr (FIRST) put_rows(reinterpret_cast<T *>(P.h) + (long long)place * P.ff, row, P.ff, P.act == NL_ACT_SILU ? activate<true>(v[0], v[1]) : activate<false>(v[0], v[1]));
        else put_rows(P.part + (long long)slot * P.dim, row, P.dim, v[0] * P.weights[slot]);
    }
}

// ---------------------------------------------------------------- close ---

// block's result of token t, columns k ..
template <typename T> __device__ __forceinline__ float close_value(const CloseParams &P, int t, int k) {
    if (P.d) return (float)reinterpret_cast<const T *>(P.d)[(long long)t * P.ldd + k];
    float v = P.base ? P.base[(long long)t * P.ldbase + k] : 0.f;
    if (P.part)
        for (int j = 0; j < P.k; j++) {
            const long long s = (long long)t * P.k + j;
            const int id = P.ids[s];
            if (id >= 0 && id < P.experts) v += P.part[s * P.dim + k];
        }
    return v;
}
// a workgroup per token
template <typename T>
__global__ void __launch_bounds__(256) close_kernel(CloseParams P) {
    __shared__ float red[2][4];
    const int t = blockIdx.x, tid = threadIdx.x;
    if (!P.x_out) {
        for (int k = tid; k < P.dim; k += 256) put(reinterpret_cast<T *>(P.y) + (long long)t * P.ldy + k, close_value<T>(P, t, k));
        return;
    }
    auto total = [&](float v, int i) {
        v = wave_sum(v);
        if ((tid & 63) == 0) red[i][tid >> 6] = v;
        __syncthreads();
        return (red[i][0] + red[i][1]) + (red[i][2] + red[i][3]);
    };
    float inv = 1.f, ss = 0.f;
    if (P.post) {
        for (int k = tid; k < P.dim; k += 256) {
            const float v = close_value<T>(P, t, k);
            ss += v * v;
        }
        inv = rsqrt_f32(total(ss, 0) / (float)P.dim + P.eps);
        ss = 0.f;
    }
    const float *x = P.x + (long long)t * P.ldx;
    float *xo = P.x_out + (long long)t * P.ldxo;
    for (int k = tid; k < P.dim; k += 256) {
        float v = close_value<T>(P, t, k);
        if (P.post) v = v * inv * P.post[k];
        if (P.gate) v *= P.gate[(long long)t * P.ldgate + k];
        v = fmaf(P.scale, v, P.add ? x[k] + P.add[(long long)t * P.ldadd + k] : x[k]);
        xo[k] = v;
        ss += v * v;
    }
    if (!P.h) return;
    inv = rsqrt_f32(total(ss, 1) / (float)P.dim + P.eps);
    T *h = reinterpret_cast<T *>(P.h) + (long long)t * P.ldh;
    for (int k = tid; k < P.dim; k += 256) put(h + k, xo[k] * inv * P.pre[k]);
}

}  // namespace nl
