// nl_experts.h -- kernels of the feed-forward of experts (include/nanollama_ops.h): choice of experts, grouping of tokens by expert, the
// experts' products, the close of a block.  Matrices and rows are plain row-major here, a product's operands are gathered as fragments
// (nl_frag.h) from where they lie: a token's row through its slot, an expert's matrix as the caller has it.
//
//   slot   t * k + j: the j-th choice of token t            place   its position among all slots ordered by (expert, slot)
#pragma once
#include "nl_frag.h"
#include "nl_ops.h"

#include <type_traits>

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
// With a bias the keys sigmoid(l) + b are 32-bit numbers within key_err(b) of the exact ones: where two neighbours among the chosen ones, or the last of them and
// anyone left, are not apart by what both may be off, the keys that matter are computed again in 64 bits.  Every expert counts with its own error: a few that
// a large negative bias keeps out do not make the others near (8191 tokens to 8 of 256 with four biases of -1e9: 11 us; 29 with the largest error for all).
// Bound by its instructions, about 500 vector ones a token: 8191 tokens to 8 of 256 11.5 us (reading the logits alone 2); 18 where the second look, which one
// token in 200 needs, went over all experts; 19 where the largest was looked for k times instead of the border once.  To 8 of 64, 384, 512 and 1024 7.4, 17,
// 18 and 47, to 32 of 1024 58 (beyond 256 experts registers leave six wavefronts a SIMD, beyond 512 two).  One token 2.5 us, 64 to 6 of 96 4.5.
// sigmoid_f32 is within 3e-7, the sum within half a step; past 2^24, where a sigmoid is lost in the sum, within 1 (a number that rounds to itself there)
__device__ __forceinline__ float key_err(float b) { return fminf(1e-6f * (1.f + fabsf(b)), 2.f); }
template <int NE>
__global__ void __launch_bounds__(256) route_kernel(RouteParams P) {
    __shared__ __align__(16) f32x4 chosen[4][64];      // of a token: key, number, logit, bias
    const int wave = threadIdx.x >> 6, t = blockIdx.x * 4 + wave, lane = threadIdx.x & 63;
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
#pragma unroll
    for (int i = 0; i < NE; i++) {
        const float v = P.bias ? sigmoid_f32(l[i]) + b[i] : l[i];
        key[i] = out[i] ? 0 : order_u32(v);
    }
    int pick = -1;                                       // lane j: the j-th choice
    float score = 0.f;                                   // ... its logit
    {
        // the border: the largest key that at least as many as are wanted reach, bit by bit until exactly as many do
        int there = 0;
#pragma unroll
        for (int i = 0; i < NE; i++) there += __popcll(__ballot(key[i] != 0));
        const int want = min(P.k, there);
        unsigned border = 0;
        int reach = there;
        for (unsigned bit = 0x80000000u; bit && reach != want; bit >>= 1) {
            const unsigned next = border | bit;
            int c = 0;
#pragma unroll
            for (int i = 0; i < NE; i++) c += __popcll(__ballot(key[i] >= next));
            if (c >= want) { border = next; reach = c; }
        }
        border = max(border, 1u);                        // (0 is out)
        int spare = reach - want;                        // that many of the keys at the border stay out: the last ones
        unsigned long long in[NE];
#pragma unroll
        for (int i = NE - 1; i >= 0; i--) {
            in[i] = __ballot(key[i] >= border);
            if (spare > 0) {
                unsigned long long even = __ballot(key[i] == border);
                for (; spare > 0 && even; spare--) {
                    const int top = 63 - __clzll((long long)even);
                    even ^= 1ull << top;
                    in[i] ^= 1ull << top;
                }
            }
        }
        // one behind the other by number, then by rank
        int at = 0;
        float left = -INFINITY;                          // (with a bias) the most that a key left may be
#pragma unroll
        for (int i = 0; i < NE; i++) {
            if (in[i] >> lane & 1) chosen[wave][at + __popcll(in[i] & ((1ull << lane) - 1))] = f32x4{__uint_as_float(key[i]), __int_as_float(lane + 64 * i), l[i], b[i]};
            else if (P.bias && key[i]) left = fmaxf(left, order_f32(key[i]) + key_err(b[i]));
            at += __popcll(in[i]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // (one wavefront's: no barrier)
        const f32x4 mine = chosen[wave][lane];
        const unsigned k = __float_as_uint(mine[0]);
        int rank = 0;
        for (int j = 0; j < want; j++) {
            const unsigned o = (unsigned)__builtin_amdgcn_readlane((int)k, j);
            rank += o > k || (o == k && j < lane);
        }
        asm volatile("" ::: "memory");
        if (lane < want) chosen[wave][rank] = mine;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const f32x4 sorted = chosen[wave][lane];
        if (lane < want) { pick = __float_as_int(sorted[1]); score = sorted[2]; }
        bool near = false;
        float last = 0.f;
        if (P.bias) {
            const float v = order_f32(__float_as_uint(sorted[0])), err = key_err(sorted[3]), next = __shfl_down(v + err, 1);
            left = order_f32(wave_umax(order_u32(left)));
            if (lane < want) near = !(v - err > (lane + 1 < want ? next : left));
            if (lane + 1 == want && left == -INFINITY) near = false;
            near = __ballot(near) != 0;
            last = order_f32(~wave_umax(lane < want ? ~order_u32(v - err) : 0u));     // nothing that cannot reach it can be among the chosen ones
        }
        int few = 0;                                     // that many can
        if (near) {
#pragma unroll
            for (int i = 0; i < NE; i++) few += __popcll(__ballot(key[i] && order_f32(key[i]) + key_err(b[i]) >= last));
        }
        if (near && few <= 64) {                         // a key in 64 bits a lane, then by rank
            int to = 0;
#pragma unroll
            for (int i = 0; i < NE; i++) {
                const bool can = key[i] && order_f32(key[i]) + key_err(b[i]) >= last;
                const unsigned long long cans = __ballot(can);
                if (can) chosen[wave][to + __popcll(cans & ((1ull << lane) - 1))] = f32x4{l[i], b[i], __int_as_float(lane + 64 * i), 0.f};
                to += __popcll(cans);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const f32x4 one = chosen[wave][lane];
            const double k64 = 1.0 / (1.0 + exp(-(double)one[0])) + (double)one[1];
            const unsigned long long bits = __builtin_bit_cast(unsigned long long, k64);
            int place = 0;
            for (int j = 0; j < few; j++) {
                const unsigned long long hi = (unsigned)__builtin_amdgcn_readlane((int)(bits >> 32), j), lo = (unsigned)__builtin_amdgcn_readlane((int)bits, j);
                const double o = __builtin_bit_cast(double, hi << 32 | lo);
                place += o > k64 || (o == k64 && j < lane);
            }
            asm volatile("" ::: "memory");
            if (lane < few && place < want) chosen[wave][place] = one;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            const f32x4 at_last = chosen[wave][lane];
            if (lane < want) { pick = __float_as_int(at_last[2]); score = at_last[0]; }
        } else if (near) {                               // (many alike: expert by expert)
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
// 384 slots of 64 experts 4.8 us; 65528 slots of 64, 256 and 1024 experts 14, 14 and 32; 524168 of 64 and 1024 96 and 212: it grows with their product.
__global__ void __launch_bounds__(1024) plan_kernel(const int *ids, int nslots, int experts, int *offs, int *order) {
    __shared__ int less[16], mine[16];
    const int e = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int per = ((nslots + 15) / 16 + 63) & ~63, lo = min(w * per, nslots), hi = min(lo + per, nslots);      // this wavefront's slots
    int nl = 0, nm = 0;
#pragma unroll 8
    for (int s = lo + lane; s < hi; s += 64) {           // (a lane counts for itself: its loads do not wait for one another)
        const int id = ids[s];
        nl += id >= 0 && id < e;
        nm += id == e;
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) { nl += __shfl_xor(nl, s); nm += __shfl_xor(nm, s); }
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
    constexpr int U = 8;
    for (int s = lo; s < hi; s += 64 * U) {
        int id[U];
#pragma unroll
        for (int i = 0; i < U; i++) id[i] = s + i * 64 + lane < hi ? ids[s + i * 64 + lane] : -1;
#pragma unroll
        for (int i = 0; i < U; i++) {
            const unsigned long long m = __ballot(id[i] == e);
            if (id[i] == e) order[at + __popcll(m & ((1ull << lane) - 1))] = s + i * 64 + lane;
            at += __popcll(m);
        }
    }
}

// The experts' places cut into tiles of BT, an expert's tiles one behind the other: which expert has tile `tile`, how many tiles are in front of
// its first one, its places [a, b).  Every wavefront finds it by itself: a lane counts the tiles of a run of experts, a scan finds the lane.
struct Group { int e, before, a, b; };
template <int BT>
struct Groups {
    int per, lo, hi, mine, upto;
    const int *offs;
    __device__ __forceinline__ Groups(const int *o, int experts) : offs(o) {
        const int lane = threadIdx.x & 63, e0 = lane * (per = (experts + 63) >> 6);
        mine = 0;
        hi = lo = offs[min(e0, experts)];
        for (int i = 0; i < per; i++) {
            const int b = offs[min(e0 + i + 1, experts)];
            mine += (b - hi + BT - 1) / BT;
            hi = b;
        }
        upto = mine;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int o2 = __shfl_up(upto, s);
            if (lane >= s) upto += o2;
        }
    }
    __device__ __forceinline__ int total() const { return __builtin_amdgcn_readlane(upto, 63); }
    __device__ __forceinline__ Group find(int tile) const {          // tile < total()
        const int at = __ffsll((long long)__ballot(upto > tile)) - 1;
        Group G;
        G.before = __builtin_amdgcn_readlane(upto - mine, at);
        G.e = at * per;
        G.a = __builtin_amdgcn_readlane(lo, at);
        if (per == 1) {
            G.b = __builtin_amdgcn_readlane(hi, at);
            return G;
        }
        for (;;) {
            G.b = __builtin_amdgcn_readfirstlane(offs[G.e + 1]);
            const int n = (G.b - G.a + BT - 1) / BT;
            if (tile - G.before < n) return G;
            G.before += n;
            G.a = G.b;
            G.e++;
        }
    }
};

// ------------------------------------------------------------- products ---

// a lane's run of 8 elements from k0 on of a row of K, zero behind its end
template <typename T> __device__ __forceinline__ Frag<T> load_run(const T *row, int k0, int K) {
    Frag<T> f;
    frag_zero(f);
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (k0 + j < K) frag_set(f, j, (float)row[k0 + j]);
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

// Rows that do not even start on 4-byte boundaries (bfloat16): 16 places x 32 rows of one expert by a workgroup, K dealt to its four wavefronts, elements one
// by one straight to registers.  FIRST: gate and up rows of the tokens -> h; else rows of down of h -> part (32-bit: a third rounding to bfloat16, beside
// the activation's and the sum's, would make the error 1.2 times as large: 2.9e-3 instead of 2.4e-3).
template <typename T, bool FIRST>
__global__ void __launch_bounds__(256) experts_any_kernel(ExpertsParams P) {
    constexpr int R = 2, M = FIRST ? 2 : 1, N = R * M;
    __shared__ __align__(16) f32x4 red[4][N][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int rows = FIRST ? P.ff : P.dim, K = FIRST ? P.dim : P.ff, row0 = blockIdx.x * 16 * R;
    const Groups<16> groups(P.offs, P.experts);
    for (int tile = blockIdx.y; tile < groups.total(); tile += gridDim.y) {
        const Group G = groups.find(tile);
        const int e = G.e, first = G.a + (tile - G.before) * 16, count = min(16, G.b - first);
        const int place = first + min(c, count - 1), slot = P.order[place];
        const T *x = FIRST ? reinterpret_cast<const T *>(P.x) + (long long)(slot / P.k) * P.ldx : reinterpret_cast<const T *>(P.h) + (long long)place * P.ff;
        const T *a[N];
#pragma unroll
        for (int r = 0; r < N; r++) {
            const T *W = reinterpret_cast<const T *>(!FIRST ? P.down : r < R ? P.gate : P.up);
            a[r] = W + ((long long)e * rows + min(row0 + r % R * 16 + c, rows - 1)) * K;
        }
        f32x4 acc[N] = {};
        for (int k = w * 32; k < K; k += 128) {
            const Frag<T> b = load_run(x, k + g * 8, K);
#pragma unroll
            for (int r = 0; r < N; r++) acc[r] = mma(load_run(a[r], k + g * 8, K), b, acc[r]);
        }
        __syncthreads();                                 // (the tile before is read)
#pragma unroll
        for (int r = 0; r < N; r++) red[w][r][lane] = acc[r];
        __syncthreads();
        if (w >= R || c >= count) continue;
        f32x4 v[M];
#pragma unroll
        for (int i = 0; i < M; i++) v[i] = (red[0][w + i * R][lane] + red[1][w + i * R][lane]) + (red[2][w + i * R][lane] + red[3][w + i * R][lane]);
        const int row = row0 + w * 16 + 4 * g;
        if constexpr (FIRST) put_rows(reinterpret_cast<T *>(P.h) + (long long)place * P.ff, row, P.ff, P.act == NL_ACT_SILU ? activate<true>(v[0], v[1]) : activate<false>(v[0], v[1]));
        else put_rows(P.part + (long long)slot * P.dim, row, P.dim, v[0] * P.weights[slot]);
    }
}

// V consecutive elements as floats
template <int V> __device__ __forceinline__ void load_vec(const float *p, float *v) {
    if constexpr (V == 4) *reinterpret_cast<f32x4 *>(v) = *reinterpret_cast<const f32x4 *>(p);
    else v[0] = *p;
}
template <int V> __device__ __forceinline__ void load_vec(const bf16 *p, float *v) {
    if constexpr (V == 4) {
        const bf16x4 b = *reinterpret_cast<const bf16x4 *>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (float)b[i];
    } else v[0] = (float)*p;
}

// A few tokens: no grouping, no matrix instructions; a row of a matrix is read by a whole wavefront in 16-byte pieces, one row for every slot that
// asks for it.  First the activations of slot blockIdx.y (h is by slot here, and 32-bit: no matrix instruction wants them rounded, and rounded ones make the
// error 1.4 times as large, by chance 1.6 times for a single token), then rows of the sum over token blockIdx.y's slots: a lane keeps its share of all of
// them, one sum over the wavefront at the end.
template <typename T> struct Piece { static constexpr int N = 16 / (int)sizeof(T); T v[N]; };
template <typename T> __device__ __forceinline__ Piece<T> load_piece(const T *p) {
    Piece<T> r;
    *reinterpret_cast<f32x4 *>(r.v) = *reinterpret_cast<const f32x4 *>(p);
    return r;
}
template <typename T> __device__ __forceinline__ float dot_piece(const Piece<T> &a, const Piece<T> &b) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < Piece<T>::N; i++) s = fmaf((float)a.v[i], (float)b.v[i], s);
    return s;
}
// (what lies behind a row's end, or belongs to no expert, is read from the front of the row, or of expert 0, and left out: behind branches the compiler
// would wait for one load before it asks for the next.  One token to 8 of 64 experts of 768 x 512: 4.8 and 6.1 us that way, 4.8 and 3.9 so; to 2 of
// 8 of 4096 x 11008 58 and 41, 5.5 TB/s of what they read)
template <typename T>
__global__ void __launch_bounds__(256) experts_token_first_kernel(ExpertsParams P) {
    constexpr int N = Piece<T>::N, U = 4;
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6), slot = blockIdx.y, e = P.ids[slot];
    if (row >= P.ff || e < 0 || e >= P.experts) return;
    const T *x = reinterpret_cast<const T *>(P.x) + (long long)(slot / P.k) * P.ldx;
    const long long at = ((long long)e * P.ff + row) * P.dim;
    const T *a = reinterpret_cast<const T *>(P.gate) + at, *b = reinterpret_cast<const T *>(P.up) + at;
    float ga = 0.f, ub = 0.f;
    auto some = [&](int k0, auto count) {                // `count` pieces a lane from column k0 on
        constexpr int C = decltype(count)::value;
        Piece<T> xv[C], av[C], bv[C];
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int k = k0 + (i * 64 + lane) * N, kc = k < P.dim ? k : 0;
            av[i] = load_piece(a + kc);
            bv[i] = load_piece(b + kc);
            xv[i] = load_piece(x + kc);
        }
#pragma unroll
        for (int i = 0; i < C; i++) {
            const bool in = k0 + (i * 64 + lane) * N < P.dim;
            const float ai = dot_piece(av[i], xv[i]), bi = dot_piece(bv[i], xv[i]);
            ga += in ? ai : 0.f;
            ub += in ? bi : 0.f;
        }
    };
    int k0 = 0;
    for (; P.dim - k0 > 2 * 64 * N; k0 += U * 64 * N) some(k0, std::integral_constant<int, U>());
    if (P.dim - k0 > 64 * N) some(k0, std::integral_constant<int, 2>());
    else if (P.dim > k0) some(k0, std::integral_constant<int, 1>());
    ga = wave_sum(ga);
    ub = wave_sum(ub);
    if (lane == 0) reinterpret_cast<float *>(P.h)[(long long)slot * P.ff + row] = ga * sigmoid_f32(P.act == NL_ACT_SILU ? ga : gelu_arg(ga)) * ub;
}
template <typename T>
__global__ void __launch_bounds__(256) experts_token_second_kernel(ExpertsParams P) {
    constexpr int N = Piece<T>::N;
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6), t = blockIdx.y;
    if (row >= P.dim) return;
    const int slot = t * P.k + min(lane, P.k - 1), id = P.ids[slot];
    const float weight = P.weights[slot];
    float sum = 0.f;
    auto some = [&](int j0, int k, auto count) {         // `count` slots from the j0-th on, a piece each
        constexpr int C = decltype(count)::value;
        const int kc = k < P.ff ? k : 0;
        Piece<T> dv[C];
        float hv[C][N];
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int j = min(j0 + i, P.k - 1), e = __builtin_amdgcn_readlane(id, j), ec = e >= 0 && e < P.experts ? e : 0;
            dv[i] = load_piece(reinterpret_cast<const T *>(P.down) + ((long long)ec * P.dim + row) * P.ff + kc);
#pragma unroll
            for (int p = 0; p < N; p += 4) load_vec<4>(reinterpret_cast<const float *>(P.h) + (long long)(t * P.k + j) * P.ff + kc + p, hv[i] + p);
        }
#pragma unroll
        for (int i = 0; i < C; i++) {
            const int j = min(j0 + i, P.k - 1), e = __builtin_amdgcn_readlane(id, j);
            const bool in = j0 + i < P.k && e >= 0 && e < P.experts && k < P.ff;
            float v = 0.f;
#pragma unroll
            for (int p = 0; p < N; p++) v = fmaf((float)dv[i].v[p], hv[i][p], v);
            v *= lane_value(weight, j);
            sum += in ? v : 0.f;
        }
    };
    for (int k = lane * N; k - lane * N < P.ff; k += 64 * N) {
        int j = 0;
        for (; P.k - j > 4; j += 8) some(j, k, std::integral_constant<int, 8>());
        if (P.k - j > 2) some(j, k, std::integral_constant<int, 4>());
        else if (P.k > j) some(j, k, std::integral_constant<int, 2>());
    }
    sum = wave_sum(sum);
    if (lane != 0) return;
    if (P.y) put(reinterpret_cast<T *>(P.y) + (long long)t * P.ldy + row, sum);
    else if (P.res_out) {
        float x = P.res[(long long)t * P.ldres + row];
        if (P.add) x += P.add[(long long)t * P.ldadd + row];
        P.res_out[(long long)t * P.ldo + row] = fmaf(P.scale, sum, x);
    } else P.part[(long long)t * P.dim + row] = sum;
}

// Prompts: WR x WT wavefronts of RTW row tiles x NTW token tiles each; 128 bytes of every row at a time go through a ring of two or three LDS stages by
// LDS-DMA, a piece of 8 rows (UNIT 16 bytes a lane), whole lines of the rows as they lie, or of 2 (UNIT 4, for rows that start on 4-byte boundaries only).  In
// LDS the 16-byte run q of row r is at q ^ (r % 8), so that the 16 rows of a fragment are read from all banks.  FIRST: row tiles alternate between gate and up.
// Bound by bringing the stages: 2047 tokens to 8 of 64 of 1536 x 768, 128 x 128, gate and up 132 us, where LDS is not read 125, without the DMA 78; 993 to 2 of 8
// of 4096 x 11008, 256 x 256, 503, 498 and 383.  L2 sends 43 KB/us a CU in the first (1.36 GB) and 28 in the second; a line is on its way for 460 to 590 cycles,
// 55 to 75 of them at a time, L1 waits for data in 41 to 60 % of its cycles and the matrix units are busy in 26 to 46 % of theirs; LDS banks never conflict.
// Workgroups b, b + 8, ... run on one XCD and take a contiguous range of (expert, row block, token tile): both operands of neighbours are in its L2.
template <typename T, int RTW_, int NTW_, int WR_, int WT_, int NST_ = 2, int UNIT_ = 16, bool PAIR_ = false> struct Grouped {
    static constexpr bool PAIR = PAIR_;
    static constexpr int NST = NST_, UNIT = UNIT_, PIECE = 64 * UNIT, RTW = RTW_, NTW = NTW_, WR = WR_, WT = WT_, RT = WR * RTW, NT = WT * NTW, STAGE = (RT + (PAIR ? 2 : 1) * NT) * 2048, LDS = NST * STAGE, NW = WR * WT, THREADS = 64 * NW,
                         PW = STAGE / PIECE / NW, BT = NT * 16, KB = 128 / (int)sizeof(T), KK = KB / 32, PER_CU = 163840 / LDS;
    static_assert(PW * NW * PIECE == STAGE && NW * PIECE % 1024 == 0 && PW * (NST - 1) < 64, "pieces");
};
__device__ const f32x4 zero_piece = {0.f, 0.f, 0.f, 0.f};
template <typename T> __device__ __forceinline__ Frag<T> swizzled_frag(const char *tile, int r, int g, int kk);
template <> __device__ __forceinline__ Frag<bf16> swizzled_frag<bf16>(const char *tile, int r, int g, int kk) {
    Frag<bf16> f;
    f.v = *reinterpret_cast<const bf16x8 *>(tile + r * 128 + (((kk * 4 + g) ^ (r & 7)) << 4));
    return f;
}
template <> __device__ __forceinline__ Frag<float> swizzled_frag<float>(const char *tile, int r, int g, int) {
    Frag<float> f;
    f.a = *reinterpret_cast<const f32x4 *>(tile + r * 128 + (((2 * g) ^ (r & 7)) << 4));
    f.b = *reinterpret_cast<const f32x4 *>(tile + r * 128 + (((2 * g + 1) ^ (r & 7)) << 4));
    return f;
}
template <typename T, bool FIRST, typename S>
__global__ void __launch_bounds__(S::THREADS, S::NW * S::PER_CU / 4) experts_many_kernel(ExpertsParams P) {
    constexpr int RT = S::RT, NST = S::NST, UNIT = S::UNIT, PIECE = S::PIECE, STAGE = S::STAGE, NW = S::NW, PW = S::PW, BT = S::BT, KB = S::KB, KK = S::KK, RTW = S::RTW, NTW = S::NTW;
    constexpr int BR = (FIRST ? RT / 2 : RT) * 16;        // output rows of the workgroup
    static_assert(!FIRST || !S::PAIR, "pairs are the activations'");
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15, wr = w % S::WR, wt = w / S::WR;
    const int rows = FIRST ? P.ff : P.dim, K = FIRST ? P.dim : P.ff, nrb = (rows + BR - 1) / BR, nks = (K + KB - 1) / KB;
    const Groups<BT> groups(P.offs, P.experts);
    const int all = groups.total() * nrb, per = (all + 7) >> 3, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= all) return;
    const Group G = groups.find(id / nrb);
    const int tiles = (G.b - G.a + BT - 1) / BT, local = id - G.before * nrb, rb = local / tiles, first = G.a + (local - rb * tiles) * BT, count = min(BT, G.b - first);
    // (XCDs start at different columns, and four row blocks in turn: 2047 tokens to 8 of 64 of 1536 x 768 126 / 85 us; all at the first one 126 / 87, every row
    // block at its own 128 / 87, every token tile too 144 / 90; down of 4096 x 11008 374, 386, 448, 528)
    const int turn = ((blockIdx.x & 7) * nks / 8 + (rb & 3)) % nks;
    const char *src[PW];
    constexpr int LR = 128 / UNIT, PR = PIECE / 128, PA = RT * 16 / PR / NW;         // lanes of a row, rows of a piece, a wavefront's pieces of the matrix
    static_assert(PA * NW * PR == RT * 16, "pieces of the matrix");
    const int run = lane % LR * UNIT / 16 ^ (w * PR + lane / LR) % 8, k0 = (run * 16 + lane % LR * UNIT % 16) / (int)sizeof(T);      // (a wavefront's pieces are whole eights of rows apart)
    int there = NST == 2 && !S::PAIR ? PA : PW;          // pieces with a token or a row of the matrix: the first ones (all, where waits count them)
    int token[PW - PA];                                  // (asked for now, needed behind the matrix's first pieces)
#pragma unroll
    for (int i = PA; i < PW; i++) {
        const int at = (i * NW + w) * PR - RT * 16;      // PAIR: the tokens' activations, then what is left of them
        if (NST == 2 && !S::PAIR && at < count) there = i + 1;
        const int place = first + min((S::PAIR ? at % (S::NT * 16) : at) + lane / LR, count - 1);
        token[i - PA] = FIRST ? P.order[place] : place;
    }
#pragma unroll
    for (int i = 0; i < PA; i++) {
        const int r = (i * NW + w) * PR + lane / LR, t = r >> 4;                      // row of the stage, its tile
        const T *W = reinterpret_cast<const T *>(!FIRST ? P.down : t & 1 ? P.up : P.gate);
        src[i] = reinterpret_cast<const char *>(W + ((long long)G.e * rows + min(rb * BR + (FIRST ? t >> 1 : t) * 16 + (r & 15), rows - 1)) * K + k0);
    }
    auto bring = [&](const void *from, int st, int i) {
        if constexpr (UNIT == 16) lds_dma16(from, lds + st * STAGE + (i * NW + w) * PIECE);
        else lds_dma4(from, lds + st * STAGE + (i * NW + w) * PIECE);
    };
    auto issue = [&](int ks, int st, auto from, auto to) {
        constexpr int I0 = decltype(from)::value, I1 = decltype(to)::value;
        if ((ks += turn) >= nks) ks -= nks;
        if ((ks + 1) * KB <= K) {
#pragma unroll
            for (int i = I0; i < I1; i++)
                if (i < PA || i < there) bring(src[i] + (long long)ks * 128, st, i);
        } else {                                         // (behind the row's end: zeros)
            const unsigned long long in = ks * KB + k0 < K ? ~0ull : 0, zero = reinterpret_cast<unsigned long long>(&zero_piece) & ~in;
#pragma unroll
            for (int i = I0; i < I1; i++)
                if (i < PA || i < there) bring(reinterpret_cast<const char *>((reinterpret_cast<unsigned long long>(src[i] + (long long)ks * 128) & in) | zero), st, i);
        }
    };
    using None = std::integral_constant<int, 0>;
    using Some = std::integral_constant<int, PA>;
    using Whole = std::integral_constant<int, PW>;
    issue(0, 0, None(), Some());
#pragma unroll
    for (int i = PA; i < PW; i++)
        src[i] = reinterpret_cast<const char *>((FIRST ? reinterpret_cast<const T *>(P.x) + (long long)(token[i - PA] / P.k) * P.ldx
                                                       : reinterpret_cast<const T *>(S::PAIR && (i * NW + w) * PR >= (RT + S::NT) * 16 ? P.h_rest : P.h) + (long long)token[i - PA] * P.ff) + k0);
    f32x4 acc[RTW][NTW] = {};
    constexpr int NF = S::PAIR ? 2 * NTW : NTW;
    Frag<T> fa[KK][RTW], fb[KK][NF];
    const bool busy = wt * NTW * 16 < count;             // (wavefronts without a token only bring pieces)
    auto read = [&](int st, int kk, Frag<T> *a, Frag<T> *b) {
        const char *base = lds + st * STAGE;
#pragma unroll
        for (int t = 0; t < NF; t++) b[t] = swizzled_frag<T>(base + (RT + wt * NTW + (t < NTW ? t : S::NT + t - NTW)) * 2048, c, g, kk);
#pragma unroll
        for (int r = 0; r < RTW; r++) a[r] = swizzled_frag<T>(base + (wr * RTW + r) * 2048, c, g, kk);
    };
    auto multiply = [&](const Frag<T> *a, const Frag<T> *b) {
#pragma unroll
        for (int t = 0; t < NTW; t++) {
            if (sizeof(T) == 4 && (wt * NTW + t) * 16 >= count) break;       // (32 bits: the matrix rate bounds it; for 16 the branches cost more)
#pragma unroll
            for (int r = 0; r < RTW; r++)                // (32 bits: a stage's 32 products by themselves, then into the sum: one chain over the row is off by twice as much)
                if constexpr (sizeof(T) == 4) acc[r][t] += mma(a[r], b[t], f32x4{});
                else {
                    acc[r][t] = mma(a[r], b[t], acc[r][t]);
                    if constexpr (S::PAIR) acc[r][t] = mma(a[r], b[NTW + t], acc[r][t]);
                }
        }
    };
    // (builtins, not lds_barrier(): the compiler has to know that nothing is on its way from LDS, or it waits for the next fragments before it
    // multiplies the present ones)
    auto arrived = [&]() { __builtin_amdgcn_s_waitcnt(0xc07f); };
    int st = 0;
    auto next_stage = [&](int s) {                       // to stage s < nks; the one before it is read and filled again
        if (NST > 2 && nks - 1 - s >= NST - 2) vm_wait<PW *(NST - 2)>();
        else vm_wait<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s - 1 + NST < nks) issue(s - 1 + NST, st, None(), Whole());
        st = st + 1 == NST ? 0 : st + 1;
    };
    issue(0, 0, Some(), Whole());
#pragma unroll
    for (int s = 1; s < NST; s++)
        if (s < nks) issue(s, s, None(), Whole());
    if (nks >= NST && there == PW) vm_wait<PW *(NST - 1)>();
    else vm_wait<0>();
    lds_barrier();
    if (!busy) {
        for (int s = 1; s < nks; s++) next_stage(s);
        return;
    }
    // 32 columns a step; a step's fragments are read while the step before it is multiplied.  Once every wavefront has read the last of a
    // stage (the barrier), the stage is filled again.
    read(0, 0, fa[0], fb[0]);
    for (int s = 0; s + 1 < nks; s++) {
        arrived();
        if constexpr (KK == 2) {
            read(st, 1, fa[1], fb[1]);
            __builtin_amdgcn_sched_barrier(0);
            multiply(fa[0], fb[0]);
            __builtin_amdgcn_sched_barrier(0);
            arrived();
        }
        next_stage(s + 1);
        if constexpr (KK == 2) {
            read(st, 0, fa[0], fb[0]);
            __builtin_amdgcn_sched_barrier(0);
            multiply(fa[1], fb[1]);
        } else {
            multiply(fa[0], fb[0]);
            read(st, 0, fa[0], fb[0]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (KK == 2) read(st, 1, fa[1], fb[1]);
    multiply(fa[0], fb[0]);
    if constexpr (KK == 2) multiply(fa[1], fb[1]);
#pragma unroll
    for (int t = 0; t < NTW; t++) {
        const int at = (wt * NTW + t) * 16 + c, place = first + at;
        if (at >= count) continue;
        if constexpr (FIRST) {
            T *h = reinterpret_cast<T *>(P.h) + (long long)place * P.ff;
#pragma unroll
            for (int r = 0; r < RTW; r += 2) {
                const f32x4 v = P.act == NL_ACT_SILU ? activate<true>(acc[r][t], acc[r + 1][t]) : activate<false>(acc[r][t], acc[r + 1][t]);
                put_rows(h, rb * BR + (wr * RTW + r) * 8 + 4 * g, P.ff, v);
                if (sizeof(T) == 2 && P.h_rest) {        // (not finite: nothing is left)
                    f32x4 rest;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float d = v[i] - (float)(T)v[i];
                        rest[i] = d - d == 0.f ? d : 0.f;
                    }
                    put_rows(reinterpret_cast<T *>(P.h_rest) + (long long)place * P.ff, rb * BR + (wr * RTW + r) * 8 + 4 * g, P.ff, rest);
                }
            }
        } else {
            const int slot = P.order[place];
            float *o = P.part + (long long)slot * P.dim;
            const float wgt = P.weights[slot];
#pragma unroll
            for (int r = 0; r < RTW; r++) put_rows(o, rb * BR + (wr * RTW + r) * 16 + 4 * g, P.dim, acc[r][t] * wgt);
        }
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
            const int id = P.ids ? P.ids[s] : 0;
            if (id >= 0 && id < P.experts) v += P.part[s * P.dim + k];
        }
    return v;
}
template <int V, typename T> __device__ __forceinline__ void store_vec(T *p, const float *v) {
    if constexpr (V == 4) put4(p, *reinterpret_cast<const f32x4 *>(v));
    else put(p, v[0]);
}
// A workgroup per token, the row in registers: C runs of V elements a thread, read once; everything that the norms do not decide is on its way before
// the first of them.
template <typename T, int V, int C>
__global__ void __launch_bounds__(256) close_rows_kernel(CloseParams P) {
    __shared__ float red[2][4];
    const int t = blockIdx.x, tid = threadIdx.x;
    float v[C][V], x[C][V], g[C][V], p[C][V];
    auto at = [&](int c) { return (c * 256 + tid) * V; };
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < V; i++) { v[c][i] = 0.f; x[c][i] = 0.f; g[c][i] = 1.f; p[c][i] = 0.f; }
    auto total = [&](int i) {
        float s = 0.f;
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int j = 0; j < V; j++) s = fmaf(v[c][j], v[c][j], s);
        s = wave_sum(s);
        if ((tid & 63) == 0) red[i][tid >> 6] = s;
        __syncthreads();
        return (red[i][0] + red[i][1]) + (red[i][2] + red[i][3]);
    };
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int k = at(c);
        if (k >= P.dim) break;
        if (P.d) load_vec<V>(reinterpret_cast<const T *>(P.d) + (long long)t * P.ldd + k, v[c]);
        else if (P.base) load_vec<V>(P.base + (long long)t * P.ldbase + k, v[c]);
        if (P.x_out) {
            load_vec<V>(P.x + (long long)t * P.ldx + k, x[c]);
            if (P.add) {
                float o[V];
                load_vec<V>(P.add + (long long)t * P.ldadd + k, o);
#pragma unroll
                for (int i = 0; i < V; i++) x[c][i] += o[i];
            }
            if (P.gate) load_vec<V>(P.gate + (long long)t * P.ldgate + k, g[c]);
            if (P.post) {
                float o[V];
                load_vec<V>(P.post + k, o);
#pragma unroll
                for (int i = 0; i < V; i++) g[c][i] *= o[i];
            }
            if (P.h) load_vec<V>(P.pre + k, p[c]);
        }
    }
    if (P.part) {
#pragma unroll 4
        for (int j = 0; j < P.k; j++) {                  // (results of slots without an expert are read and left out: the workspace has room for them)
            const long long s = (long long)t * P.k + j;
            const int id = P.ids ? P.ids[s] : 0;
            const bool in = id >= 0 && id < P.experts;
#pragma unroll
            for (int c = 0; c < C; c++) {
                if (at(c) >= P.dim) break;
                float o[V];
                load_vec<V>(P.part + s * P.dim + at(c), o);
#pragma unroll
                for (int i = 0; i < V; i++) v[c][i] += in ? o[i] : 0.f;
            }
        }
    }
    if (!P.x_out) {
#pragma unroll
        for (int c = 0; c < C; c++)
            if (at(c) < P.dim) store_vec<V>(reinterpret_cast<T *>(P.y) + (long long)t * P.ldy + at(c), v[c]);
        return;
    }
    const float inv = P.scale * (P.post ? rsqrt_f32(total(0) / (float)P.dim + P.eps) : 1.f);
#pragma unroll
    for (int c = 0; c < C; c++) {
        if (at(c) >= P.dim) break;
#pragma unroll
        for (int i = 0; i < V; i++) v[c][i] = fmaf(inv * v[c][i], g[c][i], x[c][i]);
        store_vec<V>(P.x_out + (long long)t * P.ldxo + at(c), v[c]);
    }
    if (!P.h) return;
    const float ih = rsqrt_f32(total(1) / (float)P.dim + P.eps);
#pragma unroll
    for (int c = 0; c < C; c++) {
        if (at(c) >= P.dim) break;
#pragma unroll
        for (int i = 0; i < V; i++) v[c][i] *= ih * p[c][i];
        store_vec<V>(reinterpret_cast<T *>(P.h) + (long long)t * P.ldh + at(c), v[c]);
    }
}
// rows of any length, which are read again for every step, an element a load: 2047 rows of 5120 107 us, of 11008 228 (1.2 TB/s)
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
