// nl_ops.hip -- host side of the operators on device memory (include/nanollama_ops.h): checks, launches, the rules by which a kernel is chosen.
#include "nl_experts.h"

#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <algorithm>
#include <atomic>
#include <tuple>

using namespace nl;

namespace {

template <typename... F, typename... A>
hipError_t start(void (*kernel)(F...), dim3 grid, dim3 block, size_t lds, hipStream_t st, A... args) {
    static_assert(sizeof...(F) == sizeof...(A), "kernel arguments");
    std::tuple<F...> held(args...);
    void *at[sizeof...(F)];
    std::apply([&](auto &...a) { int i = 0; ((at[i++] = (void *)&a), ...); }, held);
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, at, lds, st);
}

// the same with more dynamic LDS than a kernel has by itself, which is asked for once a device
template <auto *KERNEL, typename... A>
hipError_t start_lds(dim3 grid, dim3 block, size_t lds, hipStream_t st, A... args) {
    static std::atomic<unsigned long long> asked{0};
    int device = 0;
    hipError_t rc = hipGetDevice(&device);
    if (rc != hipSuccess) return rc;
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (!(asked.load(std::memory_order_relaxed) & bit)) {
        if ((rc = hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds)) != hipSuccess) return rc;
        asked.fetch_or(bit, std::memory_order_relaxed);
    }
    return start(KERNEL, grid, block, lds, st, args...);
}

inline bool on(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
template <typename T> inline T *behind(T *p, long long elements) { return p ? p + elements : p; }
inline const void *behind(const void *p, long long elements, size_t size) { return behind(reinterpret_cast<const char *>(p), elements * (long long)size); }
inline void *behind(void *p, long long elements, size_t size) { return behind(reinterpret_cast<char *>(p), elements * (long long)size); }

// A launch's threads are counted in 32 bits, silently: 2^24 rows at a workgroup of 256 each return without an error and leave nearly all of them unwritten.
// So many tokens go at once, others behind them.
constexpr int CLOSE_TOKENS = 1 << 23, ROUTE_TOKENS = 1 << 25;

}  // namespace

namespace nl {

static hipError_t route(const RouteParams &P, hipStream_t st) {
    const dim3 grid((P.n + 3) / 4), block(256);
    const int ne = (P.experts + 63) / 64;
    if (ne <= 1) return start(route_kernel<1>, grid, block, 0, st, P);
    if (ne <= 2) return start(route_kernel<2>, grid, block, 0, st, P);
    if (ne <= 4) return start(route_kernel<4>, grid, block, 0, st, P);
    if (ne <= 8) return start(route_kernel<8>, grid, block, 0, st, P);
    return start(route_kernel<16>, grid, block, 0, st, P);
}
hipError_t launch_route(const RouteParams &P, hipStream_t st) {
    hipError_t rc = hipSuccess;
    for (long long t = 0; t < P.n && rc == hipSuccess; t += ROUTE_TOKENS) {
        RouteParams Q = P;
        Q.n = (int)std::min<long long>(P.n - t, ROUTE_TOKENS);
        Q.logits = behind(P.logits, t * P.ld); Q.ids = behind(P.ids, t * P.k); Q.weights = behind(P.weights, t * P.k);
        rc = route(Q, st);
    }
    return rc;
}

// Slot by slot where grouping hardly saves a matrix: one token, or half as many slots as experts.  us a pass slot by slot and grouped: 1, 2, 4 and 8 tokens to 8
// of 64 of 1536 x 768 15 and 29, 24 and 34, 41 and 53, 72 and 60; 1, 2 and 4 to 2 of 8 of 4096 x 11008 103 and 140, 212 and 207, 374 and 292.
inline size_t most_by_token(int k, int experts) { return std::max(k, experts / 2); }
// Up to so many tokens an expert on the average bfloat16 activations go on as pairs (what rounding leaves beside what it makes): the weights' way from memory hides
// the second product.  us of it without and with: 64 experts of 1536 x 768, 4 tokens each 25 and 27, 16 each 31 and 37; 6 each of 1536 x 1024 33 and 35; 8 of 4096 x
// 11008, 4 each 117 and 118, 16 each 139 and 171.  Error against 64 bits 2.35e-3 and 1.66e-3, which is the result's own rounding.
constexpr size_t PAIR_TOKENS = 8;
ExpertsLayout experts_layout(int n, int k, int experts, int dim, int ff, int dtype) {
    const size_t slots = (size_t)n * k, es = dtype == NL_DTYPE_F32 ? 4 : 2;
    auto up = [](size_t b) { return (b + 255) & ~(size_t)255; };
    ExpertsLayout L;
    L.offs = 0;
    L.order = up((size_t)(experts + 1) * 4);
    L.h = L.order + up(slots * 4);
    L.part = L.h + up(std::max(slots * es, std::min(slots, std::max(most_by_token(k, experts), PAIR_TOKENS * experts)) * 4) * ff);
    L.bytes = L.part + up(slots * dim * 4);
    return L;
}
void place_experts(ExpertsParams &P, void *workspace, const ExpertsLayout &L) {
    char *ws = reinterpret_cast<char *>(workspace);
    P.offs = reinterpret_cast<int *>(ws + L.offs);
    P.order = reinterpret_cast<int *>(ws + L.order);
    P.h = ws + L.h;
    P.part = reinterpret_cast<float *>(ws + L.part);
}

// One product of the experts with tiles of S.  The most workgroups that it can need: an expert's last tile may hold one token.
template <bool FIRST, typename S> static long long workgroups(const ExpertsParams &P) {
    const int slots = P.n * P.k, hit = std::min(P.experts, slots), rows = FIRST ? P.ff : P.dim, br = S::RT * (FIRST ? 8 : 16);
    return ((hit + (slots - hit) / S::BT) * (long long)((rows + br - 1) / br) + 7) / 8 * 8;
}
template <typename T, bool FIRST, typename S> static hipError_t grouped(const ExpertsParams &P, hipStream_t st) {
    return start_lds<experts_many_kernel<T, FIRST, S>>(dim3((unsigned)workgroups<FIRST, S>(P)), dim3(S::THREADS), S::LDS, st, P);
}
// The tiles, rows x tokens.  32 bits: 64 x 32.  bfloat16: 64 x 64, 128 x 64, 128 x 128, 256 x 256; of activations in pairs 64 x 32 and 128 x 32.
template <typename T> using Small = Grouped<T, 2, sizeof(T) == 2 ? 2 : 1, 2, 2, 3>;
template <typename T> using Low = Grouped<T, 4, 2, 2, 2>;
template <typename T> using Square = Grouped<T, 4, 4, 2, 2>;
template <typename T> using Large = Grouped<T, 8, 4, 2, 4>;
template <typename T> using PairSmall = Grouped<T, 2, 1, 2, 2, 3, 16, true>;
template <typename T> using PairLow = Grouped<T, 4, 1, 2, 2, 2, 16, true>;
template <typename T> using Any = Grouped<T, 2, sizeof(T) == 2 ? 2 : 1, 2, 2, 3, 4>;       // (rows on 4-byte boundaries)
inline bool in_pairs(int slots, int experts) { return (size_t)slots <= PAIR_TOKENS * experts; }
// No product of these tokens needs more threads than 31 bits count (Small and PairSmall have the most workgroups, Large the most threads).
template <typename T> static bool one_launch(const ExpertsParams &P) {
    auto in = [](long long most, int threads) { return most <= INT_MAX / threads; };
    if (!in(workgroups<true, Small<T>>(P), Small<T>::THREADS) || !in(workgroups<false, Small<T>>(P), Small<T>::THREADS)) return false;
    if constexpr (sizeof(T) == 2)
        return in(workgroups<true, Large<T>>(P), Large<T>::THREADS) && in(workgroups<false, Large<T>>(P), Large<T>::THREADS) &&
               (!in_pairs(P.n * P.k, P.experts) || in(workgroups<false, PairSmall<T>>(P), PairSmall<T>::THREADS));
    return true;
}
// What tiles of S are expected to take (bfloat16), in us.  A CU runs its workgroups in rounds of S::PER_CU; a stage of a round takes what bounds it: bringing
// it to LDS (50 KB/us and CU), multiplying it (`tflops` a CU), reading the matrices' part (6.2 TB/s), or the way from
// memory as far as the ring does not hide it; `around`: what is in front of the stages and behind them.
template <bool FIRST, typename S> static double grouped_us(const ExpertsParams &P, double tflops, double around) {
    const int rows = FIRST ? P.ff : P.dim, K = FIRST ? P.dim : P.ff, br = S::RT * (FIRST ? 8 : 16);
    const double slots = (double)P.n * P.k, hit = std::min<double>(P.experts, slots), tiles = std::max(hit, slots / S::BT + hit / 2), per_tile = std::min<double>(S::BT, slots / tiles);
    const double all = tiles * ((rows + br - 1) / br), round = 256 * S::PER_CU, stages = (K + S::KB - 1) / S::KB;
    const double bring = (S::RT * 16 + per_tile) * 128 / 50e3, multiply = 2 * S::RT * 16 * std::max(32., std::min<double>(S::BT, per_tile + 16)) * S::KB / (tflops * 1e6);
    const double read = hit / tiles * S::RT * 16 * 128 / 6.2e6, way = S::NST > 2 ? 0.29 : 0.92;
    auto took = [&](double workgroups) {
        const double a_cu = std::ceil(workgroups / 256);
        return stages * std::max(std::max(a_cu * bring, a_cu * multiply), std::max(workgroups * read, way)) + around;
    };
    const double full = std::floor(all / round), left = all - full * round;
    return full * took(round) + (left > 0 ? took(left) : 0);
}
// Which tiles.  bfloat16: rows x tokens 64 x 64 in three stages (three workgroups a CU), 128 x 64 in two (three), 128 x 128 (two) or 256 x 256 (one), whichever
// is expected to be done first: over these products 1 % behind the best of the four on the average and 5 % at most.  us of a product with gate and up / with
// down, the median of 24 over three sets of inputs (another run of the third line's 128 x 128 has 132 / 92: the chip's clock):
//                                                                     64 x 64     128 x 64    128 x 128   256 x 256
//   64 experts of 1536 x 768, 8 a token        32 tokens              50 / 28     48 / 25     60 / 32     73 / 40
//                                              512                    80 / 47     78 / 47     75 / 46     85 / 53
//                                              2047                   179 / 116   143 / 97    124 / 84    131 / 94
//   64 of 1536 x 1024, 6 a token               64                     65 / 36     80 / 33     66 / 41     79 / 47
//   8 of 768 x 2048, 2 a token                 333                    17 / 12     14 / 21     16 / 24     24 / 48
//                                              1000                   32 / 20     28 / 29     29 / 32     28 / 55
//   8 of 4096 x 11008, 2 a token               16                     221 / 117   232 / 149   243 / 149   252 / 209
//                                              993                    732 / 399   572 / 354   505 / 361   500 / 278
// (the last one's 256 x 256 take 431 or 503 by the inputs: an expert with a few tokens past 256 is another tile, and the last of them another round.  The rule
// knows numbers, not the choices.)
// 32 bits: 64 x 32 in three stages, bound by the matrix rate; 64 x 64 and 128 x 128 beside it: 77 tokens to 4 of 16 of 760 x 500 21 / 11, 22 / 15, 55 / 38; of the
// first experts 256 tokens 166 / 87, 208 / 110, 385 / 198, 1024 tokens 507 / 260, 496 / 259, 596 / 319.
template <typename T, bool FIRST> static hipError_t grouped_product(const ExpertsParams &P, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        const double small = grouped_us<FIRST, Small<T>>(P, 5.4, 2.9), low = grouped_us<FIRST, Low<T>>(P, 5.4, 2.9), square = grouped_us<FIRST, Square<T>>(P, 5.4, 2.9), large = grouped_us<FIRST, Large<T>>(P, 3.3, 8.1);
        const double least = std::min(std::min(small, low), std::min(square, large));
        if (large == least) return grouped<T, FIRST, Large<T>>(P, st);
        if (square == least) return grouped<T, FIRST, Square<T>>(P, st);
        if (low == least) return grouped<T, FIRST, Low<T>>(P, st);
    }
    return grouped<T, FIRST, Small<T>>(P, st);
}
template <typename T> static hipError_t experts(ExpertsParams P, bool &summed, hipStream_t st) {
    P.h_rest = nullptr;
    const int slots = P.n * P.k;
    auto rows_on = [&](size_t bytes) {                   // every row starts on such a boundary
        return on(P.x, bytes) && on(P.gate, bytes) && on(P.up, bytes) && on(P.down, bytes) && P.ldx * sizeof(T) % bytes == 0 && P.dim * sizeof(T) % bytes == 0 && P.ff * sizeof(T) % bytes == 0;
    };
    const bool vec = rows_on(16);
    hipError_t rc;
    summed = vec && (size_t)slots <= most_by_token(P.k, P.experts);
    if (summed) {
        if ((rc = start(experts_token_first_kernel<T>, dim3((P.ff + 3) / 4, slots), dim3(256), 0, st, P)) != hipSuccess) return rc;
        return start(experts_token_second_kernel<T>, dim3((P.dim + 3) / 4, P.n), dim3(256), 0, st, P);
    }
    if ((rc = start(plan_kernel, dim3(P.experts), dim3(1024), 0, st, P.ids, slots, P.experts, P.offs, P.order)) != hipSuccess) return rc;
    if (vec) {
        const bool pair = sizeof(T) == 2 && in_pairs(slots, P.experts);
        if (pair) P.h_rest = reinterpret_cast<T *>(P.h) + (size_t)slots * P.ff;
        if ((rc = grouped_product<T, true>(P, st)) != hipSuccess) return rc;
        if constexpr (sizeof(T) == 2) if (pair) {
            // (reading the matrix bounds both: neither the second product nor the second half of the tokens' pieces is in the estimates)
            return grouped_us<false, PairLow<T>>(P, 5.4, 2.9) < grouped_us<false, PairSmall<T>>(P, 5.4, 2.9) ? grouped<T, false, PairLow<T>>(P, st) : grouped<T, false, PairSmall<T>>(P, st);
        }
        return grouped_product<T, false>(P, st);
    }
    // us a pass with rows on 16-byte boundaries, on 4-byte and on 2-byte ones: 333 tokens to 2 of 8 of 768 x 2048 32, 43, 580; 64 to 6 of 64 of 1536 x 1024
    // 111, 127, 871; 2047 to 8 of 64 of 1536 x 768 229, 393, 8425
    if (rows_on(4)) {
        if ((rc = grouped<T, true, Any<T>>(P, st)) != hipSuccess) return rc;
        return grouped<T, false, Any<T>>(P, st);
    }
    if constexpr (sizeof(T) == 2) {
        const int hit = std::min(P.experts, slots), tiles = std::min(hit + (slots - hit) / 16, 65535);
        if ((rc = start(experts_any_kernel<T, true>, dim3((P.ff + 31) / 32, tiles), dim3(256), 0, st, P)) != hipSuccess) return rc;
        return start(experts_any_kernel<T, false>, dim3((P.dim + 31) / 32, tiles), dim3(256), 0, st, P);
    }
    return hipErrorInvalidValue;                         // (the entry points refuse such pointers)
}

template <typename T> static hipError_t close(const CloseParams &P, hipStream_t st) {
    auto four = [](const void *p, long long ld, size_t size) { return (reinterpret_cast<uintptr_t>(p) & (4 * size - 1)) == 0 && ld % 4 == 0; };
    const bool v4 = P.dim % 4 == 0 && four(P.x, P.ldx, 4) && four(P.add, P.ldadd, 4) && four(P.base, P.ldbase, 4) && four(P.d, P.ldd, sizeof(T)) && four(P.part, 0, 4) &&
                    four(P.post, 0, 4) && four(P.gate, P.ldgate, 4) && four(P.pre, 0, 4) && four(P.x_out, P.ldxo, 4) && four(P.h, P.ldh, sizeof(T)) && four(P.y, P.ldy, sizeof(T));
    const dim3 grid(P.n), block(256);
    if (v4 && P.dim <= 1024) return start(close_rows_kernel<T, 4, 1>, grid, block, 0, st, P);
    if (v4 && P.dim <= 2048) return start(close_rows_kernel<T, 4, 2>, grid, block, 0, st, P);
    if (v4 && P.dim <= 4096) return start(close_rows_kernel<T, 4, 4>, grid, block, 0, st, P);
    if (P.dim <= 1024) return start(close_rows_kernel<T, 1, 4>, grid, block, 0, st, P);
    if (P.dim <= 4096) return start(close_rows_kernel<T, 1, 16>, grid, block, 0, st, P);
    return start(close_kernel<T>, grid, block, 0, st, P);
}
// the rows from token t on, n of them
static CloseParams rows_from(CloseParams P, long long t, int n, size_t size) {
    P.x = behind(P.x, t * P.ldx); P.add = behind(P.add, t * P.ldadd); P.base = behind(P.base, t * P.ldbase); P.d = behind(P.d, t * P.ldd, size);
    P.part = behind(P.part, t * P.k * P.dim); P.ids = behind(P.ids, t * P.k); P.gate = behind(P.gate, t * P.ldgate);
    P.x_out = behind(P.x_out, t * P.ldxo); P.h = behind(P.h, t * P.ldh, size); P.y = behind(P.y, t * P.ldy, size);
    P.n = n;
    return P;
}
hipError_t launch_close(const CloseParams &P, int dtype, hipStream_t st) {
    hipError_t rc = hipSuccess;
    for (long long t = 0; t < P.n && rc == hipSuccess; t += CLOSE_TOKENS) {
        const CloseParams Q = rows_from(P, t, (int)std::min<long long>(P.n - t, CLOSE_TOKENS), dtype == NL_DTYPE_F32 ? 4 : 2);
        rc = dtype == NL_DTYPE_F32 ? close<float>(Q, st) : close<bf16>(Q, st);
    }
    return rc;
}
template <typename T> static hipError_t experts_and_close(ExpertsParams P, CloseParams C, hipStream_t st) {
    C.part = P.part; C.ids = P.ids; C.k = P.k; C.experts = P.experts; C.n = P.n; C.dim = P.dim;
    P.y = C.x_out ? nullptr : C.y;
    P.ldy = C.ldy;
    P.res_out = C.post || C.gate || C.h ? nullptr : C.x_out;       // (nothing that needs the whole row)
    P.ldo = C.ldxo; P.res = C.x; P.ldres = C.ldx; P.add = C.add; P.ldadd = C.ldadd; P.scale = C.scale;
    bool summed = false;
    const hipError_t rc = experts<T>(P, summed, st);
    if (rc != hipSuccess || (summed && (P.y || P.res_out))) return rc;
    if (summed) { C.ids = nullptr; C.k = 1; }
    return close<T>(C, st);
}
template <typename T> static hipError_t experts_in_parts(const ExpertsParams &P, const CloseParams &C, hipStream_t st) {
    // as many tokens as a launch counts; behind one another the parts share the workspace
    ExpertsParams Q = P;
    Q.n = std::min(P.n, CLOSE_TOKENS);
    while (Q.n > 1 && !one_launch<T>(Q)) Q.n = (Q.n + 1) / 2;
    const int most = Q.n;
    hipError_t rc = hipSuccess;
    for (long long t = 0; t < P.n && rc == hipSuccess; t += most) {
        Q.n = (int)std::min<long long>(P.n - t, most);
        Q.x = behind(P.x, t * P.ldx, sizeof(T)); Q.ids = behind(P.ids, t * P.k); Q.weights = behind(P.weights, t * P.k);
        rc = experts_and_close<T>(Q, rows_from(C, t, Q.n, sizeof(T)), st);
    }
    return rc;
}
hipError_t launch_experts(const ExpertsParams &P, const CloseParams &C, int dtype, hipStream_t st) {
    return dtype == NL_DTYPE_F32 ? experts_in_parts<float>(P, C, st) : experts_in_parts<bf16>(P, C, st);
}

}  // namespace nl

// ================================================================== C ABI ===

namespace {

int fail(int code, const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_error(buf);
    return code;
}

// an error of the runtime's is told here and not kept for the program's next look at it
int hip_error(const char *name, hipError_t rc) {
    (void)hipGetLastError();
    return fail(NL_ERR_HIP, "%s: %s", name, hipGetErrorString(rc));
}
int off_elements(const char *name) { return fail(NL_ERR_INVALID, "%s: an array is not on a boundary of its elements", name); }

// the caller's current device, given back at the end
struct OnDevice {
    int before = -1;
    hipError_t rc;
    explicit OnDevice(int device) {
        if ((rc = hipGetDevice(&before)) == hipSuccess && before != device) rc = hipSetDevice(device);
        else if (rc == hipSuccess) before = -1;          // nothing to give back
    }
    ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
    OnDevice(const OnDevice &) = delete;
};

// what every operator checks behind its own arguments, then the launches
template <typename F> int on_device(const char *name, int device, void *stream, F launches) {
    static std::atomic<int> seen{0};                     // devices, once there are any
    int ndev = seen.load(std::memory_order_relaxed);
    if (ndev == 0) {
        if (hipGetDeviceCount(&ndev) != hipSuccess || ndev == 0) {
            (void)hipGetLastError();
            return fail(NL_ERR_HIP, "%s: no HIP device", name);
        }
        seen.store(ndev, std::memory_order_relaxed);
    }
    if (device < 0 || device >= ndev) return fail(NL_ERR_INVALID, "%s: device %d of %d", name, device, ndev);
    OnDevice on(device);
    if (on.rc != hipSuccess) return hip_error(name, on.rc);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    // the default streams' handles are no streams: they are of the device that is current, and a runtime that does not know hipStreamLegacy yet ends the
    // process when it is asked for that one's
    if (st == hipStreamLegacy) st = nullptr;
    hipDevice_t at = device;
    if (st && st != hipStreamPerThread) {
        const hipError_t rc = hipStreamGetDevice(st, &at);
        if (rc != hipSuccess) return hip_error(name, rc);
    }
    if (at != device) return fail(NL_ERR_INVALID, "%s: the stream is of device %d, not %d", name, at, device);
    const hipError_t rc = launches(st);
    return rc == hipSuccess ? (int)NL_OK : hip_error(name, rc);
}

const char *experts_error(const nl_experts_desc *d, int n) {
    if (!d) return "no description";
    if (d->experts < 1 || d->experts > NL_MAX_EXPERTS) return "experts: 1 to 1024";
    if (d->per_token < 1 || d->per_token > NL_MAX_PER_TOKEN) return "per_token: 1 to 32";
    if (d->dim < 1 || d->ff < 1 || d->dim > 1 << 20 || d->ff > 1 << 20) return "dim and ff: 1 to 1048576";
    if (d->act != NL_ACT_SILU && d->act != NL_ACT_GELU_TANH) return "act";
    if (d->dtype != NL_DTYPE_BF16 && d->dtype != NL_DTYPE_F32) return "dtype";
    if (n < 0 || (long long)n * d->per_token > INT_MAX / 2) return "n: 0 to 2^30 / per_token";
    return nullptr;
}

}  // namespace

extern "C" {

int nl_op_route(int device, void *stream, const nl_route_desc *d, int n, const float *logits, int64_t ld, const float *bias, int32_t *ids, float *weights) {
    if (!d || n < 0) return fail(NL_ERR_INVALID, "route: %s", d ? "n is negative" : "no description");
    if (d->experts < 1 || d->experts > NL_MAX_EXPERTS) return fail(NL_ERR_UNSUPPORTED, "route: %d experts, 1 to %d are taken", d->experts, NL_MAX_EXPERTS);
    if (d->per_token < 1 || d->per_token > NL_MAX_PER_TOKEN || d->per_token > d->experts)
        return fail(NL_ERR_INVALID, "route: %d per token, 1 to %d are taken, no more than experts", d->per_token, NL_MAX_PER_TOKEN);
    if (d->score != NL_SCORE_SOFTMAX && d->score != NL_SCORE_SIGMOID) return fail(NL_ERR_INVALID, "route: score %d", d->score);
    if (bias && d->score != NL_SCORE_SIGMOID) return fail(NL_ERR_UNSUPPORTED, "route: a bias goes with sigmoid scores");
    if (!(d->scale - d->scale == 0.f)) return fail(NL_ERR_INVALID, "route: scale is not finite");
    if (n == 0) return NL_OK;
    if (!logits || !ids || !weights) return fail(NL_ERR_INVALID, "route: null argument");
    if (!on(logits, 4) || !on(bias, 4) || !on(ids, 4) || !on(weights, 4)) return off_elements("route");
    if (ld < d->experts) return fail(NL_ERR_INVALID, "route: ld %lld is less than %d experts", (long long)ld, d->experts);
    RouteParams P{};
    P.logits = logits; P.bias = bias; P.ld = ld; P.n = n; P.experts = d->experts; P.k = d->per_token; P.sigmoid = d->score == NL_SCORE_SIGMOID;
    P.renorm = d->renorm != 0; P.scale = d->scale; P.ids = ids; P.weights = weights;
    return on_device("route", device, stream, [&](hipStream_t st) { return launch_route(P, st); });
}

uint64_t nl_op_experts_workspace(const nl_experts_desc *d, int n) {
    if (const char *m = experts_error(d, n)) { fail(NL_ERR_INVALID, "experts: %s", m); return 0; }
    return experts_layout(n, d->per_token, d->experts, d->dim, d->ff, d->dtype).bytes;
}

int nl_op_experts(int device, void *stream, const nl_experts_desc *d, int n, const void *x, int64_t ldx, const int32_t *ids, const float *weights,
                  const void *gate, const void *up, const void *down, void *y, int64_t ldy, void *workspace, uint64_t workspace_bytes) {
    if (const char *m = experts_error(d, n)) return fail(NL_ERR_INVALID, "experts: %s", m);
    if (n == 0) return NL_OK;
    if (!x || !ids || !weights || !gate || !up || !down || !y || !workspace) return fail(NL_ERR_INVALID, "experts: null argument");
    if (ldx < d->dim || ldy < d->dim) return fail(NL_ERR_INVALID, "experts: ldx %lld and ldy %lld, rows have %d elements", (long long)ldx, (long long)ldy, d->dim);
    const size_t size = d->dtype == NL_DTYPE_F32 ? 4 : 2;
    if (!on(x, size) || !on(gate, size) || !on(up, size) || !on(down, size) || !on(y, size) || !on(ids, 4) || !on(weights, 4)) return off_elements("experts");
    const ExpertsLayout L = experts_layout(n, d->per_token, d->experts, d->dim, d->ff, d->dtype);
    if (workspace_bytes < L.bytes) return fail(NL_ERR_INVALID, "experts: workspace of %llu bytes, %llu are needed", (unsigned long long)workspace_bytes, (unsigned long long)L.bytes);
    if (!on(workspace, 16)) return fail(NL_ERR_INVALID, "experts: workspace is not on a 16-byte boundary");
    ExpertsParams P{};
    P.x = x; P.gate = gate; P.up = up; P.down = down; P.ldx = ldx; P.ids = ids; P.weights = weights; P.n = n; P.k = d->per_token; P.experts = d->experts;
    P.dim = d->dim; P.ff = d->ff; P.act = d->act;
    place_experts(P, workspace, L);
    CloseParams C{};
    C.y = y; C.ldy = ldy;
    return on_device("experts", device, stream, [&](hipStream_t st) { return launch_experts(P, C, d->dtype, st); });
}

int nl_op_residual_norm(int device, void *stream, const nl_residual_norm_desc *d, int n, const float *x, int64_t ldx, const void *b, int64_t ldb, const float *post,
                        const float *gate, int64_t ldgate, const float *pre, float *x_out, int64_t ldxo, void *h, int64_t ldh) {
    if (!d || n < 0) return fail(NL_ERR_INVALID, "residual_norm: %s", d ? "n is negative" : "no description");
    if (d->dim < 1 || d->dim > 1 << 20) return fail(NL_ERR_INVALID, "residual_norm: dim %d, 1 to %d are taken", d->dim, 1 << 20);
    if (d->dtype != NL_DTYPE_BF16 && d->dtype != NL_DTYPE_F32) return fail(NL_ERR_INVALID, "residual_norm: dtype %d", d->dtype);
    if (!(d->eps >= 0.f) || !(d->eps - d->eps == 0.f) || !(d->scale - d->scale == 0.f)) return fail(NL_ERR_INVALID, "residual_norm: eps or scale");
    if (n == 0) return NL_OK;
    if (!x || !b || !x_out || (h && !pre)) return fail(NL_ERR_INVALID, "residual_norm: null argument");
    if (ldx < d->dim || ldb < d->dim || ldxo < d->dim || (gate && ldgate != 0 && ldgate < d->dim) || (h && ldh < d->dim))
        return fail(NL_ERR_INVALID, "residual_norm: a row distance is less than %d", d->dim);
    const size_t size = d->dtype == NL_DTYPE_F32 ? 4 : 2;
    if (!on(x, 4) || !on(b, size) || !on(post, 4) || !on(gate, 4) || (h && !on(pre, 4)) || !on(x_out, 4) || !on(h, size)) return off_elements("residual_norm");
    if (x_out == x && ldxo != ldx) return fail(NL_ERR_INVALID, "residual_norm: x_out is x with other rows");
    CloseParams P{};
    P.x = x; P.ldx = ldx; P.d = b; P.ldd = ldb; P.post = post; P.gate = gate; P.ldgate = ldgate; P.pre = pre; P.x_out = x_out; P.ldxo = ldxo; P.h = h; P.ldh = ldh;
    P.n = n; P.dim = d->dim; P.eps = d->eps; P.scale = d->scale;
    return on_device("residual_norm", device, stream, [&](hipStream_t st) { return launch_close(P, d->dtype, st); });
}

}  // extern "C"
