// C-ABI entry points of libjitnn_hip.so (declared in include/jitnn_hip.h): argument validation, weight
// handles, kernel selection and launch.  Host side of the path in C++; every kernel is in the headers
// included below.
#include "../../include/jitnn_hip.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cmath>
#include <cstring>
#include <mutex>
#include <new>
#include <utility>
#include <vector>

#include <sys/syscall.h>
#include <unistd.h>

#include "attn_packed.h"
#include "attn_split.h"
#include "dequant.h"
#include "experts.h"
#include "gemv.h"
#include "gemv_mfma.h"
#include "gemv_tail.h"
#include "gguf_file.h"
#include "glue.h"
#include "prefill.h"
#include "scratch.h"
#include "serving.h"
#include "tu.h"

using namespace jitnn;

struct jitnn_hip_weight {
    int fmt;  // of the blocks at dev: the caller's format, or the one an uploaded weight was rewritten into (below)
    int n, k;
    long long nbytes;
    uint8_t *dev;
    bool owned;
    int file_fmt = 0;  // != 0: what the caller uploaded, when that was another format of exactly the same values
    long long file_nbytes = 0;
};

// Scratch of the entry point that allocates nothing (jitnn_hip_linear_noalloc_dev): FP16 activations in operand order,
// their row scales and the partial sums of K slices of a many-row linear.  One copy per GPU, held until the process
// ends.  In host code this name is only a handle for hipGetSymbolAddress; the device address is kept in State.
#define JITNN_HIP_SCRATCH_BYTES (64ull << 20)
static __device__ __align__(256) unsigned char scratch[JITNN_HIP_SCRATCH_BYTES];

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
    return code;
}

#define HIP_TRY(expr)                                                                                       \
    do {                                                                                                    \
        hipError_t e_ = (expr);                                                                             \
        if (e_ != hipSuccess) return fail(JITNN_HIP_EDEVICE, "%s: %s", #expr, hipGetErrorString(e_));       \
    } while (0)

struct State {
    bool ready = false;
    int device = -1;
    int cus = 0;
    long long hbm = 0;
    char name[256] = "";
    float nib = 0.f;  // 1 / (value of E4M3 byte 0x01): 512 for OCP, 1024 for FNUZ
    size_t max_lds = 0;      // LDS one workgroup may ask for
    size_t lds_per_cu = 0;   // LDS of a compute unit
    // JITNN_HIP_GEMV_MAX_ROWS: up to this many rows run the FP32 GEMV kernels (in batches of 8), more rows the FP16
    // MFMA kernel - the counterpart of jitnn.gguf.tiledRows (core/JitnnConfig.java:423-424).  64 keeps every row
    // count the reference's own tests use (1, 5, 40) on the FP32 path, whose error meets their 2e-4 / 1e-3 bars.
    int gemv_max_rows = 64;
    bool transcode = true;            // JITNN_HIP_TRANSCODE=0: uploaded Q5_0 / Q3_K blocks stay as they are (plain kernels)
    void *scratch_ptr = nullptr;    // device address of `scratch` on g.device (hipGetSymbolAddress at init)
    bool gemv_i8 = true;            // JITNN_HIP_GEMV_I8=0: batch-1 K-quant GEMV on the FP32 register kernels instead of the INT8 matrix-core one
};
State g;
std::mutex g_mu;


__global__ void fp8_probe_kernel(float *out) {
    f32x2 p = __builtin_amdgcn_cvt_pk_f32_fp8(0x00000f01, false);
    out[0] = p.x;
    out[1] = p.y;
}

// Pure streaming read: every thread xors the 16-byte words it loads; the store can never happen for real data
// but keeps the loads alive.  U loads in flight per lane (the workgroups stride the buffer together), NT: non-temporal loads.
template <int U, bool NT>
__global__ void __launch_bounds__(256) probe_read_kernel(const u32x4 *__restrict__ p, size_t n16, uint32_t *sink, uint32_t threads) {
    const size_t stride = threads;  // (the grid's threads as an argument: gridDim is fetched from a cold argument block by the wave's first instructions)
    u32x4 acc = {0, 0, 0, 0};
    size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    for (; i + (U - 1) * stride < n16; i += U * stride) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = NT ? __builtin_nontemporal_load(p + i + u * stride) : p[i + u * stride];
#pragma unroll
        for (int u = 0; u < U; ++u) acc ^= v[u];
    }
    for (; i < n16; i += stride) acc ^= p[i];
    if ((acc.x ^ acc.y ^ acc.z ^ acc.w) == 0x9e3779b9u && sink) *sink = acc.x;
}

// ---- counters (jitnn_hip_stats): calls and tensor bytes per operator, the reference's telemetry convention
enum StatOp { ST_GEMV, ST_MFMA, ST_DEQUANT, ST_QUANT, ST_DECODE, ST_PREFILL, ST_COUNT };
const char *const kStatNames[ST_COUNT] = {"linear_gemv", "linear_mfma", "dequantize", "quantize_q8_0", "llama_decode", "llama_prefill"};
std::atomic<long long> g_stat_calls[ST_COUNT], g_stat_bytes[ST_COUNT];
thread_local int g_stat_nested = 0;  // inside a model step: its linears are the step's own traffic
void count_op(StatOp op, long long bytes) {
    if (g_stat_nested) return;
    g_stat_calls[op].fetch_add(1, std::memory_order_relaxed);
    g_stat_bytes[op].fetch_add(bytes, std::memory_order_relaxed);
}
struct StatNest {
    StatNest() { ++g_stat_nested; }
    ~StatNest() { --g_stat_nested; }
};

bool known(int fmt) { return block_values(fmt) != 0; }

bool calling_thread_is_main() { return (long)syscall(SYS_gettid) == (long)getpid(); }

// Kernels that want more than 64 KiB of dynamic LDS must be told so once; remembered per kernel so that steady-state
// launches (and launches under graph capture) make no attribute calls.
int allow_lds(const void *fn, size_t lds) {
    if (lds <= 65536) return JITNN_HIP_OK;
    static std::mutex mu;
    static std::vector<std::pair<const void *, size_t>> seen;
    std::lock_guard<std::mutex> lock(mu);
    for (auto &e : seen)
        if (e.first == fn && e.second >= lds) return JITNN_HIP_OK;
    hipError_t e = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return fail(JITNN_HIP_EDEVICE, "hipFuncSetAttribute(%zu bytes of LDS): %s", lds, hipGetErrorString(e));
    seen.emplace_back(fn, lds);
    return JITNN_HIP_OK;
}

int check_ready() {
    if (!g.ready) return fail(JITNN_HIP_ENODEVICE, "jitnn_hip_init has not succeeded in this process");
    return JITNN_HIP_OK;
}

// ------------------------------------------------------------------------------------------ launch tables

typedef void (*gemv_fn)(const uint8_t *, const float *, const float *, float *, int, int, int, int, float);

struct GemvVariant {
    gemv_fn fn;
    int B, R;
    size_t lds_per_step;  // LDS bytes per staged wave step
    int unit_values;      // values one lane decodes per step
};

template <class U, int B, int R, int NBUF>
GemvVariant variant() {
    // the fp8 nibble conversion only applies to the 4-bit formats; the others ignore CV
    constexpr int CV = (U::FMT == F_Q4_K || U::FMT == F_Q4_0 || U::FMT == F_Q4_1) ? 1 : 0;
    return GemvVariant{gemv_lds_kernel<U, B, R, CV, NBUF>, B, R, gemv_lds_bytes<U>(B, 1), U::UV};
}

// batch rows -> (rows decoded together, ring depth): chosen so that no variant spills registers
template <class U>
GemvVariant pick_unit(int rows) {
    if (rows <= 1) return variant<U, 1, 2, 2>();
    if (rows <= 2) return variant<U, 2, 2, 2>();
    if constexpr (U::FMT == F_Q8_0) {  // 17 dwords per block pair: one row at a time
        if (rows <= 4) return variant<U, 4, 1, 1>();
        return variant<U, 8, 1, 1>();
    } else {
        if (rows <= 4) return variant<U, 4, 2, 1>();
        return variant<U, 8, 2, 1>();
    }
}

GemvVariant pick(int fmt, int rows, bool pairs) {
    switch (fmt) {
    case F_Q4_0: return pairs ? pick_unit<UnitPair<F_Q4_0>>(rows) : pick_unit<Unit<F_Q4_0>>(rows);
    case F_Q4_1: return pairs ? pick_unit<UnitPair<F_Q4_1>>(rows) : pick_unit<Unit<F_Q4_1>>(rows);
    case F_Q8_0: return pairs ? pick_unit<UnitPair<F_Q8_0>>(rows) : pick_unit<Unit<F_Q8_0>>(rows);
    case F_Q4_K: return pick_unit<Unit<F_Q4_K>>(rows);
    case F_Q5_K: return pick_unit<Unit<F_Q5_K>>(rows);
    default: return pick_unit<Unit<F_Q6_K>>(rows);
    }
}

typedef void (*gemv1_fn)(const uint8_t *, const float *, const float *, float *, int, int, float);
typedef void (*xreg_fn)(const XregArgs);

// The 32-value formats decode pairs of blocks when the row holds an even number of them (aligned loads),
// single blocks otherwise.
template <int PF, bool BIAS, bool NORM, bool DUAL>
xreg_fn pick_xreg_fmt(int fmt, bool pairs) {
    switch (fmt) {
    case F_Q4_0:
        return pairs ? gemv_xreg_kernel<UnitPair<F_Q4_0>, 1, PF, BIAS, NORM, DUAL> : gemv_xreg_kernel<Unit<F_Q4_0>, 1, PF, BIAS, NORM, DUAL>;
    case F_Q4_1:
        return pairs ? gemv_xreg_kernel<UnitPair<F_Q4_1>, 1, PF, BIAS, NORM, DUAL> : gemv_xreg_kernel<Unit<F_Q4_1>, 1, PF, BIAS, NORM, DUAL>;
    case F_Q8_0:
        return pairs ? gemv_xreg_kernel<UnitPair<F_Q8_0>, 0, PF, BIAS, NORM, DUAL> : gemv_xreg_kernel<Unit<F_Q8_0>, 0, PF, BIAS, NORM, DUAL>;
    case F_Q4_K: return gemv_xreg_kernel<Unit<F_Q4_K>, 1, PF, BIAS, NORM, DUAL>;
    case F_Q5_K: return gemv_xreg_kernel<Unit<F_Q5_K>, 0, PF, BIAS, NORM, DUAL>;
    default: return gemv_xreg_kernel<Unit<F_Q6_K>, 0, PF, BIAS, NORM, DUAL>;
    }
}

// mode 0: plain; 1: with bias; 2: with fused RMSNorm; 3: fused RMSNorm + SwiGLU pair (PF 1 or 3)
xreg_fn pick_xreg(int fmt, bool pairs, int mode, int pf) {
    switch (mode) {
    case 1: return pf == 1 ? pick_xreg_fmt<1, true, false, false>(fmt, pairs) : pick_xreg_fmt<2, true, false, false>(fmt, pairs);
    case 2: return pf == 1 ? pick_xreg_fmt<1, false, true, false>(fmt, pairs) : pick_xreg_fmt<2, false, true, false>(fmt, pairs);
    case 3: return pf == 1 ? pick_xreg_fmt<1, false, true, true>(fmt, pairs) : pick_xreg_fmt<3, false, true, true>(fmt, pairs);
    default: return pf == 1 ? pick_xreg_fmt<1, false, false, false>(fmt, pairs) : pick_xreg_fmt<2, false, false, false>(fmt, pairs);
    }
}

// One launch of the register-resident batch-1 kernel (rows of at most 4096 values) over up to three matrices of one
// format and row length.  norm_w != NULL fuses the RMSNorm of x; w2 != NULL computes silu(w x) * (w2 x).
struct XregCall {
    const jitnn_hip_weight *w[3] = {nullptr, nullptr, nullptr};
    float *y[3] = {nullptr, nullptr, nullptr};
    const float *bias = nullptr;  // for w[0] only
    const jitnn_hip_weight *w2 = nullptr;
    const float *x = nullptr, *norm_w = nullptr;
    float eps = 0.f;
    Epilogue epi;  // one matrix, no norm, no w2; launch_i8 only
};

// kernel arguments of a call; returns the total number of rows
int xreg_args(const XregCall &c, XregArgs &a) {
    int n = 0;
    for (int i = 0; i < 3; ++i) {
        a.w[i] = c.w[i] ? c.w[i]->dev : c.w[0]->dev;
        a.y[i] = c.y[i] ? c.y[i] : c.y[0];
        a.bias[i] = c.bias;
        a.n[i] = c.w[i] ? c.w[i]->n : 0;
        n += a.n[i];
    }
    a.w2 = c.w2 ? c.w2->dev : nullptr;
    a.x = c.x;
    a.nw = c.norm_w;
    a.eps = c.eps;
    a.k = c.w[0]->k;
    a.nib = g.nib;
    return n;
}

// The INT8 matrix-core kernel (gemv_i8.h) takes what the register-resident kernels take of the K-quants, and rows of up
// to 16384 values.
constexpr int PREFILL_MIN_SLICE = 8;  // fewest K steps (of 64 values) a slice of a launch of several many-row weights may have

// Its row groups are four rows: at least four rows in all, and the segments of a shared launch whole groups; its buffer
// loads address a matrix with 32 bits.
bool i8_ok(const XregCall &c) {
    if (!g.gemv_i8 || !gemv_i8_supported(c.w[0]->fmt, c.w[0]->k)) return false;
    int n = 0;
    for (int i = 0; i < 3; ++i) {
        if (!c.w[i]) continue;
        n += c.w[i]->n;
        if (c.w[i]->nbytes >= (1ll << 32) || (c.w[1] && c.w[i]->n % 4 != 0)) return false;
        if ((block_values(c.w[i]->fmt) == 32 || c.w[i]->fmt == F_Q2_K) && ((uintptr_t)c.w[i]->dev & 3) != 0) return false;  // (fetched as dwords)
        if (is_extra_format(c.w[i]->fmt) && (c.w[1] || c.w2 || c.norm_w)) return false;  // (Q5_1, Q2_K: no fused launches)
    }
    if (c.w2 && c.w2->nbytes >= (1ll << 32)) return false;
    if (c.w[1] && (!c.norm_w || c.w2)) return false;  // (several matrices in one launch: the kernel has that for the fused norm only)
    return n >= 4;
}

int i8_args(const XregCall &c, I8Args &a) {
    int n = 0;
    for (int i = 0; i < 3; ++i) {
        a.w[i] = c.w[i] ? c.w[i]->dev : c.w[0]->dev;
        a.y[i] = c.y[i] ? c.y[i] : c.y[0];
        a.bias[i] = c.bias;
        a.n[i] = c.w[i] ? c.w[i]->n : 0;
        n += a.n[i];
    }
    a.w2 = c.w2 ? c.w2->dev : nullptr;
    a.x = c.x;
    a.nw = c.norm_w;
    a.eps = c.eps;
    a.k = c.w[0]->k;
    a.rows = 1;
    a.epi = c.epi;
    return n;
}

// workgroups and turns in flight for a launch of `groups` row groups (four rows each) of `waves`-wave workgroups
void i8_shape(int fmt, int groups, int waves, bool dual, int &blocks, int &pf) {
    // Measured (us, pf / workgroups per CU): Q4_K 14336 x 4096 8.40 (1/2) 8.44 (2/1) 8.48 (3/1) 9.54 (1/4); Q4_K 4096 x 4096 4.75 (1/2)
    // 4.93 (1/1) 5.82 (1/4); Q6_K 128256 x 4096 71.9 (2/1) 72.9 (3/1) 73.6 (1/1) 74.5 (1/2); Q6_K 4096 x 14336 (14 waves) 12.9
    // (1/1) 14.3 (2/1) 16.2 (1/2).  Tall matrices: one workgroup per CU with two turns in flight behind the one being
    // multiplied; short ones: two workgroups with one; long rows: one with one.
    const int turns1 = (groups + g.cus - 1) / g.cus;
    // (Q8_0, twice the bytes of a 4-bit format per turn: one workgroup per CU on short matrices too - 4096 x 4096 5.50 us (1/1) against
    // 5.74 (1/2), 5.72 (2/1), 6.31 (2/2), 6.67 (1/3), 7.15 (1/4))
    const int per_cu = waves > 4 ? 1 : turns1 >= 8 ? 1 : (fmt == F_Q8_0 && turns1 >= 4) ? 1 : 2;
    pf = waves > 4 ? 1 : turns1 >= 8 ? (dual ? 3 : 2) : 1;  // (gate + up of an 8B layer: 14.4 us with three turns in flight, 15.1 with two)
    blocks = groups < g.cus * per_cu ? groups : g.cus * per_cu;
}

int launch_i8(const XregCall &c, hipStream_t stream) {
    I8Args a{};
    const int n = i8_args(c, a);
    const int mode = c.w2 ? I8_DUAL : c.norm_w ? I8_NORM : c.epi.any() ? I8_EPI : c.bias ? I8_BIAS : I8_PLAIN;
    int blocks, pf;
    i8_shape(c.w[0]->fmt, (n + 3) / 4, (a.k + 1023) / 1024, c.w2 != nullptr, blocks, pf);
    if (c.w[0]->fmt == F_Q5_K && pf > 2) pf = 2;  // (five loads per turn: a fourth buffer does not fit 128 registers)
    if (!gemv_i8_launch(c.w[0]->fmt, mode, pf, (unsigned)blocks, stream, a))
        return fail(JITNN_HIP_EDEVICE, "no INT8 GEMV kernel for format %d in mode %d, rows of %d values", c.w[0]->fmt, mode, a.k);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

// Two to four activation rows, rows of at most 4096 values: the same kernel with the activations of all rows in registers - the
// operands and scales of the weights are made once, every row runs its own chains of products.  us per launch against the FP32
// two-row kernel / gemv_mfma_kernel - Q4_K 14336 x 4096: 8.9 (11.3) at two rows, 10.6 (13.9) at three, 11.3 (13.8) at four; Q4_0
// 11008 x 4096 at four: 9.6 (11.8); Q8_0 4096 x 4096: 6.7 (10.1); Q6_K 14336 x 4096: 14.3 (23.0).  The number of its 4x4x4 products
// grows with the rows (four rows: twelve digit planes in three products a step): eight rows (two groups of four along
// blockIdx.y) stay behind gemv_mfma_kernel, whose 16-row tiles take 14.5 us whatever the rows - from five rows on those stay
// ahead, except for Q6_K, whose tiles cost the most there (14336 x 4096 at eight rows: 22.6 against 28.4 us).
bool i8_batch_ok(const jitnn_hip_weight *w, int rows) {
    return g.gemv_i8 && rows >= 2 && rows <= (w->fmt == F_Q6_K ? 8 : 4) && gemv_i8_supported(w->fmt, w->k) && w->k <= 4096 && w->n >= 4 && w->nbytes < (1ll << 32) &&
           ((block_values(w->fmt) != 32 && w->fmt != F_Q2_K) || ((uintptr_t)w->dev & 3) == 0);
}

int launch_i8_batch(const jitnn_hip_weight *w, const float *x, int rows, const float *bias, const Epilogue &e, float *y, hipStream_t stream) {
    I8Args a{};
    for (int i = 0; i < 3; ++i) {
        a.w[i] = w->dev;
        a.y[i] = y;
        a.bias[i] = bias;
    }
    a.n[0] = w->n;
    a.x = x;
    a.k = w->k;
    a.rows = rows;
    a.epi = e;
    const int groups = (w->n + 3) / 4;
    // (us per launch by workgroups per CU / turns in flight, two rows - Q4_K 14336 x 4096: 10.4 (1 / 2) 10.3 (2 / 2) 10.6 (2 / 1) 11.6 (1 / 1)
    // 11.9 (3 / 1); Q4_0 11008 x 4096: 7.9 (1 / 2) 8.4 (2 / 1, 2 / 2) 8.6 (1 / 1); Q8_0 4096 x 4096: 6.4 (1 / 1) 6.7 (1 / 2) 6.9 (2 / 1) 7.7 (2 / 2);
    // four rows - Q4_K: 13.1 (1 / 2, 2 / 1) 14.0 (1 / 1); Q4_0: 10.6 (1 / 2) 10.9 (1 / 1) 11.0 (2 / 1); Q8_0: 7.1 (1 / 1) 7.7 (1 / 2) 9.1 (2 / 1))
    const int per_cu = 1, pf = (groups + g.cus - 1) / g.cus >= 8 ? 2 : 1;
    const int blocks = groups < g.cus * per_cu ? groups : g.cus * per_cu;
    if (!gemv_i8_launch(w->fmt, e.any() ? I8_EPI : bias ? I8_BIAS : I8_PLAIN, pf, (unsigned)blocks, stream, a))
        return fail(JITNN_HIP_EDEVICE, "no INT8 GEMV kernel for format %d at %d rows of %d values", w->fmt, rows, a.k);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int launch_xreg(const XregCall &c, hipStream_t stream) {
    if (i8_ok(c) && !(c.norm_w && c.bias)) return launch_i8(c, stream);
    XregArgs a{};
    const int n = xreg_args(c, a);
    const int threads = XREG_THREADS, waves = threads / 64;
    int blocks = (n + waves - 1) / waves;
    // Two workgroups (eight waves) per CU measured best for streaming: fewer, longer row streams keep HBM pages
    // open.  A wave that sees many rows needs one row of prefetch; when it sees only a handful (a 14336-row
    // matrix gives a wave seven rows) a second row in flight covers the start-up latency.
    // Matrices of few rows (a wave sees two to four of them: attn_o, a 4096 x 4096 weight) do better with three
    // workgroups per CU and one row of prefetch: Q8_0 4096 x 4096 6.9 -> 6.5 us, attn_o of the 8B step 5.34 -> 5.25; from
    // 11008 rows on the two-workgroup shape is level or ahead (Q4_0 11008 x 4096 7.56 against 7.78 us).
    const bool few = n <= 8192 && !c.w2;
    const int cap = g.cus * (few ? 3 : 2);
    if (blocks > cap) blocks = cap;
    const int rows_per_wave = (n + blocks * waves - 1) / (blocks * waves);
    const int pf = few || rows_per_wave >= 16 ? 1 : 2;
    a.rpw = rows_per_wave;
    const int mode = c.w2 ? 3 : c.norm_w ? 2 : c.bias ? 1 : 0;
    xreg_fn fn = pick_xreg(c.w[0]->fmt, a.k % 64 == 0, mode, pf);
    hipLaunchKernelGGL(fn, dim3(blocks), dim3(threads), 0, stream, a);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

typedef void (*xreg2_fn)(const XregArgs, const XregArgs, int);

// the pairs of K-quant formats a Q4_K_M / Q5_K_M layer mixes, first format < second
template <int PF>
xreg2_fn pick_xreg2_pf(int fa, int fb) {
    if (fa == F_Q4_K && fb == F_Q6_K) return gemv_xreg2_kernel<Unit<F_Q4_K>, 1, Unit<F_Q6_K>, 0, PF>;
    if (fa == F_Q4_K && fb == F_Q5_K) return gemv_xreg2_kernel<Unit<F_Q4_K>, 1, Unit<F_Q5_K>, 0, PF>;
    if (fa == F_Q5_K && fb == F_Q6_K) return gemv_xreg2_kernel<Unit<F_Q5_K>, 0, Unit<F_Q6_K>, 0, PF>;
    return nullptr;
}

bool xreg2_ok(int fa, int fb) { return pick_xreg2_pf<1>(fa < fb ? fa : fb, fa < fb ? fb : fa) != nullptr; }

// Two calls of different formats over the same normalised activations in one launch; the workgroups are shared out
// by the bytes each call streams.
int launch_xreg2(const XregCall &c0, const XregCall &c1, hipStream_t stream) {
    const bool swap = c0.w[0]->fmt > c1.w[0]->fmt;
    const XregCall &ca = swap ? c1 : c0, &cb = swap ? c0 : c1;
    if (i8_ok(ca) && i8_ok(cb) && ca.w[0]->k <= 4096 && gemv_i8_pair_supported(ca.w[0]->fmt, cb.w[0]->fmt)) {
        I8Args a{}, b{};
        const int ga = (i8_args(ca, a) + 3) / 4, gb = (i8_args(cb, b) + 3) / 4;
        const double ba = (double)ga * ca.w[0]->nbytes / ca.w[0]->n, bb = (double)gb * cb.w[0]->nbytes / cb.w[0]->n;
        int total, pf;
        i8_shape(ca.w[0]->fmt, ga + gb, (a.k + 1023) / 1024, false, total, pf);
        // (q, k | v of an 8B layer - 1536 row groups, six per CU -, us per launch by workgroups per CU / turns in flight: 6.7 (1 / 2)
        // 7.1 (1 / 1) 8.0 (2 / 1) 8.4 (2 / 2) 9.1 (3 / 1): the two formats' workgroups pace differently, one per CU keeps them apart)
        if (ga + gb >= 4 * g.cus) {
            total = g.cus;
            pf = 2;
        }
        if (total < 2) total = 2;
        int blocks_a = (int)(total * ba / (ba + bb) + 0.5);
        if (blocks_a < 1) blocks_a = 1;
        if (blocks_a > total - 1) blocks_a = total - 1;
        if (blocks_a > ga) blocks_a = ga;
        int blocks_b = total - blocks_a;
        if (blocks_b > gb) blocks_b = gb;
        if (!gemv_i8_pair_launch(ca.w[0]->fmt, cb.w[0]->fmt, pf > 2 ? 2 : pf, (unsigned)blocks_a, (unsigned)blocks_b, stream, a, b)) {
            // (a split the shared launch has no room for - three matrices of the first format, two of the second: a launch each)
            if (int rc = launch_i8(ca, stream)) return rc;
            return launch_i8(cb, stream);
        }
        HIP_TRY(hipGetLastError());
        return JITNN_HIP_OK;
    }
    XregArgs a{}, b{};
    const int na = xreg_args(ca, a), nb = xreg_args(cb, b);
    const int waves = XREG_THREADS / 64;
    const int cap = g.cus * 2;
    const double ba = (double)na * ca.w[0]->nbytes / ca.w[0]->n, bb = (double)nb * cb.w[0]->nbytes / cb.w[0]->n;
    int blocks_a = (int)(cap * ba / (ba + bb) + 0.5), blocks_b;
    if (blocks_a < 1) blocks_a = 1;
    if (blocks_a > cap - 1) blocks_a = cap - 1;
    blocks_b = cap - blocks_a;
    if (blocks_a > (na + waves - 1) / waves) blocks_a = (na + waves - 1) / waves;
    if (blocks_b > (nb + waves - 1) / waves) blocks_b = (nb + waves - 1) / waves;
    const int rpw_a = (na + blocks_a * waves - 1) / (blocks_a * waves), rpw_b = (nb + blocks_b * waves - 1) / (blocks_b * waves);
    // (one row of prefetch: the q, k | v launch of an 8B layer - 6144 rows, three per wave - 8.1 -> 7.7 us against two)
    const int pf = 1;
    a.rpw = rpw_a;
    b.rpw = rpw_b;
    xreg2_fn fn = pf == 1 ? pick_xreg2_pf<1>(ca.w[0]->fmt, cb.w[0]->fmt) : pick_xreg2_pf<2>(ca.w[0]->fmt, cb.w[0]->fmt);
    hipLaunchKernelGGL(fn, dim3(blocks_a + blocks_b), dim3(XREG_THREADS), 0, stream, a, b, blocks_a);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

// Batch 1, rows of at most 4096 values: activations in registers, one row per wave iteration.
int launch_gemv_xreg(const jitnn_hip_weight *w, const float *x, const float *bias, float *y, hipStream_t stream) {
    XregCall c;
    c.w[0] = w;
    c.y[0] = y;
    c.bias = bias;
    c.x = x;
    return launch_xreg(c, stream);
}

template <int PF>
gemv1_fn pick_ksplit_pf(int fmt, bool pairs) {
    switch (fmt) {
    case F_Q4_0: return pairs ? gemv_ksplit_kernel<UnitPair<F_Q4_0>, 1, PF> : gemv_ksplit_kernel<Unit<F_Q4_0>, 1, PF>;
    case F_Q4_1: return pairs ? gemv_ksplit_kernel<UnitPair<F_Q4_1>, 1, PF> : gemv_ksplit_kernel<Unit<F_Q4_1>, 1, PF>;
    case F_Q8_0: return pairs ? gemv_ksplit_kernel<UnitPair<F_Q8_0>, 0, PF> : gemv_ksplit_kernel<Unit<F_Q8_0>, 0, PF>;
    case F_Q4_K: return gemv_ksplit_kernel<Unit<F_Q4_K>, 1, PF>;
    case F_Q5_K: return gemv_ksplit_kernel<Unit<F_Q5_K>, 0, PF>;
    default: return gemv_ksplit_kernel<Unit<F_Q6_K>, 0, PF>;
    }
}

size_t ksplit_lds(int fmt, int slices) {  // the single-block units need the most: 2 x 64 x (9 quads + 1 sum)
    if (block_values(fmt) == 32) return gemv_ksplit_lds_bytes<Unit<F_Q4_0>>(slices);
    return fmt == F_Q6_K ? gemv_ksplit_lds_bytes<Unit<F_Q6_K>>(slices) : gemv_ksplit_lds_bytes<Unit<F_Q4_K>>(slices);
}

// Batch 1, rows of 4097..32768 values: one wave per 4096-value slice of the row, partial sums joined in LDS.
int launch_gemv_ksplit(const jitnn_hip_weight *w, const float *x, const float *bias, float *y, hipStream_t stream) {
    {
        XregCall c;
        c.w[0] = w;
        c.y[0] = y;
        c.bias = bias;
        c.x = x;
        if (i8_ok(c)) return launch_i8(c, stream);
    }
    const int slices = (w->k + 4095) / 4096;
    const size_t lds = ksplit_lds(w->fmt, slices);
    int per_cu = (int)((g.lds_per_cu - 4096) / lds);  // workgroups of one CU by LDS
    if (per_cu < 1) per_cu = 1;
    const int waves_cap = 16 / slices > 0 ? 16 / slices : 1;  // at most 16 waves (4 per SIMD: the kernels use ~128 VGPRs)
    if (per_cu > waves_cap) per_cu = waves_cap;
    // One row of prefetch, and for matrices of few rows at most three workgroups per CU: the ffn_down of an 8B layer (Q6_K
    // 4096 x 14336, four waves per workgroup) 14.6 -> 14.2 us against four workgroups with two rows in flight each, Q5_K
    // 14.0 -> 13.0, Q4_K 4096 x 8192 8.45 -> 8.2; with many rows per workgroup more of them are better (Q4_K 14336 x 8192
    // 15.4 against 16.8 us with three).
    if (w->n <= 8192 && per_cu > 3) per_cu = 3;
    int blocks = w->n < g.cus * per_cu ? w->n : g.cus * per_cu;
    const int pf = 1;
    gemv1_fn fn = pf == 1 ? pick_ksplit_pf<1>(w->fmt, w->k % 64 == 0) : pick_ksplit_pf<2>(w->fmt, w->k % 64 == 0);
    if (int rc = allow_lds((const void *)fn, lds)) return rc;
    hipLaunchKernelGGL(fn, dim3(blocks), dim3(64 * slices), lds, stream, w->dev, x, bias, y, w->n, w->k, g.nib);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

template <int PF, bool BIAS>
gemv1_fn pick_xreg_b2_fmt(int fmt, bool pairs) {
    switch (fmt) {
    case F_Q4_0: return pairs ? gemv_xreg_b2_kernel<UnitPair<F_Q4_0>, 1, PF, BIAS> : gemv_xreg_b2_kernel<Unit<F_Q4_0>, 1, PF, BIAS>;
    case F_Q4_1: return pairs ? gemv_xreg_b2_kernel<UnitPair<F_Q4_1>, 1, PF, BIAS> : gemv_xreg_b2_kernel<Unit<F_Q4_1>, 1, PF, BIAS>;
    case F_Q8_0: return pairs ? gemv_xreg_b2_kernel<UnitPair<F_Q8_0>, 0, PF, BIAS> : gemv_xreg_b2_kernel<Unit<F_Q8_0>, 0, PF, BIAS>;
    case F_Q4_K: return gemv_xreg_b2_kernel<Unit<F_Q4_K>, 1, PF, BIAS>;
    case F_Q5_K: return gemv_xreg_b2_kernel<Unit<F_Q5_K>, 0, PF, BIAS>;
    default: return gemv_xreg_b2_kernel<Unit<F_Q6_K>, 0, PF, BIAS>;
    }
}

// Batch 2, rows of at most 4096 values: both activation rows in registers.
int launch_gemv_xreg_b2(const jitnn_hip_weight *w, const float *x, const float *bias, float *y, hipStream_t stream) {
    const int waves = XREG_THREADS / 64;
    int blocks = (w->n + waves - 1) / waves;
    const int cap = g.cus * 2;
    if (blocks > cap) blocks = cap;
    const int rows_per_wave = (w->n + blocks * waves - 1) / (blocks * waves);
    const int pf = rows_per_wave >= 16 ? 1 : 2;
    const bool pairs = w->k % 64 == 0;
    gemv1_fn fn = bias ? (pf == 1 ? pick_xreg_b2_fmt<1, true>(w->fmt, pairs) : pick_xreg_b2_fmt<2, true>(w->fmt, pairs))
                       : (pf == 1 ? pick_xreg_b2_fmt<1, false>(w->fmt, pairs) : pick_xreg_b2_fmt<2, false>(w->fmt, pairs));
    hipLaunchKernelGGL(fn, dim3(blocks), dim3(XREG_THREADS), 0, stream, w->dev, x, bias, y, w->n, w->k, g.nib);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

// Batch 2..8, rows a multiple of 256 values long: block sums on the matrix cores, one workgroup of 8 waves per CU
// (the kernels live in gemv_mfma.hip).
int launch_gemv_mfma(const KernelRef &v, const jitnn_hip_weight *w, const float *x, int rows, const float *bias, const Epilogue &e, float *y, hipStream_t stream) {
    if (int rc = allow_lds(v.fn, v.lds)) return rc;
    const int groups = (w->n + 15) / 16;
    const int blocks = groups < g.cus ? groups : g.cus;
    gemv_mfma_launch(w->fmt, (unsigned)blocks, stream, w->dev, x, bias, e, y, w->n, w->k, rows);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

// Formats without a tuned kernel for this row count (Q5_0 and Q3_K left as they are, Q5_1 and Q2_K at more than one row or in
// shapes the INT8 kernel does not take): one wave per row on the bit-exact decoder.
int launch_gemv_plain(const jitnn_hip_weight *w, const float *x, int rows, const float *bias, float *y, hipStream_t stream) {
    int blocks = (w->n + 3) / 4;
    if (blocks > g.cus * 8) blocks = g.cus * 8;
    typedef void (*fn_t)(const uint8_t *, const float *, const float *, float *, int, int, int);
    fn_t fn = w->fmt == F_Q5_0 ? gemv_plain_kernel<F_Q5_0> : w->fmt == F_Q5_1 ? gemv_plain_kernel<F_Q5_1> : w->fmt == F_Q2_K ? gemv_plain_kernel<F_Q2_K>
                                                                                                                             : gemv_plain_kernel<F_Q3_K>;
    hipLaunchKernelGGL(fn, dim3(blocks), dim3(256), 0, stream, w->dev, x, bias, y, w->n, w->k, rows);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

// The kernels of up to eight rows.  unmet: an epilogue that is asked for; cleared by the kernels that have one.
int launch_gemv(const jitnn_hip_weight *w, const float *x, int rows, const float *bias, float *y, hipStream_t stream, Epilogue *unmet = nullptr) {
    const Epilogue e = unmet ? *unmet : Epilogue{};
    auto met = [&]() {
        if (unmet) *unmet = Epilogue{};
        return e;
    };
    if (is_extra_format(w->fmt)) {
        if (rows == 1) {  // Q5_1 and Q2_K have units of the INT8 matrix-core kernel
            XregCall c;
            c.w[0] = w;
            c.y[0] = y;
            c.bias = bias;
            c.x = x;
            if (i8_ok(c)) {
                c.epi = met();
                return launch_i8(c, stream);
            }
        } else if (i8_batch_ok(w, rows < 4 ? rows : 4)) {
            // up to four rows per launch; more rows - where the one-pass kernel of gemv_rows.h does not take the shape (it has tiles
            // for both formats: 14336 x 4096 at 5..8 rows Q5_1 23 us, Q2_K 19 us against 28, 29 as two launches here) - as a chain of
            // such launches, each streaming the weights again
            met();
            for (int r0 = 0; r0 < rows; r0 += 4) {
                const Epilogue part{e.act, e.res ? e.res + (size_t)r0 * w->n : nullptr};
                if (int rc = launch_i8_batch(w, x + (size_t)r0 * w->k, rows - r0 < 4 ? rows - r0 : 4, bias, part, y + (size_t)r0 * w->n, stream)) return rc;
            }
            return JITNN_HIP_OK;
        }
        return launch_gemv_plain(w, x, rows, bias, y, stream);
    }
    if (i8_batch_ok(w, rows)) return launch_i8_batch(w, x, rows, bias, met(), y, stream);
    if (rows == 2 && w->k <= 4096) return launch_gemv_xreg_b2(w, x, bias, y, stream);
    // Q6_K pays the most per weight on the matrix-core path (6-bit quants from two arrays, 16-value scale groups): up to
    // four rows its FP32 kernel is still ahead (measured: 33 vs 43 us at 2 rows, 151 vs 167 us at 4 rows on the output head)
    if (rows >= (w->fmt == F_Q6_K ? 5 : 2) && rows <= 8 && w->k % 256 == 0 && w->n >= 16) {
        const KernelRef v = gemv_mfma_kernel_ref(w->fmt, e.any());
        if (v.fn && v.lds <= g.max_lds) return launch_gemv_mfma(v, w, x, rows, bias, met(), y, stream);
    }
    if (rows == 1 && e.any()) {
        XregCall c;
        c.w[0] = w;
        c.y[0] = y;
        c.bias = bias;
        c.x = x;
        if (i8_ok(c)) {
            c.epi = met();
            return launch_i8(c, stream);
        }
    }
    if (rows == 1) {
        if (w->k <= 4096) return launch_gemv_xreg(w, x, bias, y, stream);
        if (w->k <= 32768 && ksplit_lds(w->fmt, (w->k + 4095) / 4096) <= g.max_lds) return launch_gemv_ksplit(w, x, bias, y, stream);
    }
    GemvVariant v = pick(w->fmt, rows, w->k % 64 == 0);
    const int units = w->k / v.unit_values;
    const int steps = (units + 63) / 64;
    // stage as many steps as fit in 64 KiB (keeps several workgroups per CU); one step may need more
    int itc = (int)(65536 / v.lds_per_step);
    if (itc < 1) itc = 1;
    if (itc > steps) itc = steps;
    const size_t lds = v.lds_per_step * itc;
    if (lds > g.max_lds) return fail(JITNN_HIP_EINVAL, "GEMV needs %zu bytes of LDS, the device offers %zu", lds, g.max_lds);
    if (int rc = allow_lds((const void *)v.fn, lds)) return rc;
    // at least eight waves per CU: big LDS footprints leave room for one or two workgroups only, so those get 8 waves each
    int per_cu = (int)((g.lds_per_cu - 2048) / lds);
    if (per_cu < 1) per_cu = 1;
    if (per_cu > 4) per_cu = 4;
    const int threads = per_cu >= 2 ? 256 : 512, waves = threads / 64;
    const int groups = (w->n + v.R - 1) / v.R;
    int blocks = (groups + waves - 1) / waves;
    const int cap = g.cus * per_cu;
    if (blocks > cap) blocks = cap;
    hipLaunchKernelGGL(v.fn, dim3(blocks), dim3(threads), lds, stream, w->dev, x, bias, y, w->n, w->k, rows, itc, g.nib);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

// Per-thread device scratch for the many-row path.  It only grows; a call on another stream than the last one first waits
// for the previous user, so concurrent streams of one thread cannot overwrite each other's activations.  What a call needs
// of `operands` depends on its activations (and, where it splits K, on its outputs); dequantised weights, whose size also
// depends on the weight and whose use depends on the route, have a block of their own, so that neither moves the other.
// A block that a stream capture was given outlives its growth (scratch.h): a recorded graph keeps its address.
struct DeviceMem {
    static void *alloc(size_t bytes) {
        void *p = nullptr;
        if (hipMalloc(&p, bytes) == hipSuccess) return p;
        (void)hipGetLastError();
        return nullptr;
    }
    static bool release(void *p) {
        if (hipFree(p) == hipSuccess) return true;
        (void)hipGetLastError();
        return false;
    }
};
struct Workspace {
    ScratchBlock<DeviceMem> operands;  // FP16 activations and their row scales, partial sums of K slices
    ScratchBlock<DeviceMem> weights;   // dequantised weights of long prompts
    hipStream_t last = nullptr;
    hipEvent_t ev = nullptr;
    bool used = false;
};
thread_local Workspace g_ws;

bool stream_recording(hipStream_t stream) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream, &st) != hipSuccess) (void)hipGetLastError();
    return st != hipStreamCaptureStatusNone;
}

// Where a many-row launch takes its scratch from: the calling thread's grow-only buffer (may allocate), or the
// library's static array (never allocates; the caller keeps calls on one GPU from overlapping).
enum ScratchSource { SCRATCH_THREAD, SCRATCH_STATIC };
void touch_thread_state();  // registers the calling thread's clean-up (defined below ThreadState)

int workspace(size_t bytes, hipStream_t stream, void **out, ScratchSource src = SCRATCH_THREAD) {
    if (src == SCRATCH_STATIC) {
        if (bytes > JITNN_HIP_SCRATCH_BYTES)
            return fail(JITNN_HIP_EINVAL, "this call needs %zu bytes of scratch; the entry point that allocates nothing has %llu", bytes,
                        (unsigned long long)JITNN_HIP_SCRATCH_BYTES);
        *out = g.scratch_ptr;
        return JITNN_HIP_OK;
    }
    Workspace &w = g_ws;
    touch_thread_state();  // a thread that only ever calls the device-pointer entry points must give its scratch back too
    if (!w.ev) HIP_TRY(hipEventCreateWithFlags(&w.ev, hipEventDisableTiming));
    bool waited = false;
    const bool recording = stream_recording(stream);
    void *p = w.operands.get(bytes, recording, &waited);
    if (!p && w.weights.give_up(&waited)) p = w.operands.get(bytes, recording, &waited);  // (dequantised weights are a convenience)
    if (!p) return fail(JITNN_HIP_ENOMEM, "no %zu bytes of device memory for scratch", bytes);
    if (waited) w.used = false;
    if (w.used && w.last != stream) HIP_TRY(hipStreamWaitEvent(stream, w.ev, 0));
    *out = p;
    return JITNN_HIP_OK;
}

// Would workspace() give `bytes` where the caller can do with less: yes, unless it cannot hold them without an allocation under a
// stream capture, or at all.
bool workspace_at_hand(size_t bytes, hipStream_t stream, ScratchSource src) {
    if (src == SCRATCH_STATIC) return bytes <= JITNN_HIP_SCRATCH_BYTES;
    touch_thread_state();
    bool waited = false;
    void *p = g_ws.operands.try_get(bytes, stream_recording(stream), &waited);
    if (waited) g_ws.used = false;
    return p != nullptr;
}

// Room for `bytes` of dequantised weights, or nullptr - without an error, and without a word to the device where that size was
// refused before: the caller then takes the kernel that decodes them as it goes, which needs none.  Between workspace(), which
// orders both blocks on the stream (and may give this one up), and the launches.
_Float16 *weight_room(size_t bytes, hipStream_t stream) {
    bool waited = false;
    void *p = g_ws.weights.try_get(bytes, stream_recording(stream), &waited);
    if (waited) g_ws.used = false;
    return (_Float16 *)p;
}

int workspace_done(hipStream_t stream, ScratchSource src = SCRATCH_THREAD) {
    if (src == SCRATCH_STATIC) return JITNN_HIP_OK;
    Workspace &w = g_ws;
    HIP_TRY(hipEventRecord(w.ev, stream));
    w.last = stream;
    w.used = true;
    return JITNN_HIP_OK;
}

// Per-thread staging of the host-pointer entry points (jitnn_hip_linear, _dequantize, _quantize_q8_0, the model steps
// on host buffers): a pinned host buffer, a device buffer and a stream, all grow-only, so that a call costs copies and
// launches but no allocation.  Buffers beyond STAGE_KEEP_MAX are not kept (a dequantised matrix goes through in pieces).
constexpr size_t STAGE_KEEP_MAX = (size_t)128 << 20;
// 16-byte pieces from one buffer to another; one side is pinned host memory as the device sees it.  For the few KB of a
// GEMV call a launch costs less than a DMA transfer's set-up, and the bytes cross the bus in whole lines.
__global__ void __launch_bounds__(256) stage_copy_kernel(uint4 *__restrict__ dst, const uint4 *__restrict__ src, size_t count16) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < count16; i += (size_t)gridDim.x * 256) dst[i] = src[i];
}
constexpr size_t STAGE_KERNEL_COPY_MAX = (size_t)1 << 20;  // above this a DMA transfer is as fast and leaves the compute units alone

struct HostStage {
    uint8_t *pinned = nullptr, *dev = nullptr;
    uint8_t *pinned_dev = nullptr;  // the pinned buffer's address on the device
    size_t pcap = 0, dcap = 0;
    hipStream_t stream = nullptr;
    void release() {
        if (pinned) (void)hipHostFree(pinned);
        if (dev) (void)hipFree(dev);
        if (stream) (void)hipStreamDestroy(stream);
        pinned = dev = pinned_dev = nullptr;
        pcap = dcap = 0;
        stream = nullptr;
    }
};
void release_workspace() {
    Workspace &w = g_ws;
    w.operands.release_all();
    w.weights.release_all();
    if (w.ev) (void)hipEventDestroy(w.ev);
    w = Workspace{};
}
struct ThreadState {
    HostStage stage;
    // A thread that ends gives its device memory back.  The process's first thread ends with the process, when the HIP
    // runtime may already be gone: its buffers are left to the process teardown.
    ~ThreadState() {
        if (is_main) return;
        stage.release();
        release_workspace();
    }
    bool is_main = false;
};
thread_local ThreadState g_thread;
bool calling_thread_is_main();
void touch_thread_state() { g_thread.is_main = calling_thread_is_main(); }

int stage_reserve(size_t pinned_bytes, size_t dev_bytes) {
    HostStage &st = g_thread.stage;
    g_thread.is_main = calling_thread_is_main();
    if (!st.stream) HIP_TRY(hipStreamCreateWithFlags(&st.stream, hipStreamNonBlocking));
    auto round = [](size_t b) { return (b + ((size_t)1 << 16) - 1) & ~(((size_t)1 << 16) - 1); };
    if (pinned_bytes > st.pcap) {
        if (st.pinned) HIP_TRY(hipHostFree(st.pinned));
        st.pinned = st.pinned_dev = nullptr;
        st.pcap = 0;
        const size_t want = round(pinned_bytes);
        hipError_t e = hipHostMalloc((void **)&st.pinned, want, hipHostMallocDefault);
        if (e != hipSuccess) return fail(JITNN_HIP_ENOMEM, "hipHostMalloc of %zu bytes of staging: %s", want, hipGetErrorString(e));
        st.pcap = want;
        if (hipHostGetDevicePointer((void **)&st.pinned_dev, st.pinned, 0) != hipSuccess) {
            (void)hipGetLastError();
            st.pinned_dev = nullptr;  // not mapped: the DMA path is used
        }
    }
    if (dev_bytes > st.dcap) {
        if (st.dev) HIP_TRY(hipFree(st.dev));
        st.dev = nullptr;
        st.dcap = 0;
        const size_t want = round(dev_bytes);
        hipError_t e = hipMalloc((void **)&st.dev, want);
        if (e != hipSuccess) return fail(JITNN_HIP_ENOMEM, "hipMalloc of %zu bytes of staging: %s", want, hipGetErrorString(e));
        st.dcap = want;
    }
    return JITNN_HIP_OK;
}

// ---- more than 512 rows: weights dequantised into operand order first, then a plain FP16 product (prefill_wide.h)

// The weight rows of a tile (32 rt) and the microseconds the product should take: whole rounds of one tile per CU, each
// `step` per 32 values of K and `fixed` for its prologue and epilogue (measured on whole rounds: 4096 x 4096 x 4096 tokens
// takes 110 us with rt 8, one round, and 125 with rt 4, two; 6144 x 4096 x 4096 takes 174 with rt 6 against 197 with rt 8).
struct WidePlan {
    int rt = 0, tiles_n = 0;
    double us = 0;
};
WidePlan wide_plan(const int *n, int count, int k, int mtiles, bool dual, int cus) {
    static const struct { int rt; double step, fixed; } kinds[] = {{8, 0.78, 10.0}, {6, 0.59, 8.0}, {4, 0.44, 5.0}};
    WidePlan best;
    const int nst = pf_ksteps(k) / 2;
    for (const auto &kind : kinds) {
        if (dual && kind.rt != 8) break;
        const int tn = dual ? 16 * kind.rt : 32 * kind.rt;
        int tiles = 0;
        for (int i = 0; i < count; ++i) tiles += (n[i] + tn - 1) / tn;
        const int rounds = (int)(((long long)tiles * mtiles + cus - 1) / cus);
        const double us = rounds * (kind.step * nst + kind.fixed);
        if (!best.rt || us < best.us) best = {kind.rt, tiles, us};
    }
    return best;
}

// Dequantised weights beyond this stay on the kernel that decodes as it goes.
constexpr size_t WIDE_MAX_BYTES = (size_t)512 << 20;
size_t wide_weight_bytes(const WidePlan &p, int k) { return (size_t)p.tiles_n * p.rt * pf_ksteps(k) * 1024; }
// what the activations of a many-row linear take as operands, and their row scales behind them
size_t operand_bytes(int rows, int k) { return (size_t)(rows + PF_BM - 1) / PF_BM * (PF_BM / 32) * pf_ksteps(k) * 1024; }
size_t row_scale_bytes(int rows) { return ((size_t)rows * 8 + 255) & ~(size_t)255; }

// Whether `count` weights of one row length (dual: a gate and an up weight) are worth dequantising first for `rows` rows:
// the estimate of both passes against that of prefill_mfma_kernel, which takes rounds of 128-row tiles (dual: 64 rows of each
// weight) by 256 tokens at `step` us per 64 values of K.  Measured, both routes, activation preparation included (us):
// 14336 x 4096 Q4_K, 1024 / 2048 / 4096 rows 139 / 262 / 490 there and 140 / 254 / 489 here; 4096 x 14336 Q6_K 159 / 277 / 555
// and 232 / 290 / 478; 4096 x 4096 Q4_K 57 / 84 / 160 and 68 / 85 / 140; Q8_0 63 / 90 / 171 and 69 / 86 / 141; 11008 x 4096 Q4_0 122 / 199 / 398
// and 112 / 205 / 375.  (The steps of Q4_K, Q6_K and Q8_0 are older than the kernel there: they were fitted when its barrier stood between two
// steps.  Where that errs: Q6_K 4096 x 14336 at 2048 rows is taken here, and Q8_0 4096 x 4096 is not.)
// Up to 1024 rows Q4_0, Q4_1 and Q5_K have the steps that lost least on 326 linears and 61 prompts of 4 layers, timed with both routes since
// prefill_mfma_kernel decodes them in packed FP16 under its products (beyond, where only whole prompts were timed, 1.06 stands): Q4_0 linears
// 0.5 % behind the faster route in the mean and not 1.3.  Of Q4_0, here -> there: 4352 x 12800 at 886 rows 172 -> 148 us, 14336 x 4096 at 900
// 140 -> 128, 800 tokens of four 4096-wide layers 2244 -> 2136; Q5_K 14336 x 4096 at 1024 rows is level, 137 us.
// Two tiles of tokens or fewer, short rows of K and launches that split K lose here, whatever the estimate (1024 x 4096 at 1024 36 and 63; at 1024 values it turns, 8448 x 1024 at 2048 rows 72 and 69, at 4096 120 and 102), and the
// estimate is good to a tenth on short launches: the margins.  For the 8B gate / up pair it errs against this route: with the margin it is
// taken at 2049 - 2304, 2561 - 2816, 3073 - 3328 and 3585 - 4096 rows, where the product's last round is full enough (whole prompts, us per layer,
// there / here: 2304 tokens 1275 / 1225, 2816 1513 / 1438, 3328 1774 / 1664, 4096 2081 / 1950), and not wherever it would win (1300 919 / 889, 1536
// 949 / 932, 2560 1379 / 1341, 3072 1655 / 1595; level at 1792 and 2048, 51, 7 and 11 us slower at 600, 800 and 1024).
// residual: prefill_mfma_kernel leaves it to add_rows_kernel (12 bytes per output at 6.5 TB/s: 31 us for 4096 x 4096), the wide
// kernel adds it as it stores: 4096 x 4096 Q4_K at 4096 rows 143 + 31 us there, 127 + 8 here.
bool wide_pays(const int *fmt, const int *rows_of, int count, int k, int rows, bool dual, bool residual, int cus, WidePlan *plan) {
    if (count > 3 || rows <= 2 * PF_BM || k < 1024) return false;
    const int mtiles = (rows + PF_BM - 1) / PF_BM, nsteps = (k + PF_BK - 1) / PF_BK;
    int n[3] = {0, 0, 0}, tiles = 0;
    double dequant = 0, step = 0;
    for (int i = 0; i < count; ++i) {
        const int f = fmt[i];
        if (!has_many_row_kernel(f)) return false;
        if (i == 0 || !dual) n[i] = rows_of[i];
        tiles += (rows_of[i] + PF_BN - 1) / PF_BN;
        dequant += 3.0 + (f == F_Q6_K ? 0.62e-6 : 0.45e-6) * rows_of[i] * (double)k;
        step = std::max(step, f == F_Q4_K ? 0.87 : f == F_Q6_K ? 1.17 : rows > 1024 ? 1.06 : f == F_Q4_0 ? 0.92 : f == F_Q4_1 || f == F_Q5_K ? 0.98 : 1.06);
    }
    *plan = wide_plan(n, dual ? 1 : count, k, mtiles, dual, cus);
    if (wide_weight_bytes(*plan, k) > WIDE_MAX_BYTES) return false;
    if ((long long)tiles * mtiles * 2 <= cus) return false;
    const double decoding = (double)(((long long)tiles * mtiles + cus - 1) / cus) * (step * nsteps + 10.0) + (residual ? 12.0 / 6.5e6 * rows * n[0] : 0.0);
    return plan->us + dequant < (decoding > 150.0 ? 0.95 : rows > 1024 ? 0.9 : 0.8) * decoding;
}
bool wide_pays(const jitnn_hip_weight *const *ws, int count, int rows, bool dual, bool residual, WidePlan *plan) {
    int fmt[3], n[3];
    if (count > 3) return false;
    for (int i = 0; i < count; ++i) {
        if (ws[i]->k != ws[0]->k) return false;
        fmt[i] = ws[i]->fmt;
        n[i] = ws[i]->n;
    }
    return wide_pays(fmt, n, count, ws[0]->k, rows, dual, residual, g.cus, plan);
}

// The arguments are those of launch_prefill_group; dual: ws is a gate and an up weight, ys[0] = silu(x gate^T) * (x up^T).
// WIDE_NO_ROOM: nothing was launched, there is no memory for the dequantised weights.
constexpr int WIDE_NO_ROOM = 1;
int launch_prefill_wide(const WidePlan &plan, const jitnn_hip_weight *const *ws, float *const *ys, int count, bool dual, const float *x, int rows,
                        const float *bias, const float *norm_w, float eps, hipStream_t stream, const float *residual, const float *swiglu_up,
                        const PfPending *pend) {
    const KernelRef kr = prefill_wide_kernel_ref(dual, plan.rt);
    if (!kr.fn) return fail(JITNN_HIP_EUNSUPPORTED, "no wide kernel of %d row blocks", plan.rt);
    if (int rc = allow_lds(kr.fn, kr.lds)) return rc;
    const int k = ws[0]->k, ksteps = pf_ksteps(k), tn = dual ? 16 * plan.rt : 32 * plan.rt;
    PwArgs a{};
    a.tiles_m = (rows + PF_BM - 1) / PF_BM;
    a.tiles_n = plan.tiles_n;
    a.m = rows;
    a.ksteps = ksteps;
    const int mblocks = a.tiles_m * (PF_BM / 32);
    const size_t xo_bytes = operand_bytes(rows, k);
    void *wsp = nullptr;
    if (int rc = workspace(xo_bytes + row_scale_bytes(rows), stream, &wsp)) return rc;
    _Float16 *xo = (_Float16 *)wsp, *wo = weight_room(wide_weight_bytes(plan, k), stream);
    if (!wo) return WIDE_NO_ROOM;
    float *scale = (float *)((uint8_t *)wsp + xo_bytes), *inv = scale + rows;
    a.wo = wo;
    a.xo = xo;
    a.inv_scale = inv;
    a.bias = bias;
    a.res = residual;
    int tile = 0;
    for (int i = 0; i < 3; ++i) {
        a.tile0[i] = tile;
        if (i >= (dual ? 1 : count)) continue;
        a.y[i] = ys[i];
        a.n[i] = ws[i]->n;
        _Float16 *dst = wo + (size_t)tile * plan.rt * ksteps * 512;
        wide_dequant_launch(ws[i]->fmt, stream, ws[i]->dev, dst, ws[i]->n, k, dual ? 0 : -1);
        if (dual) wide_dequant_launch(ws[1]->fmt, stream, ws[1]->dev, dst, ws[1]->n, k, 1);
        tile += (ws[i]->n + tn - 1) / tn;
    }
    prefill_prepare_launch(x, scale, inv, xo, rows, k, mblocks, norm_w, eps, swiglu_up, stream, pend);
    prefill_wide_launch(dual, plan.rt, stream, a);
    HIP_TRY(hipGetLastError());
    return workspace_done(stream);
}

// Whole tiles for every compute unit, or K in slices that a second kernel adds up: how many (1 to 8) a single weight of the kernel that
// decodes as it goes takes.  The estimate, in us: whole rounds of workgroups at 0.4 + `step` per 64 values of K (three quarters of it where
// the narrow wave layout serves up to 128 rows), the slices' way to memory and back, and their join - a launch of its own unless the
// next kernel reads them.  Fitted on 116 launches of six formats (256 to 18000 rows of 512 to 14336 values, 65 to 1000 activation
// rows) at 1 to 8 slices: 6 % off in the mean, and its choice 0.4 % slower than the best count, where doubling the slices as long as they
// fit the device twice over was 4.1 %.  Q8_0 8704 x 6592 at 170 rows 61.6 -> 49.8 us (three slices, not two), Q6_K 3074 x 12544 at 711 rows
// 115.8 -> 96.7.  A device that whole tiles keep more than half busy slows its clock when the rest joins in: there the estimate has to see 8 %
// (90 launches of 101 to 255 tiles: 0.26 % behind the best count, at worst 2.1, where 2 % gave 0.32 and 5.8; Q4_K 9472 x 6144 at
// 361 rows 86 us in three slices, 83 whole; Q6_K 6912 deep, 8495 at 323, 104 -> 97 in three).
double many_row_step_us(int fmt) {
    switch (fmt) {
    case F_Q4_0: case F_Q4_K: return 0.68;
    case F_Q5_K: return 0.79;
    case F_Q4_1: case F_Q8_0: return 0.82;
    default: return 0.91;
    }
}
int many_row_slices(int fmt, int n, int k, int rows, bool joined_by_reader, int cus) {
    const int tiles = (n + PF_BN - 1) / PF_BN * ((rows + PF_BM - 1) / PF_BM), nsteps = (k + PF_BK - 1) / PF_BK, unit = block_values(fmt) == 256 ? 4 : 1;
    const double step = many_row_step_us(fmt) * (rows <= PF_NARROW_ROWS ? 0.72 : 1.0), mb = 4e-6 * rows * n;
    int best = 1;
    double best_us = 0;
    for (int s = 1; s <= 8; ++s) {
        const int each = ((nsteps + s - 1) / s + unit - 1) / unit * unit;
        if (s > 1 && (each < 2 || (nsteps + each - 1) / each != s)) continue;  // (a count that whole blocks leave slices empty)
        const int rounds = (int)(((long long)tiles * s + cus - 1) / cus);
        const double us = rounds * (0.4 + step * each) + (s > 1 ? 0.4 * s * mb + (joined_by_reader ? 0.5 : 4.0) : 0.2 * mb);
        if (best_us == 0 || us < (best > 1 ? 1.0 : 2 * tiles > cus ? 0.92 : 0.98) * best_us) {
            best = s;
            best_us = us;
        }
    }
    return best;
}

// More rows than the GEMV kernels take: FP16 activations in operand order + dequantise-to-LDS MFMA kernel.
// `count` weights of one row length share the activations x [rows, k] (prepared once): ys[i] = x ws[i]^T (+ bias, one
// weight only).  norm_w != nullptr: the RMSNorm in front of the linears is fused into the preparation (rows of at most
// XP_MAXK values; the caller checks with prefill_prepare_fuses_norm).
// residual != nullptr (one weight only): y = residual + x w^T, added by the join of the K slices, or, for a launch that
// does not split K, by a pass of its own over the product left in `tmp` [rows, n].
// part_ext / defer (one weight with a residual): the K slices go to part_ext ([8][rows, n] floats, the caller's) and, when the
// launch does split K, their join is left to the caller - *defer describes it, and the activation preparation of the next
// linears can do it on the way (pend: this call's activations are that pending row, not x).
int launch_prefill_group(const jitnn_hip_weight *const *ws, float *const *ys, int count, const float *x, int rows, const float *bias,
                         const float *norm_w, float eps, hipStream_t stream, const float *residual = nullptr, float *tmp = nullptr,
                         const float *swiglu_up = nullptr, ScratchSource src = SCRATCH_THREAD, float *part_ext = nullptr, PfPending *defer = nullptr,
                         const PfPending *pend = nullptr, PfGroupPending *gdefer = nullptr) {
    // (the kernels live in prefill_k.hip, prefill_q32.hip and prefill_mixed.hip)
    // Weights of one format - and a run of one K-quant format followed by a run of another for which a two-format kernel
    // exists - share a launch: their row tiles are numbered one after the other, so that the 1024-row k and v projections
    // fill the device together with q instead of splitting K eight ways each.
    struct Launch {
        int first, count, first_b;  // weights [first, first + count); first_b: where the second format starts (count: one format)
        int splits[3], split_steps[3];
        size_t part_bytes;
    } launch[4];
    int nlaunch = 0;
    if (count < 1 || count > 4) return fail(JITNN_HIP_EINVAL, "%d weights on one activation", count);
    if (residual && (count != 1 || !tmp || ws[0]->n % 4 != 0)) return fail(JITNN_HIP_EINVAL, "a residual needs one weight, rows of whole quads and a buffer");
    const int k = ws[0]->k;
    WidePlan plan;
    const bool wide = wide_pays(ws, count, rows, false, residual != nullptr, &plan);
    if (wide && src == SCRATCH_THREAD) {
        const int rc = launch_prefill_wide(plan, ws, ys, count, false, x, rows, bias, norm_w, eps, stream, residual, swiglu_up, pend);
        if (rc != WIDE_NO_ROOM) return rc;
    }
    const int mtiles = (rows + PF_BM - 1) / PF_BM, mblocks = mtiles * (PF_BM / 32);  // operands padded to whole tiles of tokens
    const int nsteps = (k + PF_BK - 1) / PF_BK;
    auto kq = [](const jitnn_hip_weight *w) { return block_values(w->fmt) == 256; };
    auto tiles_of = [](const jitnn_hip_weight *w) { return (w->n + PF_BN - 1) / PF_BN; };
    for (int i = 0; i < count; ++i) {
        const jitnn_hip_weight *w = ws[i];
        if (w->k != k) return fail(JITNN_HIP_EINVAL, "weights of %d and %d values per row on one activation", k, w->k);
        const KernelRef kr = kq(w) ? prefill_kernel_k(w->fmt) : prefill_kernel_q32(w->fmt);
        if (!kr.fn) return fail(JITNN_HIP_EUNSUPPORTED, "no many-row kernel for format %d", w->fmt);
        if (int rc = allow_lds(kr.fn, kr.lds)) return rc;
    }
    for (int i = 0; i < count;) {
        Launch &l = launch[nlaunch++];
        l.first = i;
        int j = i + 1;
        const bool joinable = !bias && !residual;  // (several weights: partial sums of all of them are joined by one kernel)
        while (joinable && j < count && j - i < 3 && ws[j]->fmt == ws[i]->fmt && ws[j]->n % 4 == 0 && ws[i]->n % 4 == 0) ++j;
        l.first_b = j - i;
        if (joinable && j < count && j - i < 3 && ws[j]->fmt != ws[i]->fmt && ws[i]->n % 4 == 0 && ws[j]->n % 4 == 0) {
            const KernelRef kr = prefill_kernel_mixed(ws[i]->fmt, ws[j]->fmt);
            if (kr.fn) {
                if (int rc = allow_lds(kr.fn, kr.lds)) return rc;
                const int fb = ws[j]->fmt;
                while (j < count && j - i < 3 && ws[j]->fmt == fb && ws[j]->n % 4 == 0) ++j;
            }
        }
        l.count = j - i;
        int tiles = 0;
        size_t nsum = 0;
        for (int q = i; q < j; ++q) {
            tiles += tiles_of(ws[q]);
            nsum += (size_t)ws[q]->n;
        }
        // A launch that would leave CUs idle (few, large tiles) splits K: every slice writes its own partial y, a second kernel - or
        // the one that reads y next - adds the slices in order.  Several weights: twice as many slices as long as those fit the device twice.
        int splits = 1;
        if (nsum % 4 == 0 && ws[i]->n % 4 == 0) {
            while (splits < 8 && tiles * mtiles * splits * 2 <= g.cus && nsteps / (splits * 2) >= PREFILL_MIN_SLICE) splits *= 2;
        }
        if (l.count == 1 && !wide) {  // (wide: the bits of the kernel that this one stands in for)
            // One weight, with scratch to spare: the count that the estimate likes best, for outputs of any length.  (The same limit for both
            // sources of scratch, so that both entry points give the same bits; a stream capture that finds less at hand keeps the count above.)
            const int want = many_row_slices(ws[i]->fmt, ws[i]->n, k, rows, defer != nullptr, g.cus);
            const size_t need = operand_bytes(rows, k) + row_scale_bytes(rows) + (want > 1 ? (size_t)want * rows * ws[i]->n * 4 : 0);
            if (need <= JITNN_HIP_SCRATCH_BYTES && workspace_at_hand(need, stream, src)) splits = want;
        }
        int wgs = tiles * mtiles * splits;
        l.part_bytes = 0;
        for (int q = 0; q < l.count; ++q) {
            const jitnn_hip_weight *wq = ws[i + q];
            l.splits[q] = splits;
            // the second format of a two-format launch (Q6_K beside Q4_K or Q5_K) takes half as long again per step: its
            // tiles get slices half as long where the device has the room, so that the launch does not wait for them
            if (q >= l.first_b && splits > 1 && splits < 8 && wgs + tiles_of(wq) * mtiles * splits <= g.cus && nsteps / (splits * 2) >= PREFILL_MIN_SLICE) {
                l.splits[q] = splits * 2;
                wgs += tiles_of(wq) * mtiles * splits;
            }
            // slices of the 256-value formats start on whole blocks (four steps): the kernel stages their raw bytes by block
            l.split_steps[q] = (nsteps + l.splits[q] - 1) / l.splits[q];
            if (kq(wq)) l.split_steps[q] = (l.split_steps[q] + 3) & ~3;
            if (l.splits[q] > 1) l.part_bytes += (size_t)l.splits[q] * rows * wq->n * 4;
        }
        i = j;
    }
    size_t part_max = 0;
    for (int i = 0; i < nlaunch; ++i) part_max = std::max(part_max, launch[i].part_bytes);
    const size_t xo_bytes = operand_bytes(rows, k), scale_bytes = row_scale_bytes(rows);
    void *wsp = nullptr;
    if (int rc = workspace(xo_bytes + scale_bytes + part_max, stream, &wsp, src)) return rc;
    _Float16 *xo = (_Float16 *)wsp;
    float *scale = (float *)((uint8_t *)wsp + xo_bytes), *inv = scale + rows;
    float *part = part_ext && count == 1 && residual ? part_ext : (float *)((uint8_t *)wsp + xo_bytes + scale_bytes);
    prefill_prepare_launch(x, scale, inv, xo, rows, k, mblocks, norm_w, eps, swiglu_up, stream, pend);
    for (int li = 0; li < nlaunch; ++li) {
        const Launch &l = launch[li];
        const jitnn_hip_weight *w = ws[l.first];
        const bool split = l.splits[0] > 1;  // (the segments of a launch split together or not at all)
        PfSegments sg{}, out{};
        for (int q = 0; q < 3; ++q) sg.splits[q] = out.splits[q] = 1;
        size_t before = 0;  // floats of partial sums of the segments before this one
        unsigned gx = 0;
        for (int q = 0; q < l.count; ++q) {
            const jitnn_hip_weight *wq = ws[l.first + q];
            sg.W[q] = wq->dev;
            sg.n[q] = wq->n;
            sg.tiles[q] = tiles_of(wq);
            sg.splits[q] = l.splits[q];
            sg.split_steps[q] = l.split_steps[q];
            sg.y[q] = split ? part + before : (residual ? tmp : ys[l.first + q]);
            before += (size_t)l.splits[q] * rows * wq->n;
            gx += (unsigned)(sg.tiles[q] * sg.splits[q]);
            out.y[q] = ys[l.first + q];
            out.n[q] = wq->n;
            out.splits[q] = l.splits[q];
        }
        const float *b1 = split ? nullptr : bias;
        const dim3 grid(gx, mtiles);
        if (l.first_b < l.count) prefill_launch_mixed(w->fmt, ws[l.first + l.first_b]->fmt, l.first_b, grid, stream, sg, xo, inv, rows, k);
        else if (kq(w)) prefill_launch_k(w->fmt, grid, stream, sg, xo, inv, b1, rows, k);
        else prefill_launch_q32(w->fmt, grid, stream, sg, xo, inv, b1, rows, k);
        if (split && l.count > 1 && gdefer && nlaunch == 1) {
            // the caller's next kernel adds the slices up as it reads them (they stay in this thread's scratch until its
            // next many-row call)
            gdefer->part = part;
            gdefer->sg = out;
        } else if (split && l.count > 1) {  // (the stream orders the next launch's partial sums after this join)
            size_t count4 = 0;
            for (int q = 0; q < l.count; ++q) count4 += (size_t)rows * sg.n[q] / 4;
            const unsigned blocks = (unsigned)std::min<size_t>((count4 + 255) / 256, (size_t)g.cus * 8);
            prefill_join_group_launch(part, out, rows, blocks, stream);
        } else if (split && defer && part == part_ext && !bias) {  // the join rides with the next activation preparation
            defer->part = part;
            defer->res = residual;
            defer->out = ys[l.first];
            defer->splits = l.splits[0];
            defer->n = w->n;
        } else if (split) {
            prefill_join_launch(part, bias, residual, ys[l.first], rows, w->n, l.splits[0], (unsigned)g.cus * 8, stream);
        } else if (residual) {
            const size_t count4 = (size_t)rows * w->n / 4;
            const unsigned blocks = (unsigned)std::min<size_t>((count4 + 255) / 256, (size_t)g.cus * 8);
            hipLaunchKernelGGL(add_rows_kernel, dim3(blocks), dim3(256), 0, stream, reinterpret_cast<const float4 *>(tmp),
                               reinterpret_cast<const float4 *>(residual), reinterpret_cast<float4 *>(ys[l.first]), count4);
        }
    }
    HIP_TRY(hipGetLastError());
    return workspace_done(stream, src);
}

// h [rows, n] = silu(n(x) gate^T) * (n(x) up^T), n = RMSNorm with norm_w (which must fit the fused preparation): the gate
// and the up projection of a Llama FFN as one product whose epilogue forms the SwiGLU - the two [rows, n] products are
// neither stored nor read back.  pend: as in launch_prefill_group.
bool prefill_dual_ok(const jitnn_hip_weight *gate, const jitnn_hip_weight *up) {
    return gate->fmt == up->fmt && gate->n == up->n && gate->k == up->k && !is_extra_format(gate->fmt) &&
           prefill_prepare_fuses_norm(gate->k);
}

int launch_prefill_dual(const jitnn_hip_weight *gate, const jitnn_hip_weight *up, float *h, const float *x, int rows, const float *norm_w, float eps,
                        hipStream_t stream, const PfPending *pend) {
    const jitnn_hip_weight *const pair[2] = {gate, up};
    WidePlan plan;
    if (wide_pays(pair, 2, rows, true, false, &plan)) {
        const int rc = launch_prefill_wide(plan, pair, &h, 2, true, x, rows, nullptr, norm_w, eps, stream, nullptr, nullptr, pend);
        if (rc != WIDE_NO_ROOM) return rc;
    }
    const bool kq = block_values(gate->fmt) == 256;
    const KernelRef kr = kq ? prefill_kernel_dual_k(gate->fmt) : prefill_kernel_dual_q32(gate->fmt);
    if (!kr.fn) return fail(JITNN_HIP_EUNSUPPORTED, "no many-row kernel for format %d", gate->fmt);
    if (int rc = allow_lds(kr.fn, kr.lds)) return rc;
    const int k = gate->k, n = gate->n;
    const int mtiles = (rows + PF_BM - 1) / PF_BM, mblocks = mtiles * (PF_BM / 32);
    const size_t xo_bytes = operand_bytes(rows, k), scale_bytes = row_scale_bytes(rows);
    void *wsp = nullptr;
    if (int rc = workspace(xo_bytes + scale_bytes, stream, &wsp, SCRATCH_THREAD)) return rc;
    _Float16 *xo = (_Float16 *)wsp;
    float *scale = (float *)((uint8_t *)wsp + xo_bytes), *inv = scale + rows;
    prefill_prepare_launch(x, scale, inv, xo, rows, k, mblocks, norm_w, eps, nullptr, stream, pend);
    const dim3 grid((unsigned)((n + PF_BN / 2 - 1) / (PF_BN / 2)), mtiles);
    if (kq) prefill_launch_dual_k(gate->fmt, grid, stream, gate->dev, up->dev, xo, inv, h, rows, n, k);
    else prefill_launch_dual_q32(gate->fmt, grid, stream, gate->dev, up->dev, xo, inv, h, rows, n, k);
    HIP_TRY(hipGetLastError());
    return workspace_done(stream, SCRATCH_THREAD);
}

int launch_prefill(const jitnn_hip_weight *w, const float *x, int rows, const float *bias, float *y, hipStream_t stream,
                   ScratchSource src = SCRATCH_THREAD) {
    return launch_prefill_group(&w, &y, 1, x, rows, bias, nullptr, 0.f, stream, nullptr, nullptr, nullptr, src);
}

template <int FMT>
void launch_dequant(const jitnn_hip_weight *w, float *y, hipStream_t stream) {
    const size_t quads = (size_t)w->n * w->k / 4;
    size_t blocks = (quads + 255) / 256;
    const size_t cap = (size_t)g.cus * 16;
    if (blocks > cap) blocks = cap;
    if (quads * sizeof(float4) > DQ_STREAM_BYTES) hipLaunchKernelGGL((dequant_kernel<FMT, true>), dim3((unsigned)blocks), dim3(256), 0, stream, w->dev, y, quads);
    else hipLaunchKernelGGL((dequant_kernel<FMT, false>), dim3((unsigned)blocks), dim3(256), 0, stream, w->dev, y, quads);
}

int check_weight_args(int fmt, long long nbytes, int n, int k, const void *blocks, jitnn_hip_weight **out) {
    if (!out) return fail(JITNN_HIP_EINVAL, "out is NULL");
    *out = nullptr;
    if (!blocks) return fail(JITNN_HIP_EINVAL, "blocks is NULL");
    long long need = jitnn_hip_weight_nbytes(fmt, n, k);
    if (need < 0) return (int)need;
    if (nbytes != need)
        return fail(JITNN_HIP_EINVAL, "format %d weight of shape [%d, %d] needs %lld bytes, got %lld", fmt, n, k, need, nbytes);
    return JITNN_HIP_OK;
}

}  // namespace

// ================================================================================================ C ABI

extern "C" {

const char *jitnn_hip_last_error(void) { return g_err; }

int jitnn_hip_block_values(int fmt) { return block_values(fmt); }
int jitnn_hip_block_bytes(int fmt) { return block_bytes(fmt); }

long long jitnn_hip_weight_nbytes(int fmt, long long n, long long k) {
    if (!known(fmt)) return fail(JITNN_HIP_EINVAL, "ggml type id %d is not one of Q4_0, Q4_1, Q5_0, Q5_1, Q8_0, Q2_K, Q3_K, Q4_K, Q5_K, Q6_K", fmt);
    if (n < 1 || k < 1) return fail(JITNN_HIP_EINVAL, "weight shape [%lld, %lld] is empty", n, k);
    if (k % block_values(fmt) != 0)
        return fail(JITNN_HIP_EINVAL, "format %d weight of shape [%lld, %lld]: last axis not a multiple of its block of %d", fmt, n, k,
                    block_values(fmt));
    if (n > 0x7fffffffLL || k > 0x7fffffffLL || n * k > 0x7fffffffLL)  // the reference's tensors hold at most Integer.MAX_VALUE values
        return fail(JITNN_HIP_EINVAL, "weight shape [%lld, %lld] holds more than 2^31-1 values", n, k);
    return n * (k / block_values(fmt)) * block_bytes(fmt);
}

int jitnn_hip_init(int device_ordinal) {
    std::lock_guard<std::mutex> lock(g_mu);
    if (g.ready) {
        if (device_ordinal != g.device) return fail(JITNN_HIP_EINVAL, "already initialised on device %d", g.device);
        return JITNN_HIP_OK;
    }
    int count = 0;
    hipError_t e = hipGetDeviceCount(&count);
    if (e != hipSuccess || count == 0) return fail(JITNN_HIP_ENODEVICE, "no HIP device: %s", hipGetErrorString(e));
    if (device_ordinal < 0 || device_ordinal >= count) return fail(JITNN_HIP_EINVAL, "device %d of %d", device_ordinal, count);
    HIP_TRY(hipSetDevice(device_ordinal));
    hipDeviceProp_t p;
    HIP_TRY(hipGetDeviceProperties(&p, device_ordinal));
    if (strncmp(p.gcnArchName, "gfx950", 6) != 0)
        return fail(JITNN_HIP_ENODEVICE, "device %d is %s; this library holds gfx950 code only", device_ordinal, p.gcnArchName);
    snprintf(g.name, sizeof g.name, "%s (%s)", p.name, p.gcnArchName);
    g.cus = p.multiProcessorCount;
    g.hbm = (long long)p.totalGlobalMem;
    int optin = 0;
    if (hipDeviceGetAttribute(&optin, hipDeviceAttributeSharedMemPerBlockOptin, device_ordinal) != hipSuccess || optin <= 0)
        optin = (int)p.sharedMemPerBlock;
    g.max_lds = (size_t)optin;
    g.lds_per_cu = p.maxSharedMemoryPerMultiProcessor > 0 ? (size_t)p.maxSharedMemoryPerMultiProcessor : g.max_lds;
    float *probe = nullptr;
    HIP_TRY(hipMalloc(&probe, 2 * sizeof(float)));
    hipLaunchKernelGGL(fp8_probe_kernel, dim3(1), dim3(1), 0, 0, probe);
    float h[2] = {0, 0};
    hipError_t ce = hipMemcpy(h, probe, sizeof h, hipMemcpyDeviceToHost);
    (void)hipFree(probe);
    if (ce != hipSuccess) return fail(JITNN_HIP_EDEVICE, "fp8 probe: %s", hipGetErrorString(ce));
    if (!(h[0] > 0.f) || h[1] != 15.f * h[0])
        return fail(JITNN_HIP_EDEVICE, "fp8 probe: E4M3 bytes 0x01, 0x0f decode to %g, %g; expected q * 2^-9 or q * 2^-10", h[0], h[1]);
    g.nib = 1.f / h[0];
    {   // the device address of the static scratch on this GPU (every GPU holds its own copy at its own address)
        void *sp = nullptr;
        hipError_t se = hipGetSymbolAddress(&sp, HIP_SYMBOL(scratch));
        if (se != hipSuccess || !sp) return fail(JITNN_HIP_EDEVICE, "hipGetSymbolAddress(scratch): %s", hipGetErrorString(se));
        g.scratch_ptr = sp;
    }
    if (const char *e = getenv("JITNN_HIP_GEMV_MAX_ROWS")) {
        int v = atoi(e);
        if (v >= 1) g.gemv_max_rows = v;
    }
    if (const char *e = getenv("JITNN_HIP_GEMV_I8")) g.gemv_i8 = atoi(e) != 0;
    if (const char *e = getenv("JITNN_HIP_TRANSCODE")) g.transcode = atoi(e) != 0;
    g.device = device_ordinal;
    g.ready = true;
    return JITNN_HIP_OK;
}

int jitnn_hip_device_info(char *name, int cap, int *compute_units, long long *hbm_bytes) {
    if (int rc = check_ready()) return rc;
    if (name && cap > 0) {
        strncpy(name, g.name, (size_t)cap - 1);
        name[cap - 1] = 0;
    }
    if (compute_units) *compute_units = g.cus;
    if (hbm_bytes) *hbm_bytes = g.hbm;
    return JITNN_HIP_OK;
}

int jitnn_hip_sync(void) {
    if (int rc = check_ready()) return rc;
    HIP_TRY(hipDeviceSynchronize());
    return JITNN_HIP_OK;
}

int jitnn_hip_stats(jitnn_hip_stat *out, int cap) {
    if (cap > 0 && !out) return fail(JITNN_HIP_EINVAL, "output is NULL");
    for (int i = 0; i < ST_COUNT && i < cap; ++i) {
        std::snprintf(out[i].name, sizeof(out[i].name), "%s", kStatNames[i]);
        out[i].calls = g_stat_calls[i].load(std::memory_order_relaxed);
        out[i].tensor_bytes = g_stat_bytes[i].load(std::memory_order_relaxed);
    }
    return ST_COUNT;
}

int jitnn_hip_stats_reset(void) {
    for (int i = 0; i < ST_COUNT; ++i) {
        g_stat_calls[i].store(0, std::memory_order_relaxed);
        g_stat_bytes[i].store(0, std::memory_order_relaxed);
    }
    return JITNN_HIP_OK;
}

int jitnn_hip_weight_upload(int fmt, const void *blocks_host, long long nbytes, int n, int k, jitnn_hip_weight **out) {
    if (int rc = check_weight_args(fmt, nbytes, n, k, blocks_host, out)) return rc;
    if (int rc = check_ready()) return rc;
    uint8_t *dev = nullptr;
    hipError_t e = hipMalloc(&dev, (size_t)nbytes);
    if (e != hipSuccess) return fail(JITNN_HIP_ENOMEM, "hipMalloc of %lld bytes: %s", nbytes, hipGetErrorString(e));
    e = hipMemcpy(dev, blocks_host, (size_t)nbytes, hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        (void)hipFree(dev);
        return fail(JITNN_HIP_EDEVICE, "hipMemcpy of %lld bytes: %s", nbytes, hipGetErrorString(e));
    }
    // Q5_0 and Q3_K have no kernels of their own but hold exactly the values of Q8_0 / Q6_K blocks (dequant.h): rewritten
    // once, here, they run on those formats' kernels with the same results, bit for bit where the dequantiser is concerned
    int dev_fmt = fmt;
    long long dev_nbytes = nbytes;
    if (g.transcode && (fmt == F_Q5_0 || fmt == F_Q3_K)) {
        dev_fmt = fmt == F_Q5_0 ? F_Q8_0 : F_Q6_K;
        dev_nbytes = jitnn_hip_weight_nbytes(dev_fmt, n, k);
        uint8_t *dev2 = nullptr;
        e = hipMalloc(&dev2, (size_t)dev_nbytes);
        if (e != hipSuccess) {
            (void)hipFree(dev);
            return fail(JITNN_HIP_ENOMEM, "hipMalloc of %lld bytes: %s", dev_nbytes, hipGetErrorString(e));
        }
        const size_t blocks = (size_t)n * k / block_values(fmt);
        const unsigned grid = (unsigned)std::min<size_t>((blocks + 255) / 256, (size_t)g.cus * 16);
        if (fmt == F_Q5_0) hipLaunchKernelGGL(transcode_q5_0_to_q8_0_kernel, dim3(grid), dim3(256), 0, nullptr, dev, dev2, blocks);
        else hipLaunchKernelGGL(transcode_q3_k_to_q6_k_kernel, dim3(grid), dim3(256), 0, nullptr, dev, dev2, blocks);
        e = hipGetLastError();
        if (e == hipSuccess) e = hipStreamSynchronize(nullptr);
        (void)hipFree(dev);
        dev = dev2;
        if (e != hipSuccess) {
            (void)hipFree(dev);
            return fail(JITNN_HIP_EDEVICE, "rewriting the blocks: %s", hipGetErrorString(e));
        }
    }
    jitnn_hip_weight *w = new (std::nothrow) jitnn_hip_weight{dev_fmt, n, k, dev_nbytes, dev, true};
    if (!w) {
        (void)hipFree(dev);
        return fail(JITNN_HIP_ENOMEM, "out of host memory");
    }
    if (dev_fmt != fmt) {
        w->file_fmt = fmt;
        w->file_nbytes = nbytes;
    }
    *out = w;
    return JITNN_HIP_OK;
}

int jitnn_hip_weight_wrap_dev(int fmt, const void *dev_blocks, long long nbytes, int n, int k, jitnn_hip_weight **out) {
    if (int rc = check_weight_args(fmt, nbytes, n, k, dev_blocks, out)) return rc;
    if (((uintptr_t)dev_blocks & 15) != 0) return fail(JITNN_HIP_EINVAL, "device blocks must be 16-byte aligned");
    jitnn_hip_weight *w = new (std::nothrow) jitnn_hip_weight{fmt, n, k, nbytes, (uint8_t *)dev_blocks, false};
    if (!w) return fail(JITNN_HIP_ENOMEM, "out of host memory");
    *out = w;
    return JITNN_HIP_OK;
}

int jitnn_hip_weight_free(jitnn_hip_weight *w) {
    if (!w) return JITNN_HIP_OK;
    int rc = JITNN_HIP_OK;
    if (w->owned && w->dev) {
        hipError_t e = hipFree(w->dev);
        if (e != hipSuccess) rc = fail(JITNN_HIP_EDEVICE, "hipFree: %s", hipGetErrorString(e));
    }
    delete w;
    return rc;
}

int jitnn_hip_weight_info(const jitnn_hip_weight *w, int *fmt, int *n, int *k, long long *nbytes) {
    if (!w) return fail(JITNN_HIP_EINVAL, "weight is NULL");
    if (fmt) *fmt = w->file_fmt ? w->file_fmt : w->fmt;  // (the caller's format and byte count, also where the device copy is another)
    if (n) *n = w->n;
    if (k) *k = w->k;
    if (nbytes) *nbytes = w->file_fmt ? w->file_nbytes : w->nbytes;
    return JITNN_HIP_OK;
}

int jitnn_hip_dequantize_dev(const jitnn_hip_weight *w, float *y_dev, void *stream) {
    if (!w || !y_dev) return fail(JITNN_HIP_EINVAL, "weight or output is NULL");
    if (int rc = check_ready()) return rc;
    hipStream_t s = (hipStream_t)stream;
    count_op(ST_DEQUANT, (long long)w->nbytes + 4ll * w->n * w->k);
    switch (w->fmt) {
    case F_Q4_0: launch_dequant<F_Q4_0>(w, y_dev, s); break;
    case F_Q4_1: launch_dequant<F_Q4_1>(w, y_dev, s); break;
    case F_Q8_0: launch_dequant<F_Q8_0>(w, y_dev, s); break;
    case F_Q4_K: launch_dequant<F_Q4_K>(w, y_dev, s); break;
    case F_Q5_K: launch_dequant<F_Q5_K>(w, y_dev, s); break;
    case F_Q5_0: launch_dequant<F_Q5_0>(w, y_dev, s); break;
    case F_Q5_1: launch_dequant<F_Q5_1>(w, y_dev, s); break;
    case F_Q2_K: launch_dequant<F_Q2_K>(w, y_dev, s); break;
    case F_Q3_K: launch_dequant<F_Q3_K>(w, y_dev, s); break;
    default: launch_dequant<F_Q6_K>(w, y_dev, s); break;
    }
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int jitnn_hip_dequantize(const jitnn_hip_weight *w, float *y_host) {
    if (!w || !y_host) return fail(JITNN_HIP_EINVAL, "weight or output is NULL");
    if (int rc = check_ready()) return rc;
    // in pieces of whole rows through the thread's device buffer: no allocation per call, bounded memory for any matrix
    const size_t row_out = (size_t)w->k * sizeof(float), row_in = (size_t)w->nbytes / w->n;
    size_t piece_rows = ((size_t)64 << 20) / row_out;
    if (piece_rows < 1) piece_rows = 1;
    if (piece_rows > (size_t)w->n) piece_rows = (size_t)w->n;
    if (int rc = stage_reserve(0, piece_rows * row_out)) return rc;
    HostStage &st = g_thread.stage;
    count_op(ST_DEQUANT, (long long)w->nbytes + 4ll * w->n * w->k);
    StatNest nest;
    for (size_t r0 = 0; r0 < (size_t)w->n; r0 += piece_rows) {
        const size_t nr = std::min(piece_rows, (size_t)w->n - r0);
        const jitnn_hip_weight part{w->fmt, (int)nr, w->k, (long long)(nr * row_in), w->dev + r0 * row_in, false};
        if (int rc = jitnn_hip_dequantize_dev(&part, (float *)st.dev, st.stream)) return rc;
        HIP_TRY(hipMemcpyAsync((uint8_t *)y_host + r0 * row_out, st.dev, nr * row_out, hipMemcpyDeviceToHost, st.stream));
        HIP_TRY(hipStreamSynchronize(st.stream));
    }
    return JITNN_HIP_OK;
}

}  // extern "C"

namespace {

// Does a linear of `rows` rows on this weight take the one-pass kernel of gemv_rows.h?  From 9 rows; rows of 12288 values and
// more - the ffn_down of an 8B layer, 4096 x 14336 - from 3: Q6_K 35.6 against 41.5-44.6 us, Q4_K 24.5 against 26.6-27.6,
// Q4_0 22.3 against 25.4, Q8_0 27.2 against 34.4, where the kernels for up to 8 rows pay their activation set-up per
// 4096-value slice (at 8192 values they are still ahead, 15.0 against 16.9).  Q4_0 and Q4_1 with shorter rows from 12: their
// kernels for up to 8 rows are the fastest of all, and 8 + 1..3 rows in two passes still beat the one pass (14336 x 4096
// Q4_0 at 9 rows 21.9 against 27.0 us, at 12 rows 26.2 against 27.0, at 20 rows 38.9 against 29.9).
bool rows_path(const jitnn_hip_weight *w, int rows) {
    int rows_min = 9;  // (up to 8 rows gemv_mfma_kernel is faster)
    if (w->k >= 12288) rows_min = 3;
    else if (w->fmt == F_Q4_0 || w->fmt == F_Q4_1) rows_min = 12;
    else if (is_extra_format(w->fmt)) rows_min = 5;  // (Q5_1, Q2_K: up to four rows are one launch of the INT8 kernel)
    return rows >= rows_min && rows <= 64 && rows <= g.gemv_max_rows && gemv_rows_supported(w->fmt) && w->k % 256 == 0 &&
           w->n >= 16;
}

// The same for rows of 32-value blocks that are not whole columns: the whole ones in one pass, the rest by gemv_tail_kernel, instead of
// passes of eight rows, which stream the weight once each.  us, passes against this: Q4_1 5120 x 11456 at 5 / 9 / 40 / 64 rows 57 / 70 / 308 / 492
// and 26 / 29 / 44 / 55, Q8_0 8000 x 5088 48 / 68 / 276 / 441 and 29 / 32 / 43 / 55, Q4_0 2048 x 2272 at 5 / 8 / 9 / 40 16 / 18 / 23 / 88 and 17.5 / 17.5 /
// 17 / 20, Q4_0 4096 x 1504 at 9 / 11 / 16 16.4 / 16.7 / 21.0 and 17.3 / 17.8 / 17.7, Q8_0 2672 x 1056 at 8 / 9 9.6 / 17.4 and 14.0 / 14.1.
// Against FP64 (weights around zero, 288 to 14304 values, 3 to 64 rows; 2-norm) the passes' FP32 arithmetic is 2.4e-7 to 3.7e-7 off, this,
// whose sums are shorter, 0.49 (Q8_0), 0.52 (Q4_0) and 0.58 (Q4_1) times as much in the mean from nine rows on, nowhere more.
bool rows_ragged_path(const jitnn_hip_weight *w, int rows) {
    if (w->fmt != F_Q4_0 && w->fmt != F_Q4_1 && w->fmt != F_Q8_0) return false;
    const int rows_min = w->k >= 12288 ? 3 : w->k >= 3072 ? 5 : w->k >= 2048 || w->fmt == F_Q8_0 ? 9 : 13;
    return w->k % 256 != 0 && w->k > 256 && rows >= rows_min && rows <= 64 && rows <= g.gemv_max_rows && w->n >= 16;
}

// One launch of rows_path, with a join of its own where it has slices: the plan of the kernel that holds the operands, or groups_held = 0.
size_t rows_operand_bytes(int rows, int k) { return (gemv_rows_scratch_bytes(rows, k) + 255) & ~(size_t)255; }
HeldPlan rows_plan(const jitnn_hip_weight *w, int rows, bool adds, int cus) {
    const HeldPlan p = gemv_held_plan(w->fmt, w->n, w->k, rows, adds ? HELD_JOIN_ADDS : HELD_JOIN_SLICES, cus);
    // (the same limit for both sources of scratch, so that both entry points take the same kernels)
    return rows_operand_bytes(rows, w->k) + p.part_bytes(rows, w->n) <= JITNN_HIP_SCRATCH_BYTES ? p : HeldPlan{};
}

// ys[i] = x ws[i]^T (+ bias) (+ residual [rows, n]; bias and residual with one weight only) for weights that all pass
// rows_path: the activation operands are prepared once per granularity of block sums and shared by the weights.
// swiglu_up: the activations are silu(x) * swiglu_up, formed by the preparation as it reads x.
// later, defer (one weight, a residual): where the sums come in up to eight slices, they go to later and their join is left to the
// caller, as *defer.
// act: of the sum and bias, in front of the residual (one weight, nothing put off).
// together, room, gdefer (three weights): where one of them comes in slices, all three go to `together` (room floats), one after
// the other, a weight that has none as its one slice, and the caller joins them, as *gdefer.
int launch_rows_group(const jitnn_hip_weight *const *ws, float *const *ys, int count, const float *x, int rows, const float *bias, const float *residual,
                      hipStream_t s, ScratchSource src, const float *swiglu_up = nullptr, float *later = nullptr, PfPending *defer = nullptr,
                      float *together = nullptr, size_t room = 0, PfGroupPending *gdefer = nullptr, int act = JITNN_HIP_ACT_NONE) {
    const int k = ws[0]->k;
    const Epilogue epi{act, residual};
    bool need[GR_LAYOUTS] = {};  // the operand layouts the weights ask for
    const size_t one = rows_operand_bytes(rows, k);
    int layouts = 0;
    for (int i = 0; i < count; ++i) {
        if (ws[i]->k != k) return fail(JITNN_HIP_EINVAL, "weights of %d and %d values per row on one activation", k, ws[i]->k);
        bool &l = need[gemv_rows_layout(ws[i]->fmt)];
        layouts += !l;
        l = true;
    }
    // which weights take the kernel that holds the operands; its slices' sums, one weight's at a time, stand behind the operands
    HeldPlan plan[3];
    size_t part = 0;
    int later_plan = 0;  // slices whose join the caller gets
    bool grouped = false;
    if (gdefer && count == 3) {
        size_t floats = 0;
        int most = 1;
        for (int i = 0; i < 3; ++i) {
            plan[i] = gemv_held_plan(ws[i]->fmt, ws[i]->n, k, rows, HELD_JOIN_READER, g.cus);
            const int splits = plan[i].groups_held ? plan[i].slices : 1;
            floats += (size_t)splits * rows * ws[i]->n;
            most = std::max(most, splits);
        }
        grouped = most > 1 && most <= 8 && floats <= room;
    }
    for (int i = 0; i < count && !grouped; ++i) {
        // (a slice is at most eight columns; more slices only where that is less than k / 2048.  The kernels that join read the residual 16
        // bytes at a time: the caller's rows, in front of the first layer, need not be aligned to that)
        const bool put_off = defer && k <= 8 * 2048 && ((uintptr_t)residual & 15) == 0;
        if (put_off) plan[i] = gemv_held_plan(ws[i]->fmt, ws[i]->n, k, rows, HELD_JOIN_READER, g.cus);
        if (put_off && plan[i].slices > 1 && plan[i].slices <= 8) {
            later_plan = plan[i].slices;
            continue;
        }
        plan[i] = rows_plan(ws[i], rows, bias || epi.any(), g.cus);
        part = std::max(part, plan[i].part_bytes(rows, ws[i]->n));
    }
    void *scratch = nullptr;
    if (part && !workspace_at_hand(one * layouts + part, s, src)) part = 0;  // (slice after slice into the output then: the same bits)
    if (int rc = workspace(one * layouts + part, s, &scratch, src)) return rc;
    for (int i = 0; i < count; ++i) {
        const KernelRef kr = plan[i].groups_held ? gemv_held_kernel_ref(ws[i]->fmt, plan[i].groups_held)
                                                 : gemv_rows_kernel_ref(ws[i]->fmt, ws[i]->n, k, rows, (unsigned)g.cus, act != JITNN_HIP_ACT_NONE);
        if (int rc = allow_lds(kr.fn, kr.lds)) return rc;
    }
    uint8_t *sc[GR_LAYOUTS] = {};
    for (int l = 0, used = 0; l < GR_LAYOUTS; ++l)
        if (need[l]) sc[l] = (uint8_t *)scratch + one * used++;
    gemv_rows_prepare_launch(s, x, swiglu_up, (void *const *)sc, k, rows);
    for (int i = 0; i < count; ++i) {
        const void *ops = sc[gemv_rows_layout(ws[i]->fmt)];
        if (grouped) {
            const int splits = plan[i].groups_held ? plan[i].slices : 1;
            if (plan[i].groups_held) gemv_held_slices_launch(plan[i], ws[i]->fmt, s, ws[i]->dev, nullptr, ops, together, ws[i]->n, k, rows);
            else gemv_rows_main_launch(ws[i]->fmt, (unsigned)g.cus, s, ws[i]->dev, ops, nullptr, Epilogue{}, together, ws[i]->n, k, rows);
            if (i == 0) gdefer->part = together;
            gdefer->sg.splits[i] = splits;
            gdefer->sg.n[i] = ws[i]->n;
            together += (size_t)splits * rows * ws[i]->n;
        } else if (later_plan) {
            gemv_held_slices_launch(plan[i], ws[i]->fmt, s, ws[i]->dev, nullptr, ops, later, ws[i]->n, k, rows);
            defer->part = later;
            defer->res = residual;
            defer->out = ys[i];
            defer->splits = later_plan;
            defer->n = ws[i]->n;
        } else if (plan[i].groups_held)
            gemv_held_launch(plan[i], ws[i]->fmt, g.cus, s, ws[i]->dev, ops, bias, epi, ys[i], part ? (float *)((uint8_t *)scratch + one * layouts) : nullptr, ws[i]->n, k, rows);
        else gemv_rows_main_launch(ws[i]->fmt, (unsigned)g.cus, s, ws[i]->dev, ops, bias, epi, ys[i], ws[i]->n, k, rows);
    }
    HIP_TRY(hipGetLastError());
    return workspace_done(s, src);
}

// y = res + (silu(x wg^T) * (x wu^T)) wd^T, for weights that all pass rows_path, where gate and up (one format and shape) pay as one
// launch of the held kernel: 37 us for the two of an 8B layer at 40 tokens, whose slices used to be joined by launches of their
// own, 4.2 us each, and now meet in the preparation of the down projection's operands.  later, defer: as for launch_rows_group.
struct RowsFfn {
    HeldPlan pair, down;
    bool to_reader;  // the slices of the down projection are joined by whoever reads y next
    size_t ops, sums, ops_down, total;  // scratch: operands of x | slices of gate and up | operands of the gated rows | slices of down
};
bool rows_ffn_pays(const jitnn_hip_weight *wg, const jitnn_hip_weight *wu, const jitnn_hip_weight *wd, int rows, hipStream_t s, RowsFfn *f) {
    if (wg->fmt != wu->fmt || wg->n != wu->n || wg->k != wu->k || wd->k != wg->n) return false;
    if (!rows_path(wg, rows) || !rows_path(wu, rows) || !rows_path(wd, rows)) return false;
    const int n = wg->n;
    f->pair = gemv_held_plan(wg->fmt, n, wg->k, rows, HELD_JOIN_READER, g.cus, 2);
    if (!f->pair.groups_held) return false;
    f->down = gemv_held_plan(wd->fmt, wd->n, n, rows, HELD_JOIN_READER, g.cus);
    f->to_reader = f->down.slices > 1 && f->down.slices <= 8;
    if (!f->to_reader) f->down = gemv_held_plan(wd->fmt, wd->n, n, rows, HELD_JOIN_ADDS, g.cus);
    auto pad = [](size_t b) { return (b + 255) & ~(size_t)255; };
    f->ops = pad(gemv_rows_scratch_bytes(rows, wg->k));
    f->sums = pad(2 * f->pair.part_bytes(rows, n));
    f->ops_down = pad(gemv_rows_scratch_bytes(rows, n));
    f->total = f->ops + f->sums + f->ops_down + (f->to_reader ? 0 : f->down.part_bytes(rows, wd->n));
    return workspace_at_hand(f->total, s, SCRATCH_THREAD);
}
int launch_rows_ffn(const RowsFfn &f, const jitnn_hip_weight *wg, const jitnn_hip_weight *wu, const jitnn_hip_weight *wd, const float *x, int rows,
                    const float *res, float *y, hipStream_t s, float *later, PfPending *defer) {
    const int n = wg->n, k = wg->k;
    const HeldPlan &pair = f.pair, &down = f.down;
    const size_t ops = f.ops, sums = f.sums, ops_down = f.ops_down, total = f.total;
    const bool to_reader = f.to_reader;
    const KernelRef kp = gemv_held_kernel_ref(wg->fmt, pair.groups_held),
                    kd = down.groups_held ? gemv_held_kernel_ref(wd->fmt, down.groups_held) : gemv_rows_kernel_ref(wd->fmt, wd->n, n, rows, (unsigned)g.cus, false);
    if (int rc = allow_lds(kp.fn, kp.lds)) return rc;
    if (int rc = allow_lds(kd.fn, kd.lds)) return rc;
    void *scratch = nullptr;
    if (int rc = workspace(total, s, &scratch)) return rc;
    for (const jitnn_hip_weight *w : {wg, wu, wd}) count_op(ST_GEMV, (long long)w->nbytes + 4ll * rows * ((long long)w->k + w->n));
    uint8_t *base = (uint8_t *)scratch;
    float *gate = (float *)(base + ops), *up = gate + (size_t)pair.slices * rows * n;
    void *in[GR_LAYOUTS] = {}, *mid[GR_LAYOUTS] = {};
    in[gemv_rows_layout(wg->fmt)] = base;
    mid[gemv_rows_layout(wd->fmt)] = base + ops + sums;
    gemv_rows_prepare_launch(s, x, nullptr, in, k, rows);
    gemv_held_slices_launch(pair, wg->fmt, s, wg->dev, wu->dev, base, gate, n, k, rows);
    gemv_rows_prepare_launch(s, gate, up, mid, n, rows, pair.slices);
    const void *md = base + ops + sums;
    if (to_reader) {
        gemv_held_slices_launch(down, wd->fmt, s, wd->dev, nullptr, md, later, wd->n, n, rows);
        defer->part = later;
        defer->res = res;
        defer->out = y;
        defer->splits = down.slices;
        defer->n = wd->n;
    } else if (down.groups_held) {
        gemv_held_launch(down, wd->fmt, g.cus, s, wd->dev, md, nullptr, Epilogue{0, res}, y, (float *)(base + ops + sums + ops_down), wd->n, n, rows);
    } else {
        gemv_rows_main_launch(wd->fmt, (unsigned)g.cus, s, wd->dev, md, nullptr, Epilogue{0, res}, y, wd->n, n, rows);
    }
    HIP_TRY(hipGetLastError());
    return workspace_done(s);
}

template <bool EPI>
void (*gemv_tail_of(int fmt))(const uint8_t *, const float *, float *, int, int, int, int, const Epilogue) {
    return fmt == F_Q4_0 ? gemv_tail_kernel<F_Q4_0, EPI> : fmt == F_Q4_1 ? gemv_tail_kernel<F_Q4_1, EPI> : gemv_tail_kernel<F_Q8_0, EPI>;
}
int launch_gemv_tail(const jitnn_hip_weight *w, const float *x, int rows, const Epilogue &e, float *y, hipStream_t s) {
    const int blocks = w->k % 256 / 32;
    const size_t lds = gemv_tail_lds_bytes(rows, blocks);
    const auto kernel = e.any() ? gemv_tail_of<true>(w->fmt) : gemv_tail_of<false>(w->fmt);
    if (int rc = allow_lds((const void *)kernel, lds)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((w->n + GT_ROWS - 1) / GT_ROWS)), dim3(GT_THREADS), lds, s, w->dev, x, y, w->n, w->k, rows, blocks, e);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

// y = act(x W^T (+ bias)) (+ res): by the kernel that makes the sums where it has an epilogue, else by a launch behind it (many rows; rows of odd lengths).
int linear_dev(const jitnn_hip_weight *w, const float *x_dev, int rows, const float *bias_dev, float *y_dev, hipStream_t s, ScratchSource src, const Epilogue &e = Epilogue{}) {
    if (!w || !x_dev || !y_dev) return fail(JITNN_HIP_EINVAL, "weight, input or output is NULL");
    if (rows < 1) return fail(JITNN_HIP_EINVAL, "rows = %d", rows);
    if (int rc = check_ready()) return rc;
    auto behind = [&](const Epilogue &unmet, float *y, int count) -> int {
        if (!unmet.any()) return JITNN_HIP_OK;
        linear_epilogue_launch(unmet.act, unmet.res, y, (size_t)count * w->n, g.cus, s);
        HIP_TRY(hipGetLastError());
        return JITNN_HIP_OK;
    };
    const bool many = rows > g.gemv_max_rows && has_many_row_kernel(w->fmt);
    count_op(many ? ST_MFMA : ST_GEMV, (long long)w->nbytes + 4ll * rows * ((long long)w->k + w->n) + (bias_dev ? 4ll * w->n : 0) + (e.res ? 4ll * rows * w->n : 0));
    if (many) {
        if (int rc = launch_prefill(w, x_dev, rows, bias_dev, y_dev, s, src)) return rc;
        return behind(e, y_dev, rows);
    }
    // several rows, rows of whole 256-value columns: every row meets the weights in one pass over them (gemv_rows.h)
    if (rows_path(w, rows)) return launch_rows_group(&w, &y_dev, 1, x_dev, rows, bias_dev, e.res, s, src, nullptr, nullptr, nullptr, nullptr, 0, nullptr, e.act);
    // (no scratch at hand - a stream capture before the first eager call, no memory: the passes of eight, which need none)
    if (rows_ragged_path(w, rows) && workspace_at_hand(rows_operand_bytes(rows, w->k), s, src)) {
        if (int rc = launch_rows_group(&w, &y_dev, 1, x_dev, rows, bias_dev, nullptr, s, src)) return rc;
        return launch_gemv_tail(w, x_dev, rows, e, y_dev, s);
    }
    for (int r0 = 0; r0 < rows; r0 += 8) {
        const int nb = rows - r0 < 8 ? rows - r0 : 8;
        float *const y = y_dev + (size_t)r0 * w->n;
        Epilogue unmet{e.act, e.res ? e.res + (size_t)r0 * w->n : nullptr};
        if (int rc = launch_gemv(w, x_dev + (size_t)r0 * w->k, nb, bias_dev, y, s, &unmet)) return rc;
        if (int rc = behind(unmet, y, nb)) return rc;
    }
    return JITNN_HIP_OK;
}

// two arrays of so many bytes
bool overlaps(const void *a, const void *b, size_t bytes) { return (uintptr_t)a < (uintptr_t)b + bytes && (uintptr_t)b < (uintptr_t)a + bytes; }

// What an epilogue adds to the checks of a linear (which come after these): y apart from the residual, which a launch may read after another has written y.
int check_linear_act(const jitnn_hip_weight *w, int rows, int activation, const float *residual, const float *y) {
    if (activation < 0 || activation >= ACT_COUNT) return fail(JITNN_HIP_EINVAL, "activation %d", activation);
    if (w && rows > 0 && residual && y) {
        if (overlaps(residual, y, (size_t)rows * w->n * sizeof(float))) return fail(JITNN_HIP_EINVAL, "the output overlaps the residual");
    }
    return JITNN_HIP_OK;
}

}  // namespace

extern "C" {

int jitnn_hip_linear_dev(const jitnn_hip_weight *w, const float *x_dev, int rows, const float *bias_dev, float *y_dev, void *stream) {
    return linear_dev(w, x_dev, rows, bias_dev, y_dev, (hipStream_t)stream, SCRATCH_THREAD);
}

int jitnn_hip_linear_act_dev(const jitnn_hip_weight *w, const float *x_dev, int rows, const float *bias_dev, int activation, const float *residual_dev, float *y_dev, void *stream) {
    if (int rc = check_linear_act(w, rows, activation, residual_dev, y_dev)) return rc;
    return linear_dev(w, x_dev, rows, bias_dev, y_dev, (hipStream_t)stream, SCRATCH_THREAD, Epilogue{activation, residual_dev});
}

int jitnn_hip_linear_noalloc_dev(const jitnn_hip_weight *w, const float *x_dev, int rows, const float *bias_dev, float *y_dev, void *stream) {
    return linear_dev(w, x_dev, rows, bias_dev, y_dev, (hipStream_t)stream, SCRATCH_STATIC);
}

int jitnn_hip_many_row_tile(const int *fmts, const int *n, int count, int k, int rows, int gate_up, int residual, int compute_units) {
    if (!fmts || !n || count < 1 || count > 3 || k < 1 || rows < 1 || compute_units < 0) return fail(JITNN_HIP_EINVAL, "no such launch");
    if (gate_up && (count != 2 || fmts[0] != fmts[1] || n[0] != n[1])) return fail(JITNN_HIP_EINVAL, "gate and up are two weights of one format and shape");
    if (residual && count != 1) return fail(JITNN_HIP_EINVAL, "a residual goes with one weight");
    for (int i = 0; i < count; ++i) {
        const long long need = jitnn_hip_weight_nbytes(fmts[i], n[i], k);
        if (need < 0) return (int)need;
    }
    if (compute_units == 0) {
        if (int rc = check_ready()) return rc;
        compute_units = g.cus;
    }
    WidePlan plan;
    return rows > g.gemv_max_rows && wide_pays(fmts, n, count, k, rows, gate_up != 0, residual != 0, compute_units, &plan) ? 32 * plan.rt : 0;
}

int jitnn_hip_few_rows_slices(int fmt, int n, int k, int rows, int adds, int compute_units) {
    if (rows < 1 || compute_units < 0) return fail(JITNN_HIP_EINVAL, "no such launch");
    const long long need = jitnn_hip_weight_nbytes(fmt, n, k);
    if (need < 0) return (int)need;
    if (compute_units == 0) {
        if (int rc = check_ready()) return rc;
        compute_units = g.cus;
    }
    const jitnn_hip_weight w{fmt, n, k, need, nullptr, false};
    return rows_path(&w, rows) ? rows_plan(&w, rows, adds != 0, compute_units).slices : 0;
}

static int linear_host(const jitnn_hip_weight *w, const float *x_host, int rows, const float *bias_host, int activation, const float *residual_host, float *y_host);

long long jitnn_hip_noalloc_scratch_bytes(void) { return (long long)JITNN_HIP_SCRATCH_BYTES; }

int jitnn_hip_linear(const jitnn_hip_weight *w, const float *x_host, int rows, const float *bias_host, float *y_host) {
    return linear_host(w, x_host, rows, bias_host, JITNN_HIP_ACT_NONE, nullptr, y_host);
}

int jitnn_hip_linear_act(const jitnn_hip_weight *w, const float *x_host, int rows, const float *bias_host, int activation, const float *residual_host, float *y_host) {
    if (int rc = check_linear_act(w, rows, activation, nullptr, nullptr)) return rc;
    return linear_host(w, x_host, rows, bias_host, activation, residual_host, y_host);
}

static int linear_host(const jitnn_hip_weight *w, const float *x_host, int rows, const float *bias_host, int activation, const float *residual_host, float *y_host) {
    if (!w || !x_host || !y_host) return fail(JITNN_HIP_EINVAL, "weight, input or output is NULL");
    if (rows < 1) return fail(JITNN_HIP_EINVAL, "rows = %d", rows);
    if (int rc = check_ready()) return rc;
    // layout of both staging buffers: [x | bias | residual | y], x, bias and residual going up in one copy, y coming back in one
    const size_t xb = (size_t)rows * w->k * 4, yb = (size_t)rows * w->n * 4, bb = bias_host ? (size_t)w->n * 4 : 0, rb = residual_host ? yb : 0;
    const size_t bo = (xb + 255) & ~(size_t)255, ro = bo + ((bb + 255) & ~(size_t)255), yo = ro + ((rb + 255) & ~(size_t)255), total = yo + yb;
    const bool keep = total <= STAGE_KEEP_MAX;  // small calls go through pinned memory (one DMA each way, no page locking per call)
    if (int rc = stage_reserve(keep ? total : 0, total)) return rc;
    HostStage &st = g_thread.stage;
    // small calls: the device itself fetches the input from the pinned buffer and writes the result back into it
    const bool by_kernel = keep && st.pinned_dev && total <= STAGE_KERNEL_COPY_MAX;
    auto copy16 = [&](uint8_t *dst, const uint8_t *src, size_t bytes) {
        const size_t count16 = (bytes + 15) / 16;  // the sections of the layout are 256-byte aligned: rounding up stays inside
        const unsigned blocks = (unsigned)std::min<size_t>((count16 + 255) / 256, 64);
        hipLaunchKernelGGL(stage_copy_kernel, dim3(blocks), dim3(256), 0, st.stream, (uint4 *)dst, (const uint4 *)src, count16);
    };
    if (keep) {
        memcpy(st.pinned, x_host, xb);
        if (bias_host) memcpy(st.pinned + bo, bias_host, bb);
        if (residual_host) memcpy(st.pinned + ro, residual_host, rb);
        const size_t up = residual_host ? ro + rb : bias_host ? bo + bb : xb;
        if (by_kernel) copy16(st.dev, st.pinned_dev, up);
        else HIP_TRY(hipMemcpyAsync(st.dev, st.pinned, up, hipMemcpyHostToDevice, st.stream));
    } else {
        HIP_TRY(hipMemcpyAsync(st.dev, x_host, xb, hipMemcpyHostToDevice, st.stream));
        if (bias_host) HIP_TRY(hipMemcpyAsync(st.dev + bo, bias_host, bb, hipMemcpyHostToDevice, st.stream));
        if (residual_host) HIP_TRY(hipMemcpyAsync(st.dev + ro, residual_host, rb, hipMemcpyHostToDevice, st.stream));
    }
    int rc = jitnn_hip_linear_act_dev(w, (const float *)st.dev, rows, bias_host ? (const float *)(st.dev + bo) : nullptr, activation,
                                      residual_host ? (const float *)(st.dev + ro) : nullptr, (float *)(st.dev + yo), st.stream);
    if (rc == JITNN_HIP_OK) {
        if (by_kernel) {
            copy16(st.pinned_dev + yo, st.dev + yo, yb);
            HIP_TRY(hipGetLastError());
        } else {
            HIP_TRY(hipMemcpyAsync(keep ? (void *)(st.pinned + yo) : (void *)y_host, st.dev + yo, yb, hipMemcpyDeviceToHost, st.stream));
        }
        HIP_TRY(hipStreamSynchronize(st.stream));
        if (keep) memcpy(y_host, st.pinned + yo, yb);
    }
    if (!keep) {  // a buffer this large is not held on to
        (void)hipStreamSynchronize(st.stream);
        (void)hipFree(st.dev);
        st.dev = nullptr;
        st.dcap = 0;
    }
    return rc;
}

int jitnn_hip_quantize_q8_0_dev(const float *x_dev, long long numel, void *blocks_dev, void *stream) {
    if (!x_dev || !blocks_dev) return fail(JITNN_HIP_EINVAL, "input or output is NULL");
    if (numel < 0 || numel % 32 != 0) return fail(JITNN_HIP_EINVAL, "Q8_0 needs a multiple of 32 values, got %lld", numel);
    if (int rc = check_ready()) return rc;
    if (numel == 0) return JITNN_HIP_OK;
    count_op(ST_QUANT, 4ll * numel + numel / 32 * 34);
    const size_t blocks = (size_t)numel / 32;
    size_t grid = (blocks + 4 * Q8Q_BLOCKS - 1) / (4 * Q8Q_BLOCKS);
    if (grid > (size_t)g.cus * 32) grid = (size_t)g.cus * 32;
    hipLaunchKernelGGL(quantize_q8_0_kernel, dim3((unsigned)grid), dim3(256), 0, (hipStream_t)stream, x_dev, (uint8_t *)blocks_dev, blocks);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int jitnn_hip_quantize_q8_0(const float *x_host, long long numel, void *blocks_host) {
    if (!x_host || !blocks_host) return fail(JITNN_HIP_EINVAL, "input or output is NULL");
    if (numel < 0 || numel % 32 != 0) return fail(JITNN_HIP_EINVAL, "Q8_0 needs a multiple of 32 values, got %lld", numel);
    if (int rc = check_ready()) return rc;
    if (numel == 0) return JITNN_HIP_OK;
    // in pieces of whole blocks through the thread's device buffer
    const long long piece = (long long)16 << 20;  // values per piece: 64 MiB in, 17 MiB out
    const size_t xmax = (size_t)std::min(numel, piece) * 4, qo = (xmax + 255) & ~(size_t)255;
    if (int rc = stage_reserve(0, qo + (size_t)std::min(numel, piece) / 32 * 34)) return rc;
    HostStage &st = g_thread.stage;
    count_op(ST_QUANT, 4ll * numel + numel / 32 * 34);
    StatNest nest;
    for (long long v0 = 0; v0 < numel; v0 += piece) {
        const long long nv = std::min(piece, numel - v0);
        HIP_TRY(hipMemcpyAsync(st.dev, x_host + v0, (size_t)nv * 4, hipMemcpyHostToDevice, st.stream));
        if (int rc = jitnn_hip_quantize_q8_0_dev((const float *)st.dev, nv, st.dev + qo, st.stream)) return rc;
        HIP_TRY(hipMemcpyAsync((uint8_t *)blocks_host + v0 / 32 * 34, st.dev + qo, (size_t)nv / 32 * 34, hipMemcpyDeviceToHost, st.stream));
        HIP_TRY(hipStreamSynchronize(st.stream));
    }
    return JITNN_HIP_OK;
}

int jitnn_hip_thread_scratch(long long *held, long long *kept_for_graphs, int *allocations) {
    if (held) *held = (long long)(g_ws.operands.capacity() + g_ws.weights.capacity());
    if (kept_for_graphs) *kept_for_graphs = (long long)(g_ws.operands.retired_bytes() + g_ws.weights.retired_bytes());
    if (allocations) *allocations = g_ws.operands.growths() + g_ws.weights.growths();
    return JITNN_HIP_OK;
}

int jitnn_hip_thread_release(void) {
    if (!g.ready) return JITNN_HIP_OK;
    (void)hipDeviceSynchronize();
    g_thread.stage.release();
    release_workspace();
    return JITNN_HIP_OK;
}

int jitnn_hip_probe_read_shape_dev(const void *dev, long long nbytes, int workgroups_per_cu, int loads_in_flight, int nontemporal, void *stream) {
    if (!dev || nbytes < 16 || ((uintptr_t)dev & 15) != 0) return fail(JITNN_HIP_EINVAL, "need a 16-byte aligned buffer of at least 16 bytes");
    if (workgroups_per_cu < 1 || workgroups_per_cu > 16) return fail(JITNN_HIP_EINVAL, "%d workgroups per CU", workgroups_per_cu);
    if (int rc = check_ready()) return rc;
    typedef void (*fn_t)(const u32x4 *, size_t, uint32_t *, uint32_t);
    fn_t fn = nullptr;
    switch (loads_in_flight) {
    case 1: fn = nontemporal ? probe_read_kernel<1, true> : probe_read_kernel<1, false>; break;
    case 2: fn = nontemporal ? probe_read_kernel<2, true> : probe_read_kernel<2, false>; break;
    case 4: fn = nontemporal ? probe_read_kernel<4, true> : probe_read_kernel<4, false>; break;
    case 8: fn = nontemporal ? probe_read_kernel<8, true> : probe_read_kernel<8, false>; break;
    case 16: fn = nontemporal ? probe_read_kernel<16, true> : probe_read_kernel<16, false>; break;
    default: return fail(JITNN_HIP_EINVAL, "%d loads in flight (1, 2, 4, 8 or 16)", loads_in_flight);
    }
    hipLaunchKernelGGL(fn, dim3(g.cus * workgroups_per_cu), dim3(256), 0, (hipStream_t)stream, (const u32x4 *)dev, (size_t)nbytes / 16, (uint32_t *)nullptr,
                       (uint32_t)(g.cus * workgroups_per_cu * 256));
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int jitnn_hip_probe_read_dev(const void *dev, long long nbytes, void *stream) {
    return jitnn_hip_probe_read_shape_dev(dev, nbytes, 8, 1, 0, stream);  // the shape a sweep found fastest on 33 MB (6.4 us against 7.5 for 2 x 4)
}

int jitnn_hip_malloc(long long nbytes, void **dev) {
    if (!dev || nbytes < 0) return fail(JITNN_HIP_EINVAL, "bad arguments");
    *dev = nullptr;
    if (int rc = check_ready()) return rc;
    hipError_t e = hipMalloc(dev, (size_t)(nbytes > 0 ? nbytes : 1));
    if (e != hipSuccess) return fail(JITNN_HIP_ENOMEM, "hipMalloc of %lld bytes: %s", nbytes, hipGetErrorString(e));
    return JITNN_HIP_OK;
}

int jitnn_hip_free(void *dev) {
    if (!dev) return JITNN_HIP_OK;
    HIP_TRY(hipFree(dev));
    return JITNN_HIP_OK;
}

int jitnn_hip_memcpy_h2d(void *dev, const void *host, long long nbytes) {
    if (!dev || !host || nbytes < 0) return fail(JITNN_HIP_EINVAL, "bad arguments");
    if (int rc = check_ready()) return rc;
    HIP_TRY(hipMemcpy(dev, host, (size_t)nbytes, hipMemcpyHostToDevice));
    return JITNN_HIP_OK;
}

int jitnn_hip_memcpy_d2h(void *host, const void *dev, long long nbytes) {
    if (!dev || !host || nbytes < 0) return fail(JITNN_HIP_EINVAL, "bad arguments");
    if (int rc = check_ready()) return rc;
    HIP_TRY(hipMemcpy(host, dev, (size_t)nbytes, hipMemcpyDeviceToHost));
    return JITNN_HIP_OK;
}

}  // extern "C"

// ================================================================================================ GGUF files

struct jitnn_hip_gguf {
    GgufFile *f;
};

extern "C" {

int jitnn_hip_gguf_open(const char *path, jitnn_hip_gguf **out) {
    if (!out) return fail(JITNN_HIP_EINVAL, "out is NULL");
    *out = nullptr;
    if (!path) return fail(JITNN_HIP_EINVAL, "path is NULL");
    std::string err;
    GgufFile *f = gguf_open(path, err);
    if (!f) return fail(JITNN_HIP_EIO, "%s", err.c_str());
    jitnn_hip_gguf *h = new (std::nothrow) jitnn_hip_gguf{f};
    if (!h) {
        delete f;
        return fail(JITNN_HIP_ENOMEM, "out of host memory");
    }
    *out = h;
    return JITNN_HIP_OK;
}

int jitnn_hip_gguf_close(jitnn_hip_gguf *h) {
    if (!h) return JITNN_HIP_OK;
    delete h->f;
    delete h;
    return JITNN_HIP_OK;
}

int jitnn_hip_gguf_header(const jitnn_hip_gguf *h, int *version, int *alignment, long long *data_offset, long long *tensor_count,
                          long long *kv_count) {
    if (!h) return fail(JITNN_HIP_EINVAL, "file is NULL");
    if (version) *version = h->f->version;
    if (alignment) *alignment = h->f->alignment;
    if (data_offset) *data_offset = h->f->data_offset;
    if (tensor_count) *tensor_count = (long long)h->f->tensors.size();
    if (kv_count) *kv_count = h->f->kv_count;
    return JITNN_HIP_OK;
}

long long jitnn_hip_gguf_metadata_json(const jitnn_hip_gguf *h, char *buf, long long cap) {
    if (!h) return fail(JITNN_HIP_EINVAL, "file is NULL");
    const std::string &j = h->f->metadata_json;
    if (buf && cap > 0) {
        const size_t n = j.size() < (size_t)cap - 1 ? j.size() : (size_t)cap - 1;
        memcpy(buf, j.data(), n);
        buf[n] = 0;
    }
    return (long long)j.size();
}

int jitnn_hip_gguf_tensor_name(const jitnn_hip_gguf *h, long long index, char *name, int cap) {
    if (!h || !name || cap < 1) return fail(JITNN_HIP_EINVAL, "bad arguments");
    if (index < 0 || index >= (long long)h->f->tensors.size()) return fail(JITNN_HIP_EINVAL, "tensor %lld of %zu", index, h->f->tensors.size());
    strncpy(name, h->f->tensors[(size_t)index].name.c_str(), (size_t)cap - 1);
    name[cap - 1] = 0;
    return JITNN_HIP_OK;
}

int jitnn_hip_gguf_tensor_info(const jitnn_hip_gguf *h, const char *name, int *type, int *ndims, long long *dims, long long *file_offset,
                               long long *nbytes) {
    if (!h || !name) return fail(JITNN_HIP_EINVAL, "file or name is NULL");
    const GgufTensor *t = h->f->find(name);
    if (!t) return fail(JITNN_HIP_EINVAL, "%s: no tensor %s", h->f->path.c_str(), name);
    if (type) *type = t->type_id;
    if (ndims) *ndims = (int)t->shape.size();
    if (dims)
        for (size_t i = 0; i < t->shape.size(); ++i) dims[i] = t->shape[i];
    if (file_offset) *file_offset = t->offset;
    if (nbytes) *nbytes = t->bytes;
    return JITNN_HIP_OK;
}

int jitnn_hip_gguf_tensor_read(const jitnn_hip_gguf *h, const char *name, void *dst_host, long long nbytes) {
    if (!h || !name || !dst_host) return fail(JITNN_HIP_EINVAL, "NULL argument");
    const GgufTensor *t = h->f->find(name);
    if (!t) return fail(JITNN_HIP_EINVAL, "%s: no tensor %s", h->f->path.c_str(), name);
    if (t->bytes < 0) return fail(JITNN_HIP_EUNSUPPORTED, "%s: ggml type %d is unknown, so its size is too", name, t->type_id);
    if (nbytes != t->bytes) return fail(JITNN_HIP_EINVAL, "%s holds %lld bytes, asked for %lld", name, t->bytes, nbytes);
    memcpy(dst_host, h->f->map + t->offset, (size_t)nbytes);
    return JITNN_HIP_OK;
}

int jitnn_hip_gguf_tensor_upload(const jitnn_hip_gguf *h, const char *name, jitnn_hip_weight **out) {
    if (!out) return fail(JITNN_HIP_EINVAL, "out is NULL");
    *out = nullptr;
    if (!h || !name) return fail(JITNN_HIP_EINVAL, "file or name is NULL");
    const GgufTensor *t = h->f->find(name);
    if (!t) return fail(JITNN_HIP_EINVAL, "%s: no tensor %s", h->f->path.c_str(), name);
    if (!known(t->type_id)) {
        const GgmlTypeInfo *ti = ggml_type(t->type_id);
        if (ti) return fail(JITNN_HIP_EUNSUPPORTED, "%s: ggml type %s has no block-quantised tensor type on this path", name, ti->name);
        return fail(JITNN_HIP_EUNSUPPORTED, "%s: ggml type id %d has no block-quantised tensor type on this path", name, t->type_id);
    }
    if (t->shape.empty() || t->numel > 0x7fffffffLL)
        return fail(JITNN_HIP_EUNSUPPORTED, "%s: %lld values; tensors hold at most 2^31-1", name, t->numel);
    const long long k = t->shape.back(), n = k > 0 ? t->numel / k : 0;
    return jitnn_hip_weight_upload(t->type_id, h->f->map + t->offset, t->bytes, (int)n, (int)k, out);
}

}  // extern "C"

// ================================================================================================ rotary positions

struct jitnn_hip_rope {
    int rot = 0;
    bool interleaved = false;
    double magnitude = 1.0;
    std::vector<double> frequency;         // [rot / 2], after scaling
    unsigned long long *turns = nullptr;  // [rot / 2] on the device: 2^64 of a frequency as a fraction of a turn
};

namespace {

void rope_drop(jitnn_hip_rope *r) {
    if (r && r->turns) (void)hipFree(r->turns);
    delete r;
}

// Frequencies, magnitude and the device's copy; the arguments have been checked.
int rope_build(int rot, bool interleaved, double theta, const jitnn_hip_rope_scaling *sc, const float *factors, jitnn_hip_rope **out) {
    jitnn_hip_rope *r = nullptr;
    std::vector<unsigned long long> turns;
    try {
        r = new jitnn_hip_rope;
        r->frequency.resize((size_t)rot / 2);
        turns.resize((size_t)rot / 2);
    } catch (const std::bad_alloc &) {
        delete r;
        return fail(JITNN_HIP_ENOMEM, "out of host memory");
    }
    r->rot = rot;
    r->interleaved = interleaved;
    const int kind = sc ? sc->kind : JITNN_HIP_ROPE_PLAIN;
    constexpr long double two_pi = 6.283185307179586476925286766559L;
    double lo = 0, hi = 0;
    if (kind == JITNN_HIP_ROPE_YARN) {
        // the pair that turns beta times in the original context
        auto pair_of = [&](double beta) { return rot * log(sc->original_context / ((double)two_pi * beta)) / (2.0 * log(theta)); };
        lo = std::max(0.0, floor(pair_of(sc->beta_fast)));
        hi = std::min((double)rot - 1, ceil(pair_of(sc->beta_slow)));
        r->magnitude = 0.1 * log(sc->factor) + 1.0;
    }
    if (sc && sc->attention_factor != 0.0) r->magnitude = sc->attention_factor;
    for (int i = 0; i < rot / 2; ++i) {
        double f = pow(theta, -2.0 * i / rot), ramp = 0;
        if (factors) f /= (double)factors[i];
        if (kind == JITNN_HIP_ROPE_LINEAR) f /= sc->factor;
        if (kind == JITNN_HIP_ROPE_YARN) {
            ramp = std::min(1.0, std::max(0.0, (i - lo) / std::max(hi - lo, 0.001)));
            f = f * (1.0 - ramp) + f / sc->factor * ramp;
        }
        r->frequency[i] = f;
        // All 64 bits of the fraction of a turn, from the same formulas in 80-bit numbers: the 53 of a double are off by 2.6e-7 at position 2^31.
        long double whole = powl((long double)theta, -2.0L * i / rot);
        if (factors) whole /= (long double)factors[i];
        if (kind == JITNN_HIP_ROPE_LINEAR) whole /= (long double)sc->factor;
        if (kind == JITNN_HIP_ROPE_YARN) whole = whole * (1.0L - ramp) + whole / (long double)sc->factor * ramp;
        const long double turn = whole / two_pi, part = turn - floorl(turn);  // (positions are whole: whole turns of a frequency are none)
        turns[i] = part > 0 ? (unsigned long long)fminl(ldexpl(part, 64) + 0.5L, 18446744073709551615.0L) : 0;
    }
    const size_t bytes = turns.size() * sizeof(turns[0]);
    if (hipMalloc(&r->turns, bytes) != hipSuccess) {
        (void)hipGetLastError();
        r->turns = nullptr;
        rope_drop(r);
        return fail(JITNN_HIP_ENOMEM, "no %zu bytes of device memory for the rotary frequencies", bytes);
    }
    const hipError_t e = hipMemcpy(r->turns, turns.data(), bytes, hipMemcpyHostToDevice);
    if (e != hipSuccess) {
        rope_drop(r);
        return fail(JITNN_HIP_EDEVICE, "copying the rotary frequencies: %s", hipGetErrorString(e));
    }
    *out = r;
    return JITNN_HIP_OK;
}

}  // namespace

extern "C" {

int jitnn_hip_rope_create(int rot_dim, int interleaved, double theta, const jitnn_hip_rope_scaling *scaling, const float *freq_factors, jitnn_hip_rope **out) {
    if (!out) return fail(JITNN_HIP_EINVAL, "out is NULL");
    *out = nullptr;
    if (rot_dim < 2 || rot_dim > 1024 || rot_dim % 2 != 0) return fail(JITNN_HIP_EINVAL, "rot_dim %d (even, 2 to 1024)", rot_dim);
    if (!(theta > 0) || !std::isfinite(theta)) return fail(JITNN_HIP_EINVAL, "theta %g", theta);
    if (scaling) {
        if (scaling->kind < JITNN_HIP_ROPE_PLAIN || scaling->kind > JITNN_HIP_ROPE_YARN) return fail(JITNN_HIP_EINVAL, "rotary scaling %d", scaling->kind);
        if (scaling->kind != JITNN_HIP_ROPE_PLAIN && (!(scaling->factor > 0) || !std::isfinite(scaling->factor)))
            return fail(JITNN_HIP_EINVAL, "rotary scaling factor %g", scaling->factor);
        if (scaling->kind == JITNN_HIP_ROPE_YARN &&
            (scaling->original_context < 1 || !(scaling->beta_slow > 0) || !(scaling->beta_fast >= scaling->beta_slow) || !std::isfinite(scaling->beta_fast) || theta == 1.0))
            return fail(JITNN_HIP_EINVAL, "original context %d, beta_fast %g, beta_slow %g, theta %g", scaling->original_context, scaling->beta_fast, scaling->beta_slow, theta);
        if (!std::isfinite(scaling->attention_factor) || scaling->attention_factor < 0) return fail(JITNN_HIP_EINVAL, "attention factor %g", scaling->attention_factor);
    }
    for (int i = 0; freq_factors && i < rot_dim / 2; ++i)
        if (!(freq_factors[i] > 0) || !std::isfinite(freq_factors[i])) return fail(JITNN_HIP_EINVAL, "frequency factor %g of pair %d", (double)freq_factors[i], i);
    if (int rc = check_ready()) return rc;
    return rope_build(rot_dim, interleaved != 0, theta, scaling, freq_factors, out);
}

int jitnn_hip_rope_free(jitnn_hip_rope *r) {
    rope_drop(r);
    return JITNN_HIP_OK;
}

int jitnn_hip_rope_dev(const jitnn_hip_rope *r, const float *x_dev, long long x_stride, const int *positions_dev, int tokens, int heads, int head_dim, float *y_dev,
                       long long y_stride, void *stream) {
    if (!r) return fail(JITNN_HIP_EINVAL, "rope is NULL");
    if (tokens < 0 || heads < 1 || head_dim < r->rot || head_dim > 65536 || heads > 65536)
        return fail(JITNN_HIP_EINVAL, "%d tokens, %d heads of %d values (rot_dim %d)", tokens, heads, head_dim, r->rot);
    if (tokens == 0) return JITNN_HIP_OK;
    if (!x_dev || !positions_dev || !y_dev) return fail(JITNN_HIP_EINVAL, "NULL argument");
    const long long row = (long long)heads * head_dim;
    if (x_stride < row || y_stride < row) return fail(JITNN_HIP_EINVAL, "strides %lld and %lld of rows of %lld values", x_stride, y_stride, row);
    if (x_dev == y_dev && x_stride != y_stride) return fail(JITNN_HIP_EINVAL, "in place with strides %lld and %lld", x_stride, y_stride);
    RopeArgs a;
    a.x = x_dev;
    a.y = y_dev;
    a.positions = positions_dev;
    a.turns = r->turns;
    a.x_stride = x_stride;
    a.y_stride = y_stride;
    a.magnitude = (float)r->magnitude;
    a.tokens = tokens;
    a.heads = heads;
    a.D = head_dim;
    a.rot = r->rot;
    a.interleaved = r->interleaved;
    rope_launch(a, g.cus, (hipStream_t)stream);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

}  // extern "C"

// ================================================================================================ a batch over a paged cache

struct jitnn_hip_paged_cache {
    int layers, kv, hd, pages, page_tokens, type;
    uint8_t *k, *v;
    bool owned;
    size_t page_bytes() const { return (size_t)kv * page_tokens * hd * (type == 0 ? 4 : 2); }
    size_t layer_bytes() const { return page_bytes() * pages; }
    int page_shift() const { return __builtin_ctz((unsigned)page_tokens); }
};

namespace {

int check_cache(const jitnn_hip_paged_cache *c, int layer) {
    if (!c) return fail(JITNN_HIP_EINVAL, "cache is NULL");
    if (layer < 0 || layer >= c->layers) return fail(JITNN_HIP_EINVAL, "layer %d of %d", layer, c->layers);
    return JITNN_HIP_OK;
}

// The numbers of a batch; what its arrays hold is the kernels' to check.
int check_batch(const jitnn_hip_paged_cache *c, const jitnn_hip_batch *b) {
    if (!b) return fail(JITNN_HIP_EINVAL, "batch is NULL");
    if (b->sequences < 0 || b->tokens < 0 || b->max_tokens < 0 || b->max_len < 0 || b->shared_pages < 0 || b->table_stride < 0 || b->sequences > 65535)
        return fail(JITNN_HIP_EINVAL, "%d sequences, %d tokens (at most %d each), lengths to %d, %d shared of %d pages", b->sequences, b->tokens, b->max_tokens, b->max_len,
                    b->shared_pages, b->table_stride);
    if (b->max_len > 1 << 30) return fail(JITNN_HIP_EINVAL, "lengths to %d (at most 2^30)", b->max_len);
    if (b->shared_pages > b->table_stride || (long long)b->max_len > (long long)b->table_stride * c->page_tokens)
        return fail(JITNN_HIP_EINVAL, "lengths to %d and %d shared pages in tables of %d pages of %d", b->max_len, b->shared_pages, b->table_stride, c->page_tokens);
    if (b->tokens > 0 && b->sequences > 0 && (!b->starts || !b->lens || (!b->tables && b->table_stride > 0))) return fail(JITNN_HIP_EINVAL, "NULL array of the batch");
    return JITNN_HIP_OK;
}

// the positions that all sequences share (none behind the longest)
int batch_shared(const jitnn_hip_paged_cache *c, const jitnn_hip_batch *b) {
    return (int)(std::min<long long>(b->shared_pages, ((long long)b->max_len + c->page_tokens - 1) / c->page_tokens) * c->page_tokens);
}

int check_heads(const jitnn_hip_paged_cache *c, int heads) {
    if (heads < 1 || heads > 65535 || heads % c->kv != 0) return fail(JITNN_HIP_EINVAL, "%d query heads over %d key/value heads", heads, c->kv);
    return JITNN_HIP_OK;
}

AttnPlan attention_plan(const jitnn_hip_paged_cache *c, const jitnn_hip_batch *b, int heads) {
    return paged_attn_plan(c->type == 1, c->hd, heads, c->kv, b->sequences, b->tokens, std::min(std::max(b->max_tokens, 1), b->tokens), b->max_len, batch_shared(c, b), g.cus);
}

// the size of a cache, or what is wrong with it
long long cache_nbytes(int layers, int kv_heads, int head_dim, int pages, int page_tokens, int type) {
    if (layers < 1 || kv_heads < 1 || kv_heads > 65535 || pages < 1) return fail(JITNN_HIP_EINVAL, "%d layers, %d key/value heads, %d pages", layers, kv_heads, pages);
    if (head_dim != 64 && head_dim != 128 && head_dim != 192 && head_dim != 256) return fail(JITNN_HIP_EINVAL, "head_dim %d (64, 128, 192 and 256 are built)", head_dim);
    if (page_tokens < 16 || page_tokens > 256 || (page_tokens & (page_tokens - 1)) != 0)
        return fail(JITNN_HIP_EINVAL, "pages of %d positions (16, 32, 64, 128 or 256)", page_tokens);
    if (type != 0 && type != 1) return fail(JITNN_HIP_EINVAL, "a cache of ggml type %d (F32 = 0 and F16 = 1 are built)", type);
    const __int128 n = (__int128)layers * kv_heads * head_dim * pages * page_tokens * (type == 0 ? 4 : 2);
    if (n > ((__int128)1 << 46)) return fail(JITNN_HIP_EINVAL, "%d layers of %d pages do not fit any memory", layers, pages);
    return (long long)n;
}

int append_rows(const jitnn_hip_paged_cache *c, int layer, const jitnn_hip_batch *b, const jitnn_hip_rope *r, bool interleaved, const float *q_dev, long long q_stride,
                int heads, float *q_out_dev, long long q_out_stride, const float *k_dev, long long k_stride, const float *v_dev, long long v_stride, hipStream_t stream) {
    if (int rc = check_cache(c, layer)) return rc;
    if (int rc = check_batch(c, b)) return rc;
    if (heads < 0 || heads > 65535) return fail(JITNN_HIP_EINVAL, "%d query heads", heads);
    if (b->tokens == 0 || b->sequences == 0) return JITNN_HIP_OK;
    if (!k_dev || !v_dev || (heads > 0 && (!q_dev || !q_out_dev))) return fail(JITNN_HIP_EINVAL, "NULL argument");
    const long long row = (long long)c->kv * c->hd, qrow = (long long)heads * c->hd;
    if (k_stride < row || v_stride < row || (heads > 0 && (q_stride < qrow || q_out_stride < qrow)))
        return fail(JITNN_HIP_EINVAL, "strides %lld, %lld, %lld, %lld of rows of %lld queries and %lld keys and values", q_stride, q_out_stride, k_stride, v_stride, qrow, row);
    if (heads > 0 && q_dev == q_out_dev && q_stride != q_out_stride) return fail(JITNN_HIP_EINVAL, "in place with strides %lld and %lld", q_stride, q_out_stride);
    if (r && r->rot > c->hd) return fail(JITNN_HIP_EINVAL, "rot_dim %d of heads of %d values", r->rot, c->hd);
    if (r && r->rot % 8 != 0) return fail(JITNN_HIP_EUNSUPPORTED, "rot_dim %d is not a multiple of 8", r->rot);
    const uintptr_t all = (uintptr_t)k_dev | (uintptr_t)v_dev | (heads > 0 ? (uintptr_t)q_dev | (uintptr_t)q_out_dev : 0);
    if ((all & 15) != 0 || ((k_stride | v_stride | (heads > 0 ? q_stride | q_out_stride : 0)) & 3) != 0)
        return fail(JITNN_HIP_EUNSUPPORTED, "rows that are not aligned to 16 bytes");
    if (int rc = check_ready()) return rc;
    AppendArgs a;
    a.q = q_dev;
    a.k = k_dev;
    a.v = v_dev;
    a.q_out = q_out_dev;
    a.k_pages = c->k + (size_t)layer * c->layer_bytes();
    a.v_pages = c->v + (size_t)layer * c->layer_bytes();
    a.tables = b->tables;
    a.starts = b->starts;
    a.lens = b->lens;
    a.turns = r ? r->turns : nullptr;
    a.q_stride = q_stride;
    a.q_out_stride = q_out_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.magnitude = r ? (float)r->magnitude : 1.f;
    a.tokens = b->tokens;
    a.sequences = b->sequences;
    a.table_stride = b->table_stride;
    a.pages = c->pages;
    a.page_shift = c->page_shift();
    a.heads = heads;
    a.kv = c->kv;
    a.D = c->hd;
    a.rot = r ? r->rot : 0;
    a.interleaved = interleaved;
    paged_append_launch(c->type == 1, a, g.cus, stream);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

}  // namespace

extern "C" {

long long jitnn_hip_paged_cache_nbytes(int layers, int kv_heads, int head_dim, int pages, int page_tokens, int ggml_type) {
    return cache_nbytes(layers, kv_heads, head_dim, pages, page_tokens, ggml_type);
}

int jitnn_hip_paged_cache_wrap_dev(void *k_dev, void *v_dev, int layers, int kv_heads, int head_dim, int pages, int page_tokens, int ggml_type,
                                   jitnn_hip_paged_cache **out) {
    if (!out) return fail(JITNN_HIP_EINVAL, "out is NULL");
    *out = nullptr;
    const long long n = cache_nbytes(layers, kv_heads, head_dim, pages, page_tokens, ggml_type);
    if (n < 0) return (int)n;
    if (!k_dev || !v_dev || ((uintptr_t)k_dev & 15) != 0 || ((uintptr_t)v_dev & 15) != 0) return fail(JITNN_HIP_EINVAL, "cache memory is NULL or not aligned to 16 bytes");
    jitnn_hip_paged_cache *c = new (std::nothrow) jitnn_hip_paged_cache{layers, kv_heads, head_dim, pages, page_tokens, ggml_type, (uint8_t *)k_dev, (uint8_t *)v_dev, false};
    if (!c) return fail(JITNN_HIP_ENOMEM, "out of host memory");
    *out = c;
    return JITNN_HIP_OK;
}

int jitnn_hip_paged_cache_create(int layers, int kv_heads, int head_dim, int pages, int page_tokens, int ggml_type, jitnn_hip_paged_cache **out) {
    if (!out) return fail(JITNN_HIP_EINVAL, "out is NULL");
    *out = nullptr;
    const long long n = cache_nbytes(layers, kv_heads, head_dim, pages, page_tokens, ggml_type);
    if (n < 0) return (int)n;
    if (int rc = check_ready()) return rc;
    void *k = nullptr, *v = nullptr;
    if (hipMalloc(&k, (size_t)n) != hipSuccess || hipMalloc(&v, (size_t)n) != hipSuccess) {
        (void)hipGetLastError();
        if (k) (void)hipFree(k);
        return fail(JITNN_HIP_ENOMEM, "no 2 x %lld bytes of device memory for the cache", n);
    }
    const int rc = jitnn_hip_paged_cache_wrap_dev(k, v, layers, kv_heads, head_dim, pages, page_tokens, ggml_type, out);
    if (rc) {
        (void)hipFree(k);
        (void)hipFree(v);
        return rc;
    }
    (*out)->owned = true;
    return JITNN_HIP_OK;
}

int jitnn_hip_paged_cache_free(jitnn_hip_paged_cache *c) {
    if (!c) return JITNN_HIP_OK;
    if (c->owned) {
        (void)hipFree(c->k);
        (void)hipFree(c->v);
    }
    delete c;
    return JITNN_HIP_OK;
}

int jitnn_hip_paged_cache_copy_page_dev(const jitnn_hip_paged_cache *c, int from, int to, void *stream) {
    if (!c) return fail(JITNN_HIP_EINVAL, "cache is NULL");
    if (from < 0 || from >= c->pages || to < 0 || to >= c->pages) return fail(JITNN_HIP_EINVAL, "page %d to %d of %d", from, to, c->pages);
    if (from == to) return JITNN_HIP_OK;
    if (int rc = check_ready()) return rc;
    paged_copy_launch(c->k, c->v, (long long)c->page_bytes(), (long long)c->layer_bytes(), c->layers, from, to, (hipStream_t)stream);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int jitnn_hip_paged_append_dev(const jitnn_hip_paged_cache *c, int layer, const jitnn_hip_batch *b, const jitnn_hip_rope *r, const float *q_dev, long long q_stride,
                               int heads, float *q_out_dev, long long q_out_stride, const float *k_dev, long long k_stride, const float *v_dev, long long v_stride,
                               void *stream) {
    return append_rows(c, layer, b, r, r && r->interleaved, q_dev, q_stride, heads, q_out_dev, q_out_stride, k_dev, k_stride, v_dev, v_stride, (hipStream_t)stream);
}

long long jitnn_hip_paged_attention_workspace(const jitnn_hip_paged_cache *c, const jitnn_hip_batch *b, int heads) {
    if (int rc = check_cache(c, 0)) return rc;
    if (int rc = check_batch(c, b)) return rc;
    if (int rc = check_heads(c, heads)) return rc;
    if (b->tokens == 0 || b->sequences == 0) return 0;
    if (int rc = check_ready()) return rc;
    return (long long)attention_plan(c, b, heads).workspace(b->tokens, heads, c->hd);
}

int jitnn_hip_paged_attention_dev(const jitnn_hip_paged_cache *c, int layer, const jitnn_hip_batch *b, int heads, const float *q_dev, long long q_stride, float scale,
                                  float *y_dev, long long y_stride, void *workspace_dev, long long workspace_bytes, void *stream) {
    if (int rc = check_cache(c, layer)) return rc;
    if (int rc = check_batch(c, b)) return rc;
    if (int rc = check_heads(c, heads)) return rc;
    if (!std::isfinite(scale)) return fail(JITNN_HIP_EINVAL, "scale %g", (double)scale);
    if (b->tokens == 0 || b->sequences == 0) return JITNN_HIP_OK;
    if (!q_dev || !y_dev) return fail(JITNN_HIP_EINVAL, "NULL argument");
    const long long row = (long long)heads * c->hd;
    if (q_stride < row || y_stride < row) return fail(JITNN_HIP_EINVAL, "strides %lld and %lld of rows of %lld values", q_stride, y_stride, row);
    if (int rc = check_ready()) return rc;
    const AttnPlan p = attention_plan(c, b, heads);
    const size_t need = p.workspace(b->tokens, heads, c->hd);
    if (need > 0 && (!workspace_dev || workspace_bytes < (long long)need || ((uintptr_t)workspace_dev & 15) != 0))
        return fail(JITNN_HIP_EINVAL, "a workspace of %lld bytes, %zu are needed (aligned to 16)", workspace_dev ? workspace_bytes : 0ll, need);
    const long long units = (long long)p.own.spans * c->kv * b->sequences * p.own.blocks + (long long)p.ahead.spans * c->kv * p.ahead.blocks,
                    merges = (long long)b->tokens * heads;
    // (a launch holds fewer than 2^32 threads; the order of the workgroups may leave as many of them empty as there are)
    if (units > (1 << 22) || merges > (1 << 28) || (need > 0 && merges >= (1 << 24))) return fail(JITNN_HIP_EINVAL, "%d sequences of up to %d tokens are too many for one pass", b->sequences, b->max_tokens);
    AttnArgs a;
    a.k = c->k + (size_t)layer * c->layer_bytes();
    a.v = c->v + (size_t)layer * c->layer_bytes();
    a.q = q_dev;
    a.y = y_dev;
    a.part = need ? (float *)workspace_dev : nullptr;
    a.stat = need ? a.part + (size_t)b->tokens * heads * p.spans() * c->hd : nullptr;
    a.tables = b->tables;
    a.starts = b->starts;
    a.lens = b->lens;
    a.q_stride = q_stride;
    a.y_stride = y_stride;
    a.scale = (float)((double)scale * 1.44269504088896340736);
    a.tokens = b->tokens;
    a.sequences = b->sequences;
    a.heads = heads;
    a.kv = c->kv;
    a.pages = c->pages;
    a.page_shift = c->page_shift();
    a.table_stride = b->table_stride;
    a.max_len = b->max_len;
    a.shared = batch_shared(c, b);
    a.ahead = p.ahead;
    a.own = p.own;
    paged_attn_launch(c->type == 1, c->hd, g.cus, (hipStream_t)stream, a);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

// ---- drafted tokens

static int check_drafts(int rows, int sequences, int vocab) {
    if (rows < 0 || sequences < 0 || vocab < 1 || rows > 65535 || sequences > 65535 || vocab > 1 << 30)
        return fail(JITNN_HIP_EINVAL, "%d rows of %d sequences (at most 65535) over a vocabulary of %d (at most 2^30)", rows, sequences, vocab);
    return JITNN_HIP_OK;
}

long long jitnn_hip_verify_workspace(int rows, int sequences, int vocab) {
    if (int rc = check_drafts(rows, sequences, vocab)) return rc;
    return (long long)verify_workspace(rows, sequences, vocab);
}

int jitnn_hip_verify_drafts_dev(const float *logits_dev, long long logits_stride, int rows, int vocab, const int *starts_dev, int sequences, const int *tokens_dev,
                                const float *draft_probs_dev, long long draft_stride, const float *temperatures_dev, const float *uniforms_dev, int *out_dev,
                                int *accepted_dev, void *workspace_dev, long long workspace_bytes, void *stream) {
    if (int rc = check_drafts(rows, sequences, vocab)) return rc;
    if (sequences == 0) return JITNN_HIP_OK;
    if (!starts_dev || !temperatures_dev || !accepted_dev || (rows > 0 && (!logits_dev || !tokens_dev || !uniforms_dev || !out_dev)))
        return fail(JITNN_HIP_EINVAL, "NULL argument");
    if (logits_stride < vocab || (draft_probs_dev && draft_stride < vocab)) return fail(JITNN_HIP_EINVAL, "strides %lld and %lld of rows of %d values", logits_stride, draft_stride, vocab);
    const size_t need = verify_workspace(rows, sequences, vocab);
    if (!workspace_dev || workspace_bytes < (long long)need || ((uintptr_t)workspace_dev & 15) != 0)
        return fail(JITNN_HIP_EINVAL, "a workspace of %lld bytes, %zu are needed (aligned to 16)", workspace_dev ? workspace_bytes : 0ll, need);
    if (int rc = check_ready()) return rc;
    VerifyArgs a;
    a.logits = logits_dev;
    a.draft_probs = draft_probs_dev;
    a.temperatures = temperatures_dev;
    a.uniforms = uniforms_dev;
    a.starts = starts_dev;
    a.tokens = tokens_dev;
    a.out = out_dev;
    a.accepted = accepted_dev;
    a.part = workspace_dev;
    a.logits_stride = logits_stride;
    a.draft_stride = draft_stride;
    a.rows = rows;
    a.vocab = vocab;
    a.sequences = sequences;
    a.chunks = 0;
    verify_launch(a, (hipStream_t)stream);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

}  // extern "C"

// ================================================================================================ mixtures of experts

struct jitnn_hip_router {
    int experts, d, used;
    bool sigmoid, normalise;
    float scale;
    float *w = nullptr, *bias = nullptr;  // [experts, d], [experts] (one allocation)
};

struct jitnn_hip_moe {
    const jitnn_hip_router *router;
    const jitnn_hip_weight *gate, *up, *down;
    int act, ffn;
};

namespace {

constexpr int ROUTER_PASS = 8192;  // tokens of a pass of the router alone
constexpr int MOE_PASS_SLOTS = 4096;  // places (tokens x used) of a pass through the experts
constexpr int MOE_MAX_VALUES = 1 << 17;  // of a row: the operands of a pass's rows are found by 32-bit offsets, 4096 rows x 512 columns x 1152 bytes

size_t pad256(size_t b) { return (b + 255) & ~(size_t)255; }

int moe_pass_tokens(const jitnn_hip_moe *m) { return std::max(1, MOE_PASS_SLOTS / m->router->used); }

bool experts_on_rows(const jitnn_hip_weight *w) { return gemv_rows_supported(w->fmt); }  // (Q5_0 and Q3_K blocks that were not rewritten have no operands)

// Gate and up in one launch of the matrix cores' kernels.
bool experts_pair(const jitnn_hip_moe *m) { return experts_on_rows(m->gate) && m->gate->fmt == m->up->fmt; }

// Experts that so many tokens meet, where every one is as likely as any other.
double moe_met(const jitnn_hip_router *r, int tokens) { return r->experts * (1 - std::pow(1 - (double)r->used / r->experts, tokens)); }

// Chunks of so many groups that so many tokens make, about.
double moe_chunks(const jitnn_hip_router *r, int tokens, int groups) {
    return moe_met(r, tokens) * std::max(1.0, (double)tokens * r->used / r->experts / (8 * groups));
}

// Groups of eight rows in a chunk of an expert's: what most experts have where every one is as likely as any other, so that their weights are read
// and decoded once; at most what the kernels hold; fewer where gate and up, which have no shares of K, would have no workgroup for three quarters of the CUs.  us with
// none asked for / half / three quarters / all: 229 tokens, four of nine experts of 2560 x 512, Q4_K and Q5_K 112 / 78 / 71 / 72; 256, two of eight of 2048 x 2048 108 / 105 / 99 / 121;
// 512, two of eight of 1024 x 1024, Q4_K 76 / 64 / 66 / 66, Q8_0 96 / 95 / 101 / 101; 200, two of eight of 2048 x 1024, Q4_0 107 / 68 / 67 / 66.
int moe_groups(const jitnn_hip_moe *m, int tokens) {
    const jitnn_hip_router *r = m->router;
    const double mean = (double)tokens * r->used / r->experts;
    int groups = std::max(1, (int)std::ceil((mean + 2 * std::sqrt(mean)) / 8));
    for (const jitnn_hip_weight *w : {m->gate, m->up, m->down})
        if (experts_on_rows(w)) groups = std::min(groups, experts_rows_kernel_ref(w->fmt, groups, false).groups);
    if (!experts_pair(m)) return groups;
    auto workgroups = [&](int with) {
        const RowsKernelRef k = experts_rows_kernel_ref(m->gate->fmt, with, true);
        return moe_chunks(r, tokens, with) * ((m->ffn / 16 + k.tiles - 1) / k.tiles);
    };
    while (groups > 1 && 4 * workgroups(groups) < 3 * g.cus) groups = (groups + 1) / 2;
    return groups;
}

// Shares of the down projection's columns, where its workgroups alone would leave CUs idle: expected chunks x blocks against a workgroup for every CU (two of
// the small ones).
int moe_splits(const jitnn_hip_moe *m, int tokens, int groups) {
    if (!experts_on_rows(m->down)) return 1;
    const jitnn_hip_router *r = m->router;
    const RowsKernelRef k = experts_rows_kernel_ref(m->down->fmt, groups, false);
    const double blocks = moe_chunks(r, tokens, groups) * ((r->d / 16 + k.tiles - 1) / k.tiles);
    const int ncol = (m->ffn + 255) / 256, wanted = (int)std::ceil((k.threads > 256 ? 1.0 : 2.0) * g.cus / blocks);
    return std::max(1, std::min({wanted, 8, ncol / 4}));
}

// Few tokens: the INT8 products on the raw quants, for weights whose rows are whole chunks of 64 values.  (One token, seven of 36 experts of 512 x 13568, whose down projection
// comes in three parts that a launch more joins: 45 us, by the other route 71.)  They read an expert once for each token that meets it, but as
// fast as the memory gives, in three launches; the matrix cores' route reads it once, at two thirds of that, between six launches that cost what 120 MB do.  Both, rows
// / few, us: two of eight experts of 4096 x 14336, Q4_K and Q6_K, 1 token 93 / 49, 4 228 / 147, 6 256 / 218, 8 264 / 265, 12 278 / 406; four of 16 of 4096 x 2048, Q5_K,
// 4 87 / 67, 5 88 / 84, 6 89 / 98, 16 99 / 222; eight of 128 of 2048 x 768, 1 49 / 21, 8 84 / 52, 16 103 / 89, 24 127 / 136, 32 137 / 169; six of 64 of 2048 x 1408, Q8_0,
// 5 97 / 53, 16 152 / 127, 24 168 / 194; eight of 64 of 5120 x 1536 8 215 / 178, 12 264 / 268; two of eight of 4096 x 1024, Q6_K, 1 61 / 16, 12 63 / 44, 16 63 / 48, 24 55 / 77;
// eight of 256 of 2048 x 512, Q4_0, 16 109 / 49, 32 157 / 78, 64 208 / 130; two of 32 of 1024 x 2048, 32 50 / 38, 48 52 / 60.  Not measured with more tokens.
constexpr int MOE_FEW_TOKENS = 64;
bool moe_few(const jitnn_hip_moe *m, int tokens) {
    if (!g.gemv_i8 || tokens > MOE_FEW_TOKENS || m->gate->fmt != m->up->fmt) return false;
    for (const jitnn_hip_weight *w : {m->gate, m->up, m->down})
        if (w->nbytes >= (1ll << 32) || ((uintptr_t)w->dev & 3) != 0) return false;
    if (!experts_few_up_supported(m->gate->fmt, m->router->d) || !experts_few_down_supported(m->down->fmt, m->ffn, m->router->used)) return false;
    // (a wave takes 1024 values of a row of gate and up, whatever there are: 512 cost as much)
    const double pair = (double)(m->gate->nbytes + m->up->nbytes), down = (double)m->down->nbytes, whole = (m->router->d + 1023) / 1024 * 1024.0 / m->router->d;
    const double each = (double)tokens * m->router->used, met = 1.5 * moe_met(m->router, tokens);
    return tokens == 1 || (each * (pair * whole + down) - met * (pair + down)) / m->router->experts <= 120e6;
}

// What a pass of `tokens` keeps in the workspace, in bytes from its start.
struct MoeLayout {
    size_t logits, ids, weights, list, chunks, ops[GR_LAYOUTS], h_ops, g, u, part, total;
    bool layouts[GR_LAYOUTS];  // of x that gate and up ask for
    int groups, splits, chunks_most;
    bool few;
};
MoeLayout moe_layout(const jitnn_hip_moe *m, int tokens) {
    const jitnn_hip_router *r = m->router;
    const size_t slots = (size_t)tokens * r->used;
    MoeLayout l{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += pad256(bytes);
        return here;
    };
    l.few = moe_few(m, tokens);
    l.groups = moe_groups(m, tokens);
    l.splits = moe_splits(m, tokens, l.groups);
    l.chunks_most = ExpertLists::chunks_most((int)slots, r->experts, 8 * l.groups);
    l.logits = take(router_logits_bytes(tokens, r->experts, r->d, false));
    l.ids = take(slots * sizeof(int));
    l.weights = take(slots * sizeof(float));
    l.g = take(slots * m->ffn * sizeof(float));
    if (l.few) {
        const int parts = experts_few_down_parts(m->ffn, r->used);
        l.part = parts > 1 ? take((size_t)parts * tokens * r->d * sizeof(float)) : 0;
        l.total = at;
        return l;
    }
    l.list = take(slots * sizeof(int));
    l.chunks = take(((size_t)l.chunks_most + 1) * sizeof(int4));
    for (const jitnn_hip_weight *w : {m->gate, m->up})
        if (experts_on_rows(w)) l.layouts[gemv_rows_layout(w->fmt)] = true;
    for (int i = 0; i < GR_LAYOUTS; ++i) l.ops[i] = l.layouts[i] ? take(experts_ops_bytes(tokens, r->d)) : 0;
    l.h_ops = take(experts_on_rows(m->down) ? experts_ops_bytes(slots, m->ffn) : 0);
    l.u = take(experts_pair(m) ? 0 : slots * m->ffn * sizeof(float));  // (a pair's products meet in registers)
    l.part = take(slots * r->d * l.splits * sizeof(float));
    l.total = at;
    return l;
}

// The most that a pass of `from` to `to` tokens keeps there: fewer tokens may need more, for the down projection's splits and smaller chunks.
long long moe_most(const jitnn_hip_moe *m, int from, int to) {
    long long most = 0;
    for (int t = std::min(to, moe_pass_tokens(m)); t >= from; --t) most = std::max(most, (long long)moe_layout(m, t).total);
    return most;
}
// Layers of one kind have one workspace's size.
bool moe_alike(const jitnn_hip_moe *a, const jitnn_hip_moe *b) {
    auto same = [](const jitnn_hip_weight *v, const jitnn_hip_weight *w) { return v->fmt == w->fmt && v->nbytes == w->nbytes && ((uintptr_t)v->dev & 3) == ((uintptr_t)w->dev & 3); };
    return a->ffn == b->ffn && a->router->experts == b->router->experts && a->router->used == b->router->used && a->router->d == b->router->d && same(a->gate, b->gate) &&
           same(a->up, b->up) && same(a->down, b->down);
}

RouterArgs router_args(const jitnn_hip_router *r, const float *x, int tokens, int *ids, float *weights, void *logits) {
    RouterArgs a{};
    a.x = x;
    a.w = r->w;
    a.bias = r->bias;
    a.logits = (double *)logits;
    a.ids = ids;
    a.weights = weights;
    a.tokens = tokens;
    a.experts = r->experts;
    a.d = r->d;
    a.used = r->used;
    a.sigmoid = r->sigmoid;
    a.normalise = r->normalise;
    a.scale = r->scale;
    return a;
}

ExpertLists moe_lists(uint8_t *ws, const MoeLayout &l) {
    ExpertLists lists;
    lists.list = (int *)(ws + l.list);
    lists.chunks = (int4 *)(ws + l.chunks);
    lists.chunk_rows = 8 * l.groups;
    return lists;
}

// The tokens' rows as operands, in the layouts that gate and up ask for.
ExpertPrepare moe_prepare(const jitnn_hip_moe *m, const float *x, int tokens, uint8_t *ws, const MoeLayout &l) {
    uint8_t *places[GR_LAYOUTS];
    for (int i = 0; i < GR_LAYOUTS; ++i) places[i] = l.layouts[i] ? ws + l.ops[i] : nullptr;
    return experts_prepare(x, tokens, m->router->d, places);
}

ExpertWeights expert_weights(const jitnn_hip_weight *w, int experts) {
    return {w->fmt, w->n / experts, w->k, w->dev, (size_t)(w->n / experts) * (size_t)(w->k / block_values(w->fmt)) * block_bytes(w->fmt)};
}

int check_moe_call(const jitnn_hip_moe *m, const float *x, int tokens, const float *res, const float *y, const void *ws, long long ws_bytes) {
    if (!m) return fail(JITNN_HIP_EINVAL, "the layer is NULL");
    if (tokens < 0) return fail(JITNN_HIP_EINVAL, "tokens = %d", tokens);
    if (tokens == 0) return JITNN_HIP_OK;
    if (!x || !y) return fail(JITNN_HIP_EINVAL, "input or output is NULL");
    if ((((uintptr_t)x | (uintptr_t)y | (uintptr_t)res) & 15) != 0) return fail(JITNN_HIP_EINVAL, "input, residual and output must be 16-byte aligned");
    const size_t bytes = (size_t)tokens * m->router->d * sizeof(float);
    for (const float *in : {x, res})  // (the same array is read before it is written, row by row; a shifted one is not)
        if (in && in != y && overlaps(in, y, bytes)) return fail(JITNN_HIP_EINVAL, "the output overlaps the input or the residual");
    const int pass = moe_pass_tokens(m);
    long long need = (long long)moe_layout(m, std::min(tokens, pass)).total;
    if (tokens > pass && tokens % pass) need = std::max(need, (long long)moe_layout(m, tokens % pass).total);
    if (!ws || ((uintptr_t)ws & 15) != 0 || ws_bytes < need) return fail(JITNN_HIP_EINVAL, "workspace of %lld bytes, 16-byte aligned, needed; got %lld", need, ws ? ws_bytes : 0);
    return check_ready();
}

// One pass: the experts of `tokens` tokens for given choices, whose lists and operands (moe_prepare) are made.  to_choose (few tokens): the choices are still to be made, of these logits, and go to ids and
// weights.
int moe_experts(const jitnn_hip_moe *m, const float *x, int tokens, const int *ids, const float *weights, const RouterArgs *to_choose, const float *res, float *y, uint8_t *ws, const MoeLayout &l,
                hipStream_t s) {
    const jitnn_hip_router *r = m->router;
    const int slots = tokens * r->used;
    float *gb = (float *)(ws + l.g), *ub = (float *)(ws + l.u), *part = (float *)(ws + l.part);
    if (l.few) {
        ExpertFewArgs a{};
        ExpertWeights e = expert_weights(m->gate, r->experts);
        a.w = m->gate->dev;
        a.w2 = m->up->dev;
        a.expert_bytes = e.expert_bytes;
        a.x = x;
        a.ids = ids;
        a.weights = weights;
        a.y = gb;
        a.n = e.n;
        a.k = e.k;
        a.used = r->used;
        a.experts = r->experts;
        a.act = m->act;
        if (to_choose) a.route = *to_choose;
        experts_few_up_launch(m->gate->fmt, a, tokens, g.cus, s);
        e = expert_weights(m->down, r->experts);
        a.w = m->down->dev;
        a.expert_bytes = e.expert_bytes;
        const int parts = experts_few_down_parts(m->ffn, r->used);
        a.x = gb;
        a.res = parts > 1 ? nullptr : res;
        a.y = parts > 1 ? part : y;
        a.n = e.n;
        a.k = e.k;
        experts_few_down_launch(m->down->fmt, a, tokens, g.cus, s);
        if (parts > 1) rows_join_launch(s, part, y, tokens, r->d, parts, nullptr, Epilogue{0, res}, (unsigned)g.cus);
        HIP_TRY(hipGetLastError());
        return JITNN_HIP_OK;
    }
    // out [slots, n] = the products of w (with w2: of both, gated) with rows [rows, k], whose operands stand at ops
    auto rows = [&](const jitnn_hip_weight *w, const jitnn_hip_weight *w2, const uint8_t *ops, int count, int per_row, int splits, float *out) -> int {
        const ExpertWeights e = expert_weights(w, r->experts);
        ExpertRowsArgs a{};
        a.w = w->dev;
        a.w2 = w2 ? w2->dev : nullptr;
        a.expert_bytes = e.expert_bytes;
        a.ops = ops;
        a.inv = (const float *)(ops + (experts_ops_bytes(count, w->k) - (size_t)count * ((w->k + 255) / 256) * sizeof(float)));
        a.list = (const int *)(ws + l.list);
        a.chunks = (const int4 *)(ws + l.chunks);
        a.y = out;
        a.n = e.n;
        a.k = e.k;
        a.experts = r->experts;
        a.per_row = per_row;
        a.act = m->act;
        a.splits = splits;
        a.split_floats = (size_t)slots * e.n;
        const RowsKernelRef k = experts_rows_kernel_ref(w->fmt, l.groups, w2 != nullptr);
        if (int rc = allow_lds((const void *)k.fn, k.lds)) return rc;
        experts_rows_launch(k, a, l.chunks_most, s);
        return JITNN_HIP_OK;
    };
    uint8_t *places[GR_LAYOUTS] = {};
    for (int i = 0; i < GR_LAYOUTS; ++i) places[i] = l.layouts[i] ? ws + l.ops[i] : nullptr;
    if (experts_pair(m)) {
        if (int rc = rows(m->gate, m->up, places[gemv_rows_layout(m->gate->fmt)], tokens, r->used, 1, gb)) return rc;
    } else {
        const jitnn_hip_weight *ws2[2] = {m->gate, m->up};
        float *outs[2] = {gb, ub};
        for (int i = 0; i < 2; ++i) {
            if (!experts_on_rows(ws2[i])) experts_value_launch(expert_weights(ws2[i], r->experts), r->experts, ids, slots, r->used, x, outs[i], s);
            else if (int rc = rows(ws2[i], nullptr, places[gemv_rows_layout(ws2[i]->fmt)], tokens, r->used, 1, outs[i])) return rc;
        }
        experts_gate_launch(m->act, gb, ub, gb, (size_t)slots * m->ffn, g.cus, s);
    }
    if (experts_on_rows(m->down)) {
        uint8_t *h_places[GR_LAYOUTS] = {};
        h_places[gemv_rows_layout(m->down->fmt)] = ws + l.h_ops;
        experts_prepare_launch(experts_prepare(gb, slots, m->ffn, h_places), s);
        if (int rc = rows(m->down, nullptr, ws + l.h_ops, slots, 1, l.splits, part)) return rc;
    } else {
        experts_value_launch(expert_weights(m->down, r->experts), r->experts, ids, slots, 1, gb, part, s);
    }
    experts_combine_launch(part, l.splits, ids, weights, res, y, tokens, r->used, r->experts, r->d, s);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

}  // namespace

extern "C" {

int jitnn_hip_router_create(int experts, int d_model, int used, int gating, int normalise, float scale, const float *weights_host, const float *selection_bias_host,
                            jitnn_hip_router **out) {
    if (!out) return fail(JITNN_HIP_EINVAL, "out is NULL");
    *out = nullptr;
    if (experts < 1 || experts > MAX_EXPERTS) return fail(JITNN_HIP_EINVAL, "%d experts (1 to %d)", experts, MAX_EXPERTS);
    if (used < 1 || used > experts || used > MAX_USED) return fail(JITNN_HIP_EINVAL, "%d of %d experts (at most %d)", used, experts, MAX_USED);
    if (d_model < 4 || d_model % 4 != 0) return fail(JITNN_HIP_EINVAL, "d_model %d (a multiple of 4)", d_model);
    if (gating != JITNN_HIP_GATING_SOFTMAX && gating != JITNN_HIP_GATING_SIGMOID) return fail(JITNN_HIP_EINVAL, "gating %d", gating);
    if (!std::isfinite(scale)) return fail(JITNN_HIP_EINVAL, "scale %g", (double)scale);
    if (!weights_host) return fail(JITNN_HIP_EINVAL, "weights are NULL");
    if (int rc = check_ready()) return rc;
    jitnn_hip_router *r = new (std::nothrow) jitnn_hip_router{experts, d_model, used, gating == JITNN_HIP_GATING_SIGMOID, normalise != 0, scale};
    if (!r) return fail(JITNN_HIP_ENOMEM, "out of host memory");
    const size_t count = (size_t)experts * d_model, bytes = (count + experts) * sizeof(float);
    if (hipMalloc(&r->w, bytes) != hipSuccess) {
        (void)hipGetLastError();
        delete r;
        return fail(JITNN_HIP_ENOMEM, "no %zu bytes of device memory for the router", bytes);
    }
    hipError_t e = hipMemcpy(r->w, weights_host, count * sizeof(float), hipMemcpyHostToDevice);
    if (e == hipSuccess && selection_bias_host) {
        r->bias = r->w + count;
        e = hipMemcpy(r->bias, selection_bias_host, (size_t)experts * sizeof(float), hipMemcpyHostToDevice);
    }
    if (e != hipSuccess) {
        (void)hipFree(r->w);
        delete r;
        return fail(JITNN_HIP_EDEVICE, "copying the router: %s", hipGetErrorString(e));
    }
    *out = r;
    return JITNN_HIP_OK;
}

int jitnn_hip_router_free(jitnn_hip_router *r) {
    if (!r) return JITNN_HIP_OK;
    (void)hipFree(r->w);
    delete r;
    return JITNN_HIP_OK;
}

long long jitnn_hip_router_workspace(const jitnn_hip_router *r, int tokens) {
    if (!r) return fail(JITNN_HIP_EINVAL, "the router is NULL");
    if (tokens < 0) return fail(JITNN_HIP_EINVAL, "tokens = %d", tokens);
    long long most = 0;  // (fewer tokens may need more: sums in splits)
    for (int t = std::min(tokens, ROUTER_PASS); t > 0; --t) most = std::max(most, (long long)router_logits_bytes(t, r->experts, r->d, true));
    return most;
}

int jitnn_hip_router_dev(const jitnn_hip_router *r, const float *x_dev, int tokens, int *ids_dev, float *weights_dev, void *workspace_dev, long long workspace_bytes,
                         void *stream) {
    if (!r) return fail(JITNN_HIP_EINVAL, "the router is NULL");
    if (tokens < 0) return fail(JITNN_HIP_EINVAL, "tokens = %d", tokens);
    if (tokens == 0) return JITNN_HIP_OK;
    if (!x_dev || !ids_dev || !weights_dev) return fail(JITNN_HIP_EINVAL, "input or output is NULL");
    if (((uintptr_t)x_dev & 15) != 0) return fail(JITNN_HIP_EINVAL, "the input must be 16-byte aligned");
    long long need = 0;
    for (const int t : {std::min(tokens, ROUTER_PASS), tokens % ROUTER_PASS})
        if (t) need = std::max(need, (long long)router_logits_bytes(t, r->experts, r->d, true));
    if (need > 0 && (!workspace_dev || ((uintptr_t)workspace_dev & 15) != 0 || workspace_bytes < need))
        return fail(JITNN_HIP_EINVAL, "workspace of %lld bytes, 16-byte aligned, needed; got %lld", need, workspace_dev ? workspace_bytes : 0);
    if (int rc = check_ready()) return rc;
    for (int t = 0; t < tokens; t += ROUTER_PASS)
        router_launch(router_args(r, x_dev + (size_t)t * r->d, std::min(ROUTER_PASS, tokens - t), ids_dev + (size_t)t * r->used, weights_dev + (size_t)t * r->used, workspace_dev),
                      (hipStream_t)stream);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int jitnn_hip_moe_create(const jitnn_hip_router *router, const jitnn_hip_weight *gate, const jitnn_hip_weight *up, const jitnn_hip_weight *down, int activation,
                         jitnn_hip_moe **out) {
    if (!out) return fail(JITNN_HIP_EINVAL, "out is NULL");
    *out = nullptr;
    if (!router || !gate || !up || !down) return fail(JITNN_HIP_EINVAL, "router or weight is NULL");
    if (activation < 0 || activation >= ACT_COUNT) return fail(JITNN_HIP_EINVAL, "activation %d", activation);
    const int e = router->experts, d = router->d, ffn = down->k;
    if (gate->k != d || up->k != d || (long long)e * ffn != gate->n || gate->n != up->n || (long long)e * d != down->n)
        return fail(JITNN_HIP_EINVAL, "experts of shapes gate [%d, %d], up [%d, %d], down [%d, %d] for a router of %d experts on %d values", gate->n, gate->k, up->n, up->k, down->n,
                    down->k, e, d);
    if (d > MOE_MAX_VALUES || ffn > MOE_MAX_VALUES) return fail(JITNN_HIP_EINVAL, "experts on %d and %d values (at most %d)", d, ffn, MOE_MAX_VALUES);
    jitnn_hip_moe *m = new (std::nothrow) jitnn_hip_moe{router, gate, up, down, activation, ffn};
    if (!m) return fail(JITNN_HIP_ENOMEM, "out of host memory");
    *out = m;
    return JITNN_HIP_OK;
}

int jitnn_hip_moe_free(jitnn_hip_moe *m) {
    delete m;
    return JITNN_HIP_OK;
}

long long jitnn_hip_moe_workspace(const jitnn_hip_moe *m, int tokens) {
    if (!m) return fail(JITNN_HIP_EINVAL, "the layer is NULL");
    if (tokens < 0) return fail(JITNN_HIP_EINVAL, "tokens = %d", tokens);
    return moe_most(m, 1, tokens);
}

int jitnn_hip_moe_dev(const jitnn_hip_moe *m, const float *x_dev, int tokens, const float *residual_dev, float *y_dev, void *workspace_dev, long long workspace_bytes, void *stream) {
    if (int rc = check_moe_call(m, x_dev, tokens, residual_dev, y_dev, workspace_dev, workspace_bytes)) return rc;
    const int pass = moe_pass_tokens(m);
    uint8_t *ws = (uint8_t *)workspace_dev;
    for (int t = 0; t < tokens; t += pass) {
        const int count = std::min(pass, tokens - t), d = m->router->d;
        const MoeLayout l = moe_layout(m, count);
        const float *x = x_dev + (size_t)t * d;
        RouterArgs a = router_args(m->router, x, count, (int *)(ws + l.ids), (float *)(ws + l.weights), ws + l.logits);
        const bool choose_there = l.few && experts_few_chooses(a.experts);
        if (!l.few) {
            a.lists = moe_lists(ws, l);
            a.prepare = moe_prepare(m, x, count, ws, l);
        }
        if (choose_there) router_logits_launch(a, (hipStream_t)stream);
        else router_launch(a, (hipStream_t)stream);
        if (int rc = moe_experts(m, x, count, (const int *)(ws + l.ids), (const float *)(ws + l.weights), choose_there ? &a : nullptr, residual_dev ? residual_dev + (size_t)t * d : nullptr, y_dev + (size_t)t * d,
                                 ws, l, (hipStream_t)stream))
            return rc;
    }
    return JITNN_HIP_OK;
}

int jitnn_hip_moe_experts_dev(const jitnn_hip_moe *m, const float *x_dev, int tokens, const int *ids_dev, const float *weights_dev, const float *residual_dev, float *y_dev,
                              void *workspace_dev, long long workspace_bytes, void *stream) {
    if (int rc = check_moe_call(m, x_dev, tokens, residual_dev, y_dev, workspace_dev, workspace_bytes)) return rc;
    if (tokens > 0 && (!ids_dev || !weights_dev)) return fail(JITNN_HIP_EINVAL, "ids or weights are NULL");
    const int pass = moe_pass_tokens(m);
    for (int t = 0; t < tokens; t += pass) {
        const int count = std::min(pass, tokens - t), d = m->router->d, used = m->router->used;
        const MoeLayout l = moe_layout(m, count);
        const int *ids = ids_dev + (size_t)t * used;
        uint8_t *const ws = (uint8_t *)workspace_dev;
        const float *const x = x_dev + (size_t)t * d;
        if (!l.few) expert_lists_launch(ids, count * used, m->router->experts, moe_lists(ws, l), moe_prepare(m, x, count, ws, l), (hipStream_t)stream);
        if (int rc = moe_experts(m, x, count, ids, weights_dev + (size_t)t * used, nullptr, residual_dev ? residual_dev + (size_t)t * d : nullptr,
                                 y_dev + (size_t)t * d, ws, l, (hipStream_t)stream))
            return rc;
    }
    return JITNN_HIP_OK;
}

}  // extern "C"

// ================================================================================================ decode step

struct jitnn_hip_llama {
    int layers, d, heads, kv, hd, ffn, vocab, max_ctx;
    float eps, theta;
    const jitnn_hip_weight **w;  // [layers][7] then output
    const jitnn_hip_weight *w_out;
    const jitnn_hip_moe **moe;   // [layers]: the experts in place of a layer's gate, up and down, nullptr: it has those
    void *moe_ws[2];             // their workspace: of one token (decode steps), of up to moe_cap (passes of many), allocated with the many-token buffers
    size_t moe_ws_bytes[2];
    int moe_cap;
    float *norms;                // [layers][2][d] then output norm [d]
    float *kc, *vc;              // [layers][max_ctx][kv][hd]
    float *cosv, *sinv;          // [max_ctx][hd/2]
    float *xin, *xa, *xb, *xn, *q, *k, *v, *att, *gate, *up, *h, *part, *logits;  // (k and v: inside the buffer of q, behind it)
    int chunks_max;
    // many-token (prefill) buffers, [pf_cap, ...] each, allocated by the first prefill call and grown when a longer one comes
    int pf_cap;
    float *pf[11];  // xn, q, k, v, att, xa, xb, gate, up, h, the K slices of a linear whose join is deferred (8 x d per token)
    _Float16 *packed;  // keys and values of one layer as attn_packed_kernel reads them, up to max_ctx positions: allocated by the first long prompt
    bool no_packing;    // the caller's wish: packed stays as it is and unused
    int attention;      // the PromptAttention of the last prompt pass, -1: there was none
    int rope_interleaved;  // 0: rotate-half pairs (i, i + D/2); 1: pairs (2i, 2i + 1)
    jitnn_hip_rope *rope;  // what cosv and sinv hold, for positions of a paged cache (the pairing is rope_interleaved)
    void *paged_ws;        // workspace of the attention over a paged cache, grown by jitnn_hip_llama_step_dev
    size_t paged_ws_bytes;
    bool recorded;         // a pass over a paged cache has been recorded: buffers that its replays use are kept, not freed, where larger ones take their place
    struct Kept {
        void *p;
        Kept *next;
    } *kept;
    // token embedding table [vocab, d] in ggml type embd_fmt (F32 = 0, F16 = 1 or a block format), owned
    uint8_t *embd;
    int embd_fmt;
    int *tok_dev;   // [max_ctx] token ids of the generation loop (device)
    int *tok_pin;   // one token id in pinned host memory
};

namespace {

using AttnDecodeKernel = void (*)(const float *, const float *, const float *, float *, float *, float *, uint32_t, uint32_t);
template <int D, int P>
AttnDecodeKernel attn_split_of(int group) {
    switch (group) {
    case 1: return attn_split_kernel<D, 1, P>;
    case 2: return attn_split_kernel<D, 2, P>;
    case 3: return attn_split_kernel<D, 3, P>;
    default: return attn_split_kernel<D, 4, P>;
    }
}

// Passes of 8 keys per wave that one token's attention takes in attn_split_kernel, 0: attn_decode_kernel.  Both with their merge and what one
// waits for the other, us per layer more than the shortest cache takes, attn_decode_kernel / 2 / 4 passes: 32 heads of 128 values
// over 8, 700 keys 1.0 / 1.0 / 1.8, 1000 1.6 / 1.1 / 2.1, 1400 3.7 / 1.8 / 2.5 (more than 32 chunks: the merge takes its longer form), 2000
// 4.5 / 2.3 / 2.9, 3000 6.2 / 6.1 / 4.4, 4000 10.0 / 7.8 / 5.8, 8000 20.0 / 16.1 / 14.9; 8 over 8, 1000 1.4 / 0.7 / 0.5, 4000 9.1 / 6.0 / 3.7; 32
// heads of 64 values over 8, 1000 0.5 / 0.4 / 0.7, 4000 4.0 / 3.3 / 2.2.  Two passes while their workgroups have a CU each.
int attn_split_passes(int D, int group, int kv, int keys, int cus) {
    if ((D != 64 && D != 128) || group > AS_GMAX || keys < 1024) return 0;
    return (keys + as_keys(2) - 1) / as_keys(2) * kv <= cus ? 2 : 4;
}

template <int D>
void launch_attention(const jitnn_hip_llama *m, int layer, int pos, hipStream_t st) {
    const size_t lo = (size_t)layer * m->max_ctx * m->kv * m->hd;
    AttnDecodeKernel kernel = attn_decode_kernel<D>;
    int keys = AttCfg<D>::CH;  // of a chunk
    if constexpr (D == 64 || D == 128) {
        if (const int passes = attn_split_passes(D, m->heads / m->kv, m->kv, pos + 1, g.cus)) {
            kernel = passes == 2 ? attn_split_of<D, 2>(m->heads / m->kv) : attn_split_of<D, 4>(m->heads / m->kv);
            keys = as_keys(passes);
        }
    }
    const int chunks = (pos + keys) / keys;
    // (q, k, v: one buffer, see jitnn_hip_llama_create)
    hipLaunchKernelGGL(kernel, dim3(chunks, m->kv), dim3(256), 0, st, m->q, m->cosv, m->sinv, m->kc + lo, m->vc + lo, m->part, (uint32_t)m->heads | ((uint32_t)m->kv << 16),
                       (uint32_t)pos | (m->rope_interleaved ? 0x80000000u : 0u));
    constexpr int NPL = 1024 / D < 8 ? 1024 / D : 8;  // long contexts: more threads per value share the chunks
    if (chunks > 32) hipLaunchKernelGGL((attn_merge_kernel<D, NPL>), dim3(m->heads), dim3(NPL * D), 0, st, m->part, m->att, chunks);
    else hipLaunchKernelGGL((attn_merge_kernel<D, 2>), dim3(m->heads), dim3(2 * D), 0, st, m->part, m->att, chunks);
}

bool xreg_ok(const jitnn_hip_weight *w) { return w->k <= 4096 && !is_extra_format(w->fmt); }

// y_i = W_i RMSNorm(x; nw) for `count` (at most 3) weights over the same x.  Weights the register-resident kernel
// takes get the norm fused into their launch, neighbours of one format share the launch; anything else goes through
// a separate RMSNorm and the general GEMV.
int normed_linears(const jitnn_hip_llama *m, const jitnn_hip_weight *const *ws, float *const *ys, int count, const float *x, const float *nw,
                   hipStream_t st) {
    // runs of neighbours of one format and row length the register-resident kernel takes
    XregCall calls[3];
    int ncalls = 0;
    bool all = true;
    for (int i = 0; i < count;) {
        if (!xreg_ok(ws[i])) {
            all = false;
            break;
        }
        XregCall &c = calls[ncalls++];
        int j = 0;
        while (i + j < count && j < 3 && xreg_ok(ws[i + j]) && ws[i + j]->fmt == ws[i]->fmt && ws[i + j]->k == ws[i]->k) {
            c.w[j] = ws[i + j];
            c.y[j] = ys[i + j];
            ++j;
        }
        c.x = x;
        c.norm_w = nw;
        c.eps = m->eps;
        i += j;
    }
    if (all) {
        if (ncalls == 2 && calls[0].w[0]->k == calls[1].w[0]->k && calls[0].w[0]->k % 256 == 0 && xreg2_ok(calls[0].w[0]->fmt, calls[1].w[0]->fmt))
            return launch_xreg2(calls[0], calls[1], st);
        for (int c = 0; c < ncalls; ++c)
            if (int rc = launch_xreg(calls[c], st)) return rc;
        return JITNN_HIP_OK;
    }
    hipLaunchKernelGGL(rms_norm_kernel, dim3(1), dim3(256), 0, st, x, nw, m->xn, m->d, m->eps);
    for (int i = 0; i < count; ++i)
        if (int rc = launch_gemv(ws[i], m->xn, 1, nullptr, ys[i], st)) return rc;
    return JITNN_HIP_OK;
}

int check_model(const jitnn_hip_llama *m) {
    if (!m) return fail(JITNN_HIP_EINVAL, "model is NULL");
    for (int l = 0; l < m->layers; ++l)
        for (int i = 0; i < (m->moe[l] ? (int)JITNN_HIP_W_FFN_GATE : 7); ++i)
            if (!m->w[l * 7 + i]) return fail(JITNN_HIP_EINVAL, "layer %d has no weight %d", l, i);
    if (!m->w_out) return fail(JITNN_HIP_EINVAL, "no output weight");
    return JITNN_HIP_OK;
}

// bytes of every weight a step of the model reads (norm vectors included; of experts, as many as so many tokens can meet)
long long model_weight_bytes(const jitnn_hip_llama *m, int tokens) {
    long long b = m->w_out->nbytes + 4ll * (2 * m->layers + 1) * m->d;
    for (int l = 0; l < m->layers; ++l) {
        const jitnn_hip_moe *e = m->moe[l];
        for (int i = 0; i < (e ? (int)JITNN_HIP_W_FFN_GATE : 7); ++i) b += m->w[l * 7 + i]->nbytes;
        if (!e) continue;
        const long long met = std::min<long long>(e->router->experts, (long long)tokens * e->router->used);
        b += 4ll * e->router->experts * m->d + (long long)(e->gate->nbytes + e->up->nbytes + e->down->nbytes) / e->router->experts * met;
    }
    return b;
}

// ys[i] = RMSNorm(x) ws[i]^T for `rows` rows.  With more rows than the GEMV kernels take (and formats the many-row
// kernels know) the norm is part of the one activation preparation the weights share; otherwise it is a kernel of its
// own into `xn` [rows, d] and the linears take their usual route.
// The join of a linear's K slices that a caller deferred and nobody could fuse: prefill_join_kernel after all.
void flush_pending(PfPending &p, int rows, hipStream_t st) {
    if (!p.part) return;
    prefill_join_launch(p.part, nullptr, p.res, p.out, rows, p.n, p.splits, (unsigned)g.cus * 8, st);
    p = PfPending{};
}

// xn = RMSNorm(x) for `rows` rows; x - the output of the linear before - may still be in K slices, which meet here.
void norm_rows(const jitnn_hip_llama *m, const float *x, int rows, const float *nw, float *xn, hipStream_t st, PfPending *pend) {
    PfPending join;
    if (pend && pend->part && pend->out == x && pend->n == m->d && pend->res) {
        join = *pend;
        *pend = PfPending{};
    } else if (pend) {
        flush_pending(*pend, rows, st);
    }
    // (four values a load: the model's own rows are aligned to that; the caller's, in front of the first layer, need not be)
    const float *in = join.part ? join.res : x;
    if (((uintptr_t)in & 15) != 0) {
        flush_pending(join, rows, st);  // (slices of a many-row launch, whose preparation reads such rows 16 bytes at a time too)
        hipLaunchKernelGGL(rms_norm_rows_kernel, dim3(rows), dim3(256), 0, st, x, nw, xn, m->d, m->eps);
    } else {
        hipLaunchKernelGGL(rms_norm_rows_join_kernel, dim3(rows), dim3(NR_THREADS), 0, st, in, join.part, join.splits, join.out, nw, xn, rows, m->d, m->eps);
    }
}

// (pend: x - the output of the linear before - may still be in K slices; the shared preparation then adds them up)
int normed_linears_rows(const jitnn_hip_llama *m, const jitnn_hip_weight *const *ws, float *const *ys, int count, const float *x, int rows,
                        const float *nw, float *xn, hipStream_t st, PfPending *pend = nullptr, PfGroupPending *gdefer = nullptr) {
    bool group = rows > g.gemv_max_rows && prefill_prepare_fuses_norm(m->d);
    for (int i = 0; i < count; ++i) group = group && has_many_row_kernel(ws[i]->fmt);
    if (group) {
        const bool fused = pend && pend->part && pend->out == x && pend->n == m->d;
        const int rc = launch_prefill_group(ws, ys, count, x, rows, nullptr, nw, m->eps, st, nullptr, nullptr, nullptr, SCRATCH_THREAD, nullptr, nullptr,
                                            fused ? pend : nullptr, gdefer);
        if (fused) *pend = PfPending{};
        else if (pend) flush_pending(*pend, rows, st);  // (never both: a pending join is flushed before anybody reads its row)
        return rc;
    }
    norm_rows(m, x, rows, nw, xn, st, pend);
    // the one-pass kernel for several rows prepares its activation operands once for all the weights that take it
    bool shared = count > 1;
    for (int i = 0; i < count; ++i) shared = shared && rows_path(ws[i], rows);
    if (shared) {
        for (int i = 0; i < count; ++i) count_op(ST_GEMV, (long long)ws[i]->nbytes + 4ll * rows * ((long long)ws[i]->k + ws[i]->n));
        // (the slices in the buffer of the gate projection, which is written after they are read)
        return launch_rows_group(ws, ys, count, xn, rows, nullptr, nullptr, st, SCRATCH_THREAD, nullptr, nullptr, nullptr, m->pf[7], (size_t)rows * m->ffn, gdefer);
    }
    for (int i = 0; i < count; ++i)
        if (int rc = jitnn_hip_linear_dev(ws[i], xn, rows, nullptr, ys[i], (void *)st)) return rc;
    return JITNN_HIP_OK;
}

// y = res + x w^T for `rows` rows (tmp [rows, n] is scratch).  up != nullptr: the activations are silu(x) * up (the FFN's
// gate and up projections); on the many-row path they are formed inside the activation preparation, otherwise by
// swiglu_kernel into `h` [rows, k].
// part / defer: see launch_prefill_group - the join of the K slices may be left to the caller.
int residual_linear_rows(const jitnn_hip_weight *w, const float *x, int rows, const float *res, float *tmp, float *y, hipStream_t st,
                         const float *up = nullptr, float *h = nullptr, float *part = nullptr, PfPending *defer = nullptr) {
    const bool many = rows > g.gemv_max_rows && has_many_row_kernel(w->fmt) && w->n % 4 == 0;
    if (many && (!up || prefill_prepare_fuses_norm(w->k))) {
        return launch_prefill_group(&w, &y, 1, x, rows, nullptr, nullptr, 0.f, st, res, tmp, up, SCRATCH_THREAD, part, defer);
    }
    if (up && rows_path(w, rows)) {  // silu(x) * up is formed by the preparation of the one-pass kernel
        count_op(ST_GEMV, (long long)w->nbytes + 4ll * rows * ((long long)w->k + w->n));
        return launch_rows_group(&w, &y, 1, x, rows, nullptr, res, st, SCRATCH_THREAD, up, part, defer);
    }
    if (up) {
        const long long count = (long long)rows * w->k;
        const unsigned blocks = (unsigned)std::min<long long>((count + 1023) / 1024, (long long)g.cus * 16);
        hipLaunchKernelGGL(swiglu_kernel, dim3(blocks), dim3(256), 0, st, x, up, h, (int)count);
        x = h;
        if (many) return launch_prefill_group(&w, &y, 1, x, rows, nullptr, nullptr, 0.f, st, res, tmp);
    }
    if (rows_path(w, rows)) {  // the one-pass kernel adds the residual as it stores
        count_op(ST_GEMV, (long long)w->nbytes + 4ll * rows * ((long long)w->k + w->n));
        return launch_rows_group(&w, &y, 1, x, rows, nullptr, res, st, SCRATCH_THREAD, nullptr, part, defer);
    }
    if (int rc = jitnn_hip_linear_dev(w, x, rows, nullptr, tmp, (void *)st)) return rc;
    const size_t count4 = (size_t)rows * w->n / 4;
    const unsigned blocks = (unsigned)std::min<size_t>((count4 + 255) / 256, (size_t)g.cus * 8);
    hipLaunchKernelGGL(add_rows_kernel, dim3(blocks), dim3(256), 0, st, reinterpret_cast<const float4 *>(res), reinterpret_cast<const float4 *>(tmp),
                       reinterpret_cast<float4 *>(y), count4);
    return JITNN_HIP_OK;
}

// A buffer that a larger one replaces.
void release_or_keep(jitnn_hip_llama *m, void *p) {
    if (!p) return;
    jitnn_hip_llama::Kept *k = m->recorded ? new (std::nothrow) jitnn_hip_llama::Kept{p, m->kept} : nullptr;
    if (k) m->kept = k;
    else if (!m->recorded) (void)hipFree(p);  // (no memory to note it: left to the process)
}

// What the workspace of a model's experts has to be for passes of up to `tokens`, which 0: of one token's; less than there is where it has been made for as many.
size_t moe_need(const jitnn_hip_llama *m, int which, int tokens) {
    long long need = 0;
    const jitnn_hip_moe *last = nullptr;
    for (int l = 0; l < m->layers; ++l) {
        const jitnn_hip_moe *e = m->moe[l];
        if (!e || (last && moe_alike(e, last))) continue;
        need = std::max(need, moe_most(e, which ? m->moe_cap + 1 : 1, tokens));
        last = e;
    }
    return (size_t)need;
}

// That workspace.  The device may still use the old one.  A decode step's stays where there is no room for a larger one: the experts that are there go on.
int moe_reserve(jitnn_hip_llama *m, int which, int tokens) {
    const size_t need = moe_need(m, which, tokens);
    if (need <= m->moe_ws_bytes[which]) return JITNN_HIP_OK;
    HIP_TRY(hipDeviceSynchronize());
    auto alloc = [](size_t bytes) -> void * {
        void *p = nullptr;
        if (hipMalloc(&p, bytes) == hipSuccess) return p;
        (void)hipGetLastError();
        return nullptr;
    };
    const bool ok = replace_buffer(m->moe_ws[which], m->moe_ws_bytes[which], need, which != 0, alloc, [&](void *p) { release_or_keep(m, p); });
    if (which && !m->moe_ws[which]) m->moe_cap = 0;  // (the next pass asks for all it needs)
    return ok ? JITNN_HIP_OK : fail(JITNN_HIP_ENOMEM, "no %zu bytes of device memory for the experts of %d tokens", need, tokens);
}

// The many-token buffers of a model, for at least `tokens` rows.
int ensure_prefill(jitnn_hip_llama *m, int tokens) {
    if (tokens > m->moe_cap) {
        if (int rc = moe_reserve(m, 1, tokens)) return rc;
        m->moe_cap = tokens;
    }
    if (tokens <= m->pf_cap) return JITNN_HIP_OK;
    HIP_TRY(hipDeviceSynchronize());  // earlier calls may still use the old buffers
    m->pf_cap = 0;
    for (float *&b : m->pf) {
        release_or_keep(m, b);
        b = nullptr;
    }
    const size_t qd = (size_t)m->heads * m->hd, kd = (size_t)m->kv * m->hd;
    const size_t per[11] = {(size_t)m->d, qd, kd, kd, qd, (size_t)m->d, (size_t)m->d, (size_t)m->ffn, (size_t)m->ffn, (size_t)m->ffn, (size_t)8 * m->d};
    for (int i = 0; i < 11; ++i) {
        if (hipMalloc(&m->pf[i], per[i] * tokens * sizeof(float)) != hipSuccess) {
            (void)hipGetLastError();
            for (float *&b : m->pf) {
                if (b) (void)hipFree(b);
                b = nullptr;
            }
            return fail(JITNN_HIP_ENOMEM, "allocating the buffers of a %d-token prefill failed", tokens);
        }
    }
    m->pf_cap = tokens;
    return JITNN_HIP_OK;
}

// Grows the thread's scratch once, to what the largest launch of a prompt pass over dequantised weights takes, instead of
// step by step along the first layer (every growth waits for the device).  Where there is no room the launches ask, each for its own.
void prefill_reserve(const jitnn_hip_llama *m, int tokens, hipStream_t st) {
    if (stream_recording(st)) return;
    size_t most_weights = 0, most_operands = 0;
    WidePlan p;
    for (int l = 0; l < m->layers && tokens > g.gemv_max_rows; ++l) {
        const jitnn_hip_weight *const *w = m->w + (size_t)l * 7;
        auto want = [&](int which, int count, bool dual, bool residual) {
            if (!wide_pays(w + which, count, tokens, dual, residual, &p)) return;
            const int k = w[which]->k;
            most_weights = std::max(most_weights, wide_weight_bytes(p, k));
            most_operands = std::max(most_operands, operand_bytes(tokens, k) + row_scale_bytes(tokens));
        };
        want(JITNN_HIP_W_ATTN_Q, 3, false, false);
        want(JITNN_HIP_W_ATTN_O, 1, false, true);
        if (m->moe[l]) continue;
        want(JITNN_HIP_W_FFN_GATE, 2, prefill_dual_ok(w[JITNN_HIP_W_FFN_GATE], w[JITNN_HIP_W_FFN_UP]), false);
        want(JITNN_HIP_W_FFN_DOWN, 1, false, true);
    }
    bool waited = false;
    touch_thread_state();
    start_pass(g_ws.operands, g_ws.weights, most_operands, most_weights, &waited);
    if (waited) g_ws.used = false;
}

// Room for a layer's packed keys and values, for the life of the model (a 64th part of its FP32 cache at 32 layers): false where there is
// none, or none may be allocated; the next prompt pass asks again.
bool packed_room(jitnn_hip_llama *m, hipStream_t st) {
    if (m->packed || stream_recording(st)) return m->packed != nullptr;
    if (hipMalloc(&m->packed, ap_bytes(m->hd, m->kv, m->max_ctx)) != hipSuccess) {
        (void)hipGetLastError();
        m->packed = nullptr;
    }
    return m->packed != nullptr;
}
// The kernels that the attention of a prompt pass may take.  Prompts beyond the GEMV range have FP16-operand linears on both sides of it:
// FP16 operands there too.
enum PromptAttention {
    ATTN_FP32 = JITNN_HIP_ATTN_FP32,          // attn_prefill_kernel
    ATTN_DOT2 = JITNN_HIP_ATTN_DOT2,          // attn_prefill_h_kernel
    ATTN_MFMA_64 = JITNN_HIP_ATTN_MFMA_64,    // attn_prefill_mfma_kernel<D, 1>
    ATTN_MFMA_128 = JITNN_HIP_ATTN_MFMA_128,  // attn_prefill_mfma_kernel<D, 2>
    ATTN_PACKED = JITNN_HIP_ATTN_PACKED,      // attn_packed_kernel (with room for the packed keys and values)
};
PromptAttention prompt_attention(int hd, int heads, int kv, int pos0, int tokens, bool room, int cus) {
    const int group = heads / kv;
    if (tokens <= g.gemv_max_rows) return ATTN_FP32;
    if ((hd != 64 && hd != 128) || group > AM_ROWS) return ATTN_DOT2;
    static_assert(AP_ROWS == 2 * AM_ROWS, "one count of blocks for both");
    const int qt = AP_ROWS / group, blocks = (tokens + qt - 1) / qt * kv;
    // (a head's chunks behind one buffer descriptor of less than 2 GiB)
    if (room && attn_packed_pays(hd, blocks, pos0, tokens, cus) && ap_bytes(hd, 1, pos0 + tokens) < (size_t)1 << 31) return ATTN_PACKED;
    return blocks >= attn_two_tiles_from(hd, cus) ? ATTN_MFMA_128 : ATTN_MFMA_64;
}

template <int D>
int launch_attention_rows(const jitnn_hip_llama *m, int layer, int pos0, int tokens, PromptAttention how, const float *q, float *att, hipStream_t st) {
    const int group = m->heads / m->kv;
    const size_t lo = (size_t)layer * m->max_ctx * m->kv * m->hd;
    const float scale = 1.0f / sqrtf((float)D);
    if constexpr (D == 64 || D == 128) {
        if (how == ATTN_PACKED) {
            const int qt = AP_ROWS / group, keys = pos0 + tokens, chunks = (keys + AP_CH - 1) / AP_CH;
            if (int rc = allow_lds((const void *)attn_packed_kernel<D>, ap_lds_bytes(D))) return rc;
            hipLaunchKernelGGL(attn_pack_kernel<D>, dim3(chunks, m->kv), dim3(AP_THREADS), 0, st, m->kc + lo, m->vc + lo, m->packed, m->kv, keys);
            hipLaunchKernelGGL(attn_packed_kernel<D>, dim3(m->kv, (tokens + qt - 1) / qt), dim3(AP_THREADS), ap_lds_bytes(D), st, q, m->packed, att, m->heads, m->kv,
                               pos0, tokens, chunks, scale);
            return JITNN_HIP_OK;
        }
        if (how == ATTN_MFMA_128) {
            const int qt = 2 * AM_ROWS / group;
            constexpr size_t lds = attn_prefill_mfma_lds_bytes<D, 2>();
            if (int rc = allow_lds((const void *)attn_prefill_mfma_kernel<D, 2>, lds)) return rc;
            hipLaunchKernelGGL((attn_prefill_mfma_kernel<D, 2>), dim3(m->kv, (tokens + qt - 1) / qt), dim3(AM_THREADS), lds, st, q, m->kc + lo, m->vc + lo, att,
                               m->heads, m->kv, pos0, tokens, scale);
            return JITNN_HIP_OK;
        }
        if (how == ATTN_MFMA_64) {
            const int qt = AM_ROWS / group;
            constexpr size_t lds = attn_prefill_mfma_lds_bytes<D, 1>();
            if (int rc = allow_lds((const void *)attn_prefill_mfma_kernel<D, 1>, lds)) return rc;
            hipLaunchKernelGGL((attn_prefill_mfma_kernel<D, 1>), dim3((tokens + qt - 1) / qt, m->kv), dim3(AM_THREADS), lds, st, q, m->kc + lo, m->vc + lo, att,
                               m->heads, m->kv, pos0, tokens, scale);
            return JITNN_HIP_OK;
        }
    }
    const int qt = ATT_ROWS / group;
    const dim3 grid((tokens + qt - 1) / qt, m->kv);
    if (how == ATTN_DOT2) {
        constexpr size_t lds = attn_prefill_h_lds_bytes<D>();
        if (int rc = allow_lds((const void *)attn_prefill_h_kernel<D>, lds)) return rc;
        hipLaunchKernelGGL(attn_prefill_h_kernel<D>, grid, dim3(256), lds, st, q, m->kc + lo, m->vc + lo, att, m->heads, m->kv, pos0, tokens, scale);
    } else {
        // few tokens: blocks of half the rows on twice the CUs (40 tokens of 32 heads over 8: 40 blocks, 14.1 us per layer, -> 80, 11.5).
        // With more blocks than that it depends on head size and context: 160 blocks of 32 rows 3 to 25 % slower than 320 of 16, but at
        // 128 values and 352 blocks 16.0 against 21.9 us (64 tokens of 160 heads over 16), 204 against 328 from position 900.
        if (2 * grid.x * grid.y <= (unsigned)g.cus) {
            const int qt1 = 16 / group;
            constexpr size_t lds = attn_prefill_lds_bytes<D, 1>();
            if (int rc = allow_lds((const void *)attn_prefill_kernel<D, 1>, lds)) return rc;
            hipLaunchKernelGGL((attn_prefill_kernel<D, 1>), dim3((tokens + qt1 - 1) / qt1, m->kv), dim3(256), lds, st, q, m->kc + lo, m->vc + lo, att, m->heads,
                               m->kv, pos0, tokens, scale);
            return JITNN_HIP_OK;
        }
        constexpr size_t lds = attn_prefill_lds_bytes<D, ATT_RT>();
        if (int rc = allow_lds((const void *)attn_prefill_kernel<D, ATT_RT>, lds)) return rc;
        hipLaunchKernelGGL((attn_prefill_kernel<D, ATT_RT>), grid, dim3(256), lds, st, q, m->kc + lo, m->vc + lo, att, m->heads, m->kv, pos0, tokens, scale);
    }
    return JITNN_HIP_OK;
}

// The layers of a pass over T rows x [T, d]: attend(layer, q, k, v, att, pending) turns the queries, appends keys and values and writes the
// attention's output.  defer: q, k and v may reach it in K slices (pending.part).  *out: the rows behind the last layer, in a buffer of the model.
template <class Attend>
int run_layers(jitnn_hip_llama *m, const float *x_dev, int T, bool defer, hipStream_t st, const float **out, Attend &&attend) {
    const int d = m->d;
    float *xn = m->pf[0], *q = m->pf[1], *k = m->pf[2], *v = m->pf[3], *att = m->pf[4], *xa = m->pf[5], *xb = m->pf[6], *gate = m->pf[7],
          *up = m->pf[8], *h = m->pf[9];
    const float *x = x_dev;
    PfPending pend;  // the K slices of the linear that wrote x, when their join is still to come
    PfGroupPending gp;  // the K slices of q, k and v between their launch and the rotation
    for (int l = 0; l < m->layers; ++l) {
        const jitnn_hip_weight *const *w = m->w + (size_t)l * 7;
        const float *nw = m->norms + (size_t)l * 2 * d;
        {
            const jitnn_hip_weight *ws[3] = {w[JITNN_HIP_W_ATTN_Q], w[JITNN_HIP_W_ATTN_K], w[JITNN_HIP_W_ATTN_V]};
            float *ys[3] = {q, k, v};
            if (int rc = normed_linears_rows(m, ws, ys, 3, x, T, nw, xn, st, &pend, defer ? &gp : nullptr)) return rc;
        }
        if (int rc = attend(l, q, k, v, att, gp)) return rc;
        // xa = x + Wo att, xb = xa + W2 (silu(W1 n) * (W3 n)), n = RMSNorm(xa)
        if (int rc = residual_linear_rows(w[JITNN_HIP_W_ATTN_O], att, T, x, xn, xa, st, nullptr, nullptr, m->pf[10], &pend)) return rc;
        if (m->moe[l]) {
            norm_rows(m, xa, T, nw + d, xn, st, &pend);
            if (int rc = jitnn_hip_moe_dev(m->moe[l], xn, T, xa, xb, m->moe_ws[1], (long long)m->moe_ws_bytes[1], st)) return rc;
        } else if (T > g.gemv_max_rows && prefill_dual_ok(w[JITNN_HIP_W_FFN_GATE], w[JITNN_HIP_W_FFN_UP])) {
            // gate and up as one product with the SwiGLU in its epilogue: h = silu(W1 n) * (W3 n) directly
            const bool fused = pend.part && pend.out == xa && pend.n == d;
            if (!fused) flush_pending(pend, T, st);
            const int rc = launch_prefill_dual(w[JITNN_HIP_W_FFN_GATE], w[JITNN_HIP_W_FFN_UP], h, xa, T, nw + d, m->eps, st, fused ? &pend : nullptr);
            if (fused) pend = PfPending{};
            if (rc) return rc;
            if (int rc2 = residual_linear_rows(w[JITNN_HIP_W_FFN_DOWN], h, T, xa, xn, xb, st, nullptr, nullptr, m->pf[10], &pend)) return rc2;
        } else {
            const jitnn_hip_weight *ws[2] = {w[JITNN_HIP_W_FFN_GATE], w[JITNN_HIP_W_FFN_UP]};
            float *ys[2] = {gate, up};
            RowsFfn ffn;
            if (T <= g.gemv_max_rows && rows_ffn_pays(ws[0], ws[1], w[JITNN_HIP_W_FFN_DOWN], T, st, &ffn)) {
                norm_rows(m, xa, T, nw + d, xn, st, &pend);
                if (int rc = launch_rows_ffn(ffn, ws[0], ws[1], w[JITNN_HIP_W_FFN_DOWN], xn, T, xa, xb, st, m->pf[10], &pend)) return rc;
            } else {
                if (int rc = normed_linears_rows(m, ws, ys, 2, xa, T, nw + d, xn, st, &pend)) return rc;
                if (int rc = residual_linear_rows(w[JITNN_HIP_W_FFN_DOWN], gate, T, xa, xn, xb, st, up, h, m->pf[10], &pend)) return rc;
            }
        }
        x = xb;
    }
    flush_pending(pend, T, st);  // the last layer's output exists whole
    *out = x;
    return JITNN_HIP_OK;
}

// cos/sin of t * base^(-2i/D) in double, stored FP32: Rope.tables (core/ops/Rope.java:86-102); other frequencies and a magnitude where the model has
// been given some.  Pairs behind the rotated part do not turn.
// The tables stay where they are, and change together or not at all: they come to the device aside, and go to their places when both are there.
int rope_tables(jitnn_hip_llama *m, const jitnn_hip_rope *r) {
    const int half = m->hd / 2;
    const size_t n = (size_t)m->max_ctx * half;
    float *host = new (std::nothrow) float[2 * n], *aside = nullptr;
    if (!host) return fail(JITNN_HIP_ENOMEM, "out of host memory");
    for (int t = 0; t < m->max_ctx; ++t)
        for (int i = 0; i < half; ++i) {
            const bool turns = i < r->rot / 2;
            const double angle = turns ? t * r->frequency[i] : 0.0, magnitude = turns ? r->magnitude : 1.0;
            host[(size_t)t * half + i] = (float)(magnitude * cos(angle));
            host[n + (size_t)t * half + i] = (float)(magnitude * sin(angle));
        }
    if (hipMalloc(&aside, 2 * n * sizeof(float)) != hipSuccess) {
        (void)hipGetLastError();
        delete[] host;
        return fail(JITNN_HIP_ENOMEM, "no %zu bytes of device memory for the rotary tables", 2 * n * sizeof(float));
    }
    hipError_t e = hipMemcpy(aside, host, 2 * n * sizeof(float), hipMemcpyHostToDevice);
    delete[] host;
    if (e == hipSuccess) e = hipMemcpy(m->cosv, aside, n * sizeof(float), hipMemcpyDeviceToDevice);
    if (e == hipSuccess) e = hipMemcpy(m->sinv, aside + n, n * sizeof(float), hipMemcpyDeviceToDevice);
    if (e == hipSuccess) e = hipDeviceSynchronize();
    (void)hipFree(aside);
    return e == hipSuccess ? JITNN_HIP_OK : fail(JITNN_HIP_EDEVICE, "copying the rotary tables: %s", hipGetErrorString(e));
}

}  // namespace

extern "C" {

int jitnn_hip_llama_create(int layers, int d_model, int heads, int kv_heads, int head_dim, int ffn, int vocab, int max_ctx, float rms_eps,
                           float rope_theta, jitnn_hip_llama **out) {
    if (!out) return fail(JITNN_HIP_EINVAL, "out is NULL");
    *out = nullptr;
    if (layers < 1 || d_model < 1 || heads < 1 || kv_heads < 1 || ffn < 1 || vocab < 1 || max_ctx < 1)
        return fail(JITNN_HIP_EINVAL, "non-positive model dimension");
    if (heads % kv_heads != 0) return fail(JITNN_HIP_EINVAL, "grouped-query attention: %d query heads over %d key/value heads", heads, kv_heads);
    if (heads > 65535) return fail(JITNN_HIP_EINVAL, "%d query heads (the attention kernel's packed head counts hold 16 bits each)", heads);
    if (heads / kv_heads > ATT_GMAX) return fail(JITNN_HIP_EINVAL, "%d query heads per key/value head (at most %d are built)", heads / kv_heads, ATT_GMAX);
    if (head_dim != 64 && head_dim != 128 && head_dim != 192 && head_dim != 256)
        return fail(JITNN_HIP_EINVAL, "head_dim %d (64, 128, 192 and 256 are built)", head_dim);
    if (int rc = check_ready()) return rc;
    jitnn_hip_llama *m = new (std::nothrow) jitnn_hip_llama();
    if (!m) return fail(JITNN_HIP_ENOMEM, "out of host memory");
    *m = jitnn_hip_llama{};
    m->layers = layers; m->d = d_model; m->heads = heads; m->kv = kv_heads; m->hd = head_dim; m->ffn = ffn; m->vocab = vocab;
    m->max_ctx = max_ctx; m->eps = rms_eps; m->theta = rope_theta;
    m->attention = -1;
    m->w = new (std::nothrow) const jitnn_hip_weight *[(size_t)layers * 7]();
    m->moe = new (std::nothrow) const jitnn_hip_moe *[(size_t)layers]();
    m->chunks_max = (max_ctx + 15) / 16;  // the smallest key chunk any head size uses
    const size_t cache = (size_t)layers * max_ctx * kv_heads * head_dim;
    const int qd = heads * head_dim, kd = kv_heads * head_dim, half = head_dim / 2;
    struct { float **p; size_t n; } bufs[] = {
        {&m->norms, ((size_t)layers * 2 + 1) * d_model}, {&m->kc, cache}, {&m->vc, cache}, {&m->cosv, (size_t)max_ctx * half},
        {&m->sinv, (size_t)max_ctx * half}, {&m->xin, (size_t)d_model}, {&m->xa, (size_t)d_model}, {&m->xb, (size_t)d_model}, {&m->xn, (size_t)d_model},
        {&m->q, (size_t)qd + 2 * (size_t)kd}, {&m->att, (size_t)qd}, {&m->gate, (size_t)ffn}, {&m->up, (size_t)ffn},
        {&m->h, (size_t)ffn}, {&m->part, (size_t)heads * m->chunks_max * (head_dim + 2)}, {&m->logits, (size_t)vocab}};
    bool ok = m->w != nullptr && m->moe != nullptr;
    for (auto &b : bufs) {
        if (!ok) break;
        ok = hipMalloc(b.p, b.n * sizeof(float)) == hipSuccess;
    }
    if (ok) {  // the projections of a decode step: q [heads, D], k [kv_heads, D], v [kv_heads, D] in one buffer (one pointer for the attention kernel)
        m->k = m->q + qd;
        m->v = m->k + kd;
    }
    ok = ok && rope_build(head_dim, false, (double)rope_theta, nullptr, nullptr, &m->rope) == JITNN_HIP_OK && rope_tables(m, m->rope) == JITNN_HIP_OK;
    if (!ok) {
        jitnn_hip_llama_free(m);
        return fail(JITNN_HIP_ENOMEM, "allocating the model buffers (%zu bytes of KV cache) failed", 2 * cache * sizeof(float));
    }
    *out = m;
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_free(jitnn_hip_llama *m) {
    if (!m) return JITNN_HIP_OK;
    float *bufs[] = {m->norms, m->kc, m->vc, m->cosv, m->sinv, m->xin, m->xa, m->xb, m->xn, m->q, m->att, m->gate, m->up, m->h, m->part, m->logits};
    for (float *b : bufs)
        if (b) (void)hipFree(b);
    for (float *b : m->pf)
        if (b) (void)hipFree(b);
    if (m->packed) (void)hipFree(m->packed);
    if (m->paged_ws) (void)hipFree(m->paged_ws);
    for (void *b : m->moe_ws)
        if (b) (void)hipFree(b);
    while (m->kept) {
        jitnn_hip_llama::Kept *k = m->kept;
        m->kept = k->next;
        (void)hipFree(k->p);
        delete k;
    }
    rope_drop(m->rope);
    if (m->embd) (void)hipFree(m->embd);
    if (m->tok_dev) (void)hipFree(m->tok_dev);
    if (m->tok_pin) (void)hipHostFree(m->tok_pin);
    delete[] m->w;
    delete[] m->moe;
    delete m;
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_set_weight(jitnn_hip_llama *m, int layer, int which, const jitnn_hip_weight *w) {
    if (!m || !w) return fail(JITNN_HIP_EINVAL, "model or weight is NULL");
    if (which < 0 || which > JITNN_HIP_W_OUTPUT) return fail(JITNN_HIP_EINVAL, "weight slot %d", which);
    const int qd = m->heads * m->hd, kd = m->kv * m->hd;
    const int en[] = {qd, kd, kd, m->d, m->ffn, m->ffn, m->d, m->vocab};
    const int ek[] = {m->d, m->d, m->d, qd, m->d, m->d, m->ffn, m->d};
    if (w->n != en[which] || w->k != ek[which])
        return fail(JITNN_HIP_EINVAL, "weight slot %d needs shape [%d, %d], got [%d, %d]", which, en[which], ek[which], w->n, w->k);
    if (which == JITNN_HIP_W_OUTPUT) {
        m->w_out = w;
        return JITNN_HIP_OK;
    }
    if (layer < 0 || layer >= m->layers) return fail(JITNN_HIP_EINVAL, "layer %d of %d", layer, m->layers);
    m->w[layer * 7 + which] = w;
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_set_moe(jitnn_hip_llama *m, int layer, const jitnn_hip_moe *e) {
    if (!m) return fail(JITNN_HIP_EINVAL, "model is NULL");
    if (layer < 0 || layer >= m->layers) return fail(JITNN_HIP_EINVAL, "layer %d of %d", layer, m->layers);
    if (e && e->router->d != m->d) return fail(JITNN_HIP_EINVAL, "experts on %d values for a model of %d", e->router->d, m->d);
    const jitnn_hip_moe *was = m->moe[layer];
    m->moe[layer] = e;
    m->moe_cap = 0;  // (the next pass of many tokens looks whether its workspace does)
    if (!e) return JITNN_HIP_OK;
    if (int rc = moe_reserve(m, 0, 1)) {
        m->moe[layer] = was;
        return rc;
    }
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_set_norm(jitnn_hip_llama *m, int layer, int which, const float *w_host) {
    if (!m || !w_host) return fail(JITNN_HIP_EINVAL, "model or weights are NULL");
    size_t off;
    if (which == JITNN_HIP_NORM_OUTPUT) {
        off = (size_t)m->layers * 2 * m->d;
    } else if (which == JITNN_HIP_NORM_ATTN || which == JITNN_HIP_NORM_FFN) {
        if (layer < 0 || layer >= m->layers) return fail(JITNN_HIP_EINVAL, "layer %d of %d", layer, m->layers);
        off = ((size_t)layer * 2 + which) * m->d;
    } else {
        return fail(JITNN_HIP_EINVAL, "norm slot %d", which);
    }
    HIP_TRY(hipMemcpy(m->norms + off, w_host, (size_t)m->d * 4, hipMemcpyHostToDevice));
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_kv_write(jitnn_hip_llama *m, int layer, int pos0, int count, const float *k_host, const float *v_host) {
    if (!m || !k_host || !v_host) return fail(JITNN_HIP_EINVAL, "NULL argument");
    if (layer < 0 || layer >= m->layers || pos0 < 0 || count < 0 || pos0 + count > m->max_ctx)
        return fail(JITNN_HIP_EINVAL, "layer %d positions [%d, %d) of a cache of %d", layer, pos0, pos0 + count, m->max_ctx);
    const size_t row = (size_t)m->kv * m->hd, off = ((size_t)layer * m->max_ctx + pos0) * row;
    HIP_TRY(hipMemcpy(m->kc + off, k_host, count * row * 4, hipMemcpyHostToDevice));
    HIP_TRY(hipMemcpy(m->vc + off, v_host, count * row * 4, hipMemcpyHostToDevice));
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_kv_read(const jitnn_hip_llama *m, int layer, int pos0, int count, float *k_host, float *v_host) {
    if (!m || !k_host || !v_host) return fail(JITNN_HIP_EINVAL, "NULL argument");
    if (layer < 0 || layer >= m->layers || pos0 < 0 || count < 0 || pos0 + count > m->max_ctx)
        return fail(JITNN_HIP_EINVAL, "layer %d positions [%d, %d) of a cache of %d", layer, pos0, pos0 + count, m->max_ctx);
    const size_t row = (size_t)m->kv * m->hd, off = ((size_t)layer * m->max_ctx + pos0) * row;
    HIP_TRY(hipMemcpy(k_host, m->kc + off, count * row * 4, hipMemcpyDeviceToHost));
    HIP_TRY(hipMemcpy(v_host, m->vc + off, count * row * 4, hipMemcpyDeviceToHost));
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_decode_dev(jitnn_hip_llama *m, const float *x_dev, int pos, float *logits_dev, void *stream) {
    if (int rc = check_model(m)) return rc;
    if (!x_dev || !logits_dev) return fail(JITNN_HIP_EINVAL, "input or output is NULL");
    if (pos < 0 || pos >= m->max_ctx) return fail(JITNN_HIP_EINVAL, "position %d of a cache of %d", pos, m->max_ctx);
    hipStream_t st = (hipStream_t)stream;
    const int d = m->d;
    count_op(ST_DECODE, model_weight_bytes(m, 1) + 4ll * m->layers * 2 * (pos + 1) * m->kv * m->hd + 4ll * (d + m->vocab));
    StatNest nest;
    // residual stream: layer input x (the caller's buffer for layer 0, xb afterwards) -> xa after attention -> xb after the FFN
    const float *x = x_dev;
    for (int l = 0; l < m->layers; ++l) {
        const jitnn_hip_weight *const *w = m->w + (size_t)l * 7;
        const float *nw = m->norms + (size_t)l * 2 * d;
        // q, k, v = W (RMSNorm x): the norm is fused into the linears; projections of one format share a launch
        {
            const jitnn_hip_weight *ws[3] = {w[JITNN_HIP_W_ATTN_Q], w[JITNN_HIP_W_ATTN_K], w[JITNN_HIP_W_ATTN_V]};
            float *ys[3] = {m->q, m->k, m->v};
            if (int rc = normed_linears(m, ws, ys, 3, x, nw, st)) return rc;
        }
        switch (m->hd) {  // RoPE, cache append and attention per key chunk, then the merge of the chunks
        case 64: launch_attention<64>(m, l, pos, st); break;
        case 128: launch_attention<128>(m, l, pos, st); break;
        case 192: launch_attention<192>(m, l, pos, st); break;
        default: launch_attention<256>(m, l, pos, st); break;
        }
        // xa = x + Wo att, xb = xa + W2 h: the residual rides in the linear's bias slot
        if (int rc = launch_gemv(w[JITNN_HIP_W_ATTN_O], m->att, 1, x, m->xa, st)) return rc;
        if (m->moe[l]) {
            norm_rows(m, m->xa, 1, nw + d, m->xn, st, nullptr);
            if (int rc = jitnn_hip_moe_dev(m->moe[l], m->xn, 1, m->xa, m->xb, m->moe_ws[0], (long long)m->moe_ws_bytes[0], st)) return rc;
            x = m->xb;
            continue;
        }
        // h = silu(W1 n) * (W3 n), n = RMSNorm(xa): one launch when gate and up share a format
        const jitnn_hip_weight *wg = w[JITNN_HIP_W_FFN_GATE], *wu = w[JITNN_HIP_W_FFN_UP];
        if (xreg_ok(wg) && wg->fmt == wu->fmt) {
            XregCall c;
            c.w[0] = wg;
            c.w2 = wu;
            c.y[0] = m->h;
            c.x = m->xa;
            c.norm_w = nw + d;
            c.eps = m->eps;
            if (int rc = launch_xreg(c, st)) return rc;
        } else {
            const jitnn_hip_weight *ws[2] = {wg, wu};
            float *ys[2] = {m->gate, m->up};
            if (int rc = normed_linears(m, ws, ys, 2, m->xa, nw + d, st)) return rc;
            hipLaunchKernelGGL(swiglu_kernel, dim3((m->ffn + 1023) / 1024), dim3(256), 0, st, m->gate, m->up, m->h, m->ffn);
        }
        if (int rc = launch_gemv(w[JITNN_HIP_W_FFN_DOWN], m->h, 1, m->xa, m->xb, st)) return rc;
        x = m->xb;
    }
    {
        const jitnn_hip_weight *ws[1] = {m->w_out};
        float *ys[1] = {logits_dev};
        if (int rc = normed_linears(m, ws, ys, 1, x, m->norms + (size_t)m->layers * 2 * d, st)) return rc;
    }
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_prefill_dev(jitnn_hip_llama *m, const float *x_dev, int pos0, int tokens, float *logits_dev, void *stream) {
    if (int rc = check_model(m)) return rc;
    if (!x_dev) return fail(JITNN_HIP_EINVAL, "input is NULL");
    if (tokens < 1 || pos0 < 0 || pos0 > m->max_ctx - tokens)
        return fail(JITNN_HIP_EINVAL, "%d tokens from position %d in a cache of %d", tokens, pos0, m->max_ctx);
    if (m->d % 4 != 0) return fail(JITNN_HIP_EUNSUPPORTED, "d_model %d is not a multiple of 4", m->d);
    if (int rc = ensure_prefill(m, tokens)) return rc;
    hipStream_t st = (hipStream_t)stream;
    count_op(ST_PREFILL, model_weight_bytes(m, tokens) + 4ll * m->layers * 2 * (pos0 + tokens) * m->kv * m->hd + 4ll * ((long long)tokens * m->d + (logits_dev ? m->vocab : 0)));
    StatNest nest;
    const int d = m->d, T = tokens;
    prefill_reserve(m, T, st);
    PromptAttention how = prompt_attention(m->hd, m->heads, m->kv, pos0, T, !m->no_packing, g.cus);
    if (how == ATTN_PACKED && !packed_room(m, st)) how = prompt_attention(m->hd, m->heads, m->kv, pos0, T, false, g.cus);
    m->attention = how;
    const float *x = nullptr;
    const int rc = run_layers(m, x_dev, T, true, st, &x, [&](int l, float *q, const float *k, const float *v, float *att, PfGroupPending &gp) {
        const size_t lo = (size_t)l * m->max_ctx * m->kv * m->hd;
        if (gp.part) {  // q, k and v still lie in K slices: the rotation adds them up as it reads them
            hipLaunchKernelGGL(rope_append_rows_join_kernel, dim3(T, T < 256 ? 4 : 1), dim3(256), 0, st, gp.part, gp.sg.splits[0], gp.sg.splits[1], gp.sg.splits[2], T, q,
                               m->kc + lo, m->vc + lo, m->cosv, m->sinv, m->heads, m->kv, m->hd, pos0, m->rope_interleaved);
            gp.part = nullptr;
        } else {
            hipLaunchKernelGGL(rope_append_rows_kernel, dim3(T, T < 256 ? 4 : 1), dim3(256), 0, st, q, k, v, m->kc + lo, m->vc + lo, m->cosv, m->sinv, m->heads, m->kv,
                               m->hd, pos0, m->rope_interleaved);
        }
        switch (m->hd) {
        case 64: return launch_attention_rows<64>(m, l, pos0, T, how, q, att, st);
        case 128: return launch_attention_rows<128>(m, l, pos0, T, how, q, att, st);
        case 192: return launch_attention_rows<192>(m, l, pos0, T, how, q, att, st);
        default: return launch_attention_rows<256>(m, l, pos0, T, how, q, att, st);
        }
    });
    if (rc) return rc;
    if (logits_dev) {  // the last token's logits
        const jitnn_hip_weight *ws[1] = {m->w_out};
        float *ys[1] = {logits_dev};
        if (int rc2 = normed_linears(m, ws, ys, 1, x + (size_t)(T - 1) * d, m->norms + (size_t)m->layers * 2 * d, st)) return rc2;
    }
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_set_rope(jitnn_hip_llama *m, const jitnn_hip_rope *r) {
    if (!m || !r) return fail(JITNN_HIP_EINVAL, "model or rope is NULL");
    if (r->rot > m->hd || (r->rot < m->hd && !r->interleaved))
        return fail(JITNN_HIP_EINVAL, "rot_dim %d of heads of %d values (a part of a head: interleaved pairs only)", r->rot, m->hd);
    if (int rc = check_ready()) return rc;
    jitnn_hip_rope *copy = nullptr;
    const size_t bytes = (size_t)r->rot / 2 * sizeof(unsigned long long);
    try {
        copy = new jitnn_hip_rope(*r);
    } catch (const std::bad_alloc &) {
        return fail(JITNN_HIP_ENOMEM, "out of host memory");
    }
    copy->turns = nullptr;
    if (hipMalloc(&copy->turns, bytes) != hipSuccess) {
        (void)hipGetLastError();
        copy->turns = nullptr;
        rope_drop(copy);
        return fail(JITNN_HIP_ENOMEM, "no %zu bytes of device memory for the rotary frequencies", bytes);
    }
    const hipError_t e = hipMemcpy(copy->turns, r->turns, bytes, hipMemcpyDeviceToDevice);
    if (const int rc = e == hipSuccess ? rope_tables(m, copy) : fail(JITNN_HIP_EDEVICE, "copying the rotary frequencies: %s", hipGetErrorString(e))) {
        rope_drop(copy);
        return rc;
    }
    rope_drop(m->rope);
    m->rope = copy;
    m->rope_interleaved = copy->interleaved;
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_step_dev(jitnn_hip_llama *m, const jitnn_hip_paged_cache *c, const jitnn_hip_batch *b, const float *x_dev, const int *logit_rows_dev, int logit_count,
                             float *logits_dev, void *stream) {
    if (int rc = check_model(m)) return rc;
    if (int rc = check_cache(c, 0)) return rc;
    if (int rc = check_batch(c, b)) return rc;
    if (c->layers != m->layers || c->kv != m->kv || c->hd != m->hd)
        return fail(JITNN_HIP_EINVAL, "a cache of %d layers of %d heads of %d values for a model of %d layers of %d of %d", c->layers, c->kv, c->hd, m->layers, m->kv, m->hd);
    if (logit_count < 0 || logit_count > b->tokens || (logit_count > 0 && (!logit_rows_dev || !logits_dev)))
        return fail(JITNN_HIP_EINVAL, "logits of %d rows of %d", logit_count, b->tokens);
    if (m->d % 4 != 0) return fail(JITNN_HIP_EUNSUPPORTED, "d_model %d is not a multiple of 4", m->d);
    if (m->rope->rot % 8 != 0) return fail(JITNN_HIP_EUNSUPPORTED, "rot_dim %d is not a multiple of 8", m->rope->rot);
    if (b->tokens == 0 || (b->sequences == 0 && logit_count == 0)) return JITNN_HIP_OK;
    if (!x_dev) return fail(JITNN_HIP_EINVAL, "input is NULL");
    hipStream_t st = (hipStream_t)stream;
    const int d = m->d, T = b->tokens;
    const long long need = jitnn_hip_paged_attention_workspace(c, b, m->heads);
    if (need < 0) return (int)need;
    const bool recording = stream_recording(st);
    if (recording && (T > m->pf_cap || (T > m->moe_cap && moe_need(m, 1, T) > m->moe_ws_bytes[1]) || (size_t)need > m->paged_ws_bytes))
        return fail(JITNN_HIP_EINVAL, "a pass of %d tokens needs larger buffers than the model has, which a recording cannot allocate", T);
    if (recording) m->recorded = true;
    if (int rc = ensure_prefill(m, T)) return rc;
    if ((size_t)need > m->paged_ws_bytes) {
        HIP_TRY(hipDeviceSynchronize());  // earlier passes may still use the old one
        release_or_keep(m, m->paged_ws);
        m->paged_ws = nullptr;
        m->paged_ws_bytes = 0;
        if (hipMalloc(&m->paged_ws, (size_t)need) != hipSuccess) {
            (void)hipGetLastError();
            m->paged_ws = nullptr;
            return fail(JITNN_HIP_ENOMEM, "no %lld bytes of device memory for the attention's workspace", need);
        }
        m->paged_ws_bytes = (size_t)need;
    }
    count_op(ST_PREFILL, model_weight_bytes(m, T) + 4ll * ((long long)T * d + (long long)logit_count * m->vocab));
    StatNest nest;
    prefill_reserve(m, T, st);
    const long long qd = (long long)m->heads * m->hd, kd = (long long)m->kv * m->hd;
    const float scale = 1.0f / sqrtf((float)m->hd);
    const float *x = x_dev;  // (of no sequence at all, only the logits are to be said to be none)
    const int rc = b->sequences == 0 ? JITNN_HIP_OK : run_layers(m, x_dev, T, false, st, &x, [&](int l, float *q, const float *k, const float *v, float *att, PfGroupPending &) {
        if (int arc = append_rows(c, l, b, m->rope, m->rope_interleaved != 0, q, qd, m->heads, q, qd, k, kd, v, kd, st)) return arc;
        return jitnn_hip_paged_attention_dev(c, l, b, m->heads, q, qd, scale, att, qd, m->paged_ws, (long long)m->paged_ws_bytes, stream);
    });
    if (rc) return rc;
    if (logit_count > 0) {
        float *rows = m->pf[5], *xn = m->pf[0];  // (free behind the last layer)
        hipLaunchKernelGGL(batch_rows_kernel, dim3((unsigned)logit_count), dim3(256), 0, st, x, logit_rows_dev, b->starts, b->sequences, T, rows, d);
        const jitnn_hip_weight *ws[1] = {m->w_out};
        float *ys[1] = {logits_dev};
        const float *nw = m->norms + (size_t)m->layers * 2 * d;
        if (int rc2 = logit_count == 1 ? normed_linears(m, ws, ys, 1, rows, nw, st) : normed_linears_rows(m, ws, ys, 1, rows, logit_count, nw, xn, st)) return rc2;
    }
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

// ---- generation loop: embedding lookup, greedy choice, prompt + token-by-token decode --------------------------------

int jitnn_hip_prompt_attention(int heads, int kv_heads, int head_dim, int pos0, int tokens, int packing, int compute_units) {
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads / kv_heads > ATT_GMAX || (head_dim != 64 && head_dim != 128 && head_dim != 192 && head_dim != 256) ||
        pos0 < 0 || tokens < 1 || pos0 > INT_MAX - tokens || compute_units < 0)
        return fail(JITNN_HIP_EINVAL, "no such prompt");
    if (compute_units == 0) {
        if (int rc = check_ready()) return rc;
        compute_units = g.cus;
    }
    return prompt_attention(head_dim, heads, kv_heads, pos0, tokens, packing != 0, compute_units);
}

int jitnn_hip_llama_set_packing(jitnn_hip_llama *m, int allow) {
    if (!m) return fail(JITNN_HIP_EINVAL, "model is NULL");
    m->no_packing = !allow;
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_last_attention(const jitnn_hip_llama *m) {
    if (!m) return fail(JITNN_HIP_EINVAL, "model is NULL");
    return m->attention < 0 ? fail(JITNN_HIP_EINVAL, "no prompt pass yet") : m->attention;
}

int jitnn_hip_llama_set_rope_interleaved(jitnn_hip_llama *m, int interleaved) {
    if (!m) return fail(JITNN_HIP_EINVAL, "model is NULL");
    if (!interleaved && m->rope->rot < m->hd) return fail(JITNN_HIP_EINVAL, "%d of %d values of a head turn: interleaved pairs only", m->rope->rot, m->hd);
    m->rope_interleaved = interleaved != 0;
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_set_embedding(jitnn_hip_llama *m, int ggml_type, const void *table_host, long long nbytes) {
    if (!m || !table_host) return fail(JITNN_HIP_EINVAL, "model or table is NULL");
    long long need;
    if (ggml_type == 0 || ggml_type == 1) {
        need = (long long)m->vocab * m->d * (ggml_type == 0 ? 4 : 2);
    } else {
        need = jitnn_hip_weight_nbytes(ggml_type, m->vocab, m->d);
        if (need < 0) return (int)need;
    }
    if (nbytes != need) return fail(JITNN_HIP_EINVAL, "an embedding table [%d, %d] of ggml type %d holds %lld bytes, got %lld", m->vocab, m->d, ggml_type, need, nbytes);
    if (m->d % 4 != 0) return fail(JITNN_HIP_EUNSUPPORTED, "d_model %d is not a multiple of 4", m->d);
    if (int rc = check_ready()) return rc;
    if (m->embd) HIP_TRY(hipFree(m->embd));
    m->embd = nullptr;
    hipError_t e = hipMalloc(&m->embd, (size_t)nbytes);
    if (e != hipSuccess) return fail(JITNN_HIP_ENOMEM, "hipMalloc of %lld bytes: %s", nbytes, hipGetErrorString(e));
    HIP_TRY(hipMemcpy(m->embd, table_host, (size_t)nbytes, hipMemcpyHostToDevice));
    m->embd_fmt = ggml_type;
    if (!m->tok_dev) HIP_TRY(hipMalloc(&m->tok_dev, (size_t)m->max_ctx * sizeof(int)));
    if (!m->tok_pin) HIP_TRY(hipHostMalloc((void **)&m->tok_pin, sizeof(int), hipHostMallocDefault));
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_embed_dev(jitnn_hip_llama *m, const int *tokens_dev, int count, float *x_dev, void *stream) {
    if (!m || !tokens_dev || !x_dev) return fail(JITNN_HIP_EINVAL, "NULL argument");
    if (!m->embd) return fail(JITNN_HIP_EINVAL, "the model has no embedding table");
    if (count < 1) return fail(JITNN_HIP_EINVAL, "%d tokens", count);
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)count), block(256);
    switch (m->embd_fmt) {
    case 0:
    case 1: hipLaunchKernelGGL(embed_plain_rows_kernel, grid, block, 0, st, (const void *)m->embd, m->embd_fmt, tokens_dev, x_dev, m->d, m->vocab); break;
    case F_Q4_0: hipLaunchKernelGGL(dequant_rows_kernel<F_Q4_0>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    case F_Q4_1: hipLaunchKernelGGL(dequant_rows_kernel<F_Q4_1>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    case F_Q5_0: hipLaunchKernelGGL(dequant_rows_kernel<F_Q5_0>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    case F_Q5_1: hipLaunchKernelGGL(dequant_rows_kernel<F_Q5_1>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    case F_Q8_0: hipLaunchKernelGGL(dequant_rows_kernel<F_Q8_0>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    case F_Q2_K: hipLaunchKernelGGL(dequant_rows_kernel<F_Q2_K>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    case F_Q3_K: hipLaunchKernelGGL(dequant_rows_kernel<F_Q3_K>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    case F_Q4_K: hipLaunchKernelGGL(dequant_rows_kernel<F_Q4_K>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    case F_Q5_K: hipLaunchKernelGGL(dequant_rows_kernel<F_Q5_K>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    default: hipLaunchKernelGGL(dequant_rows_kernel<F_Q6_K>, grid, block, 0, st, m->embd, tokens_dev, x_dev, m->d, m->vocab); break;
    }
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_argmax_dev(jitnn_hip_llama *m, const float *logits_dev, int *token_dev, void *stream) {
    if (!m || !logits_dev || !token_dev) return fail(JITNN_HIP_EINVAL, "NULL argument");
    hipLaunchKernelGGL(argmax_kernel, dim3(1), dim3(ARG_THREADS), 0, (hipStream_t)stream, logits_dev, m->vocab, token_dev);
    HIP_TRY(hipGetLastError());
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_generate(jitnn_hip_llama *m, const int *prompt, int prompt_tokens, int pos0, int max_new_tokens, int eos_token, int *out_tokens,
                             void (*on_token)(int token, void *user), void *user) {
    if (int rc = check_model(m)) return rc;
    if (!prompt || (!out_tokens && max_new_tokens > 0)) return fail(JITNN_HIP_EINVAL, "prompt or output is NULL");
    if (!m->embd) return fail(JITNN_HIP_EINVAL, "the model has no embedding table");
    if (prompt_tokens < 1 || max_new_tokens < 0 || pos0 < 0) return fail(JITNN_HIP_EINVAL, "%d prompt tokens from position %d, %d new tokens", prompt_tokens, pos0, max_new_tokens);
    if ((long long)pos0 + prompt_tokens + max_new_tokens > (long long)m->max_ctx + 1)
        return fail(JITNN_HIP_EINVAL, "positions %d .. %d do not fit a cache of %d", pos0, pos0 + prompt_tokens + max_new_tokens - 2, m->max_ctx);
    for (int i = 0; i < prompt_tokens; ++i)
        if (prompt[i] < 0 || prompt[i] >= m->vocab) return fail(JITNN_HIP_EINVAL, "token %d of a vocabulary of %d", prompt[i], m->vocab);
    if (max_new_tokens == 0) return 0;
    if (int rc = stage_reserve(0, (size_t)prompt_tokens * m->d * 4)) return rc;
    HostStage &hs = g_thread.stage;
    hipStream_t st = hs.stream;
    // the prompt: embeddings of all tokens, one pass through the layers, logits of the last token
    HIP_TRY(hipMemcpyAsync(m->tok_dev, prompt, (size_t)prompt_tokens * sizeof(int), hipMemcpyHostToDevice, st));
    float *x = (float *)hs.dev;
    if (int rc = jitnn_hip_llama_embed_dev(m, m->tok_dev, prompt_tokens, x, st)) return rc;
    if (prompt_tokens == 1) {
        if (int rc = jitnn_hip_llama_decode_dev(m, x, pos0, m->logits, st)) return rc;
    } else {
        if (int rc = jitnn_hip_llama_prefill_dev(m, x, pos0, prompt_tokens, m->logits, st)) return rc;
    }
    int produced = 0;
    for (int pos = pos0 + prompt_tokens;; ++pos) {
        // greedy: the largest logit (Llm.generate runs at temperature 0, jitnn-llm/.../llm/Llm.java:74-76)
        if (int rc = jitnn_hip_llama_argmax_dev(m, m->logits, m->tok_dev, st)) return rc;
        HIP_TRY(hipMemcpyAsync(m->tok_pin, m->tok_dev, sizeof(int), hipMemcpyDeviceToHost, st));
        HIP_TRY(hipStreamSynchronize(st));
        const int tok = *m->tok_pin;
        if (tok == eos_token) break;
        out_tokens[produced++] = tok;
        if (on_token) on_token(tok, user);
        if (produced == max_new_tokens) break;
        if (int rc = jitnn_hip_llama_embed_dev(m, m->tok_dev, 1, m->xin, st)) return rc;
        if (int rc = jitnn_hip_llama_decode_dev(m, m->xin, pos, m->logits, st)) return rc;
    }
    HIP_TRY(hipStreamSynchronize(st));
    return produced;
}

int jitnn_hip_llama_prefill(jitnn_hip_llama *m, const float *x_host, int pos0, int tokens, float *logits_host) {
    if (int rc = check_model(m)) return rc;
    if (!x_host) return fail(JITNN_HIP_EINVAL, "input is NULL");
    if (tokens < 1) return fail(JITNN_HIP_EINVAL, "%d tokens", tokens);
    const size_t bytes = (size_t)tokens * m->d * 4;
    if (int rc = stage_reserve(0, bytes)) return rc;  // the embeddings go through the calling thread's device buffer
    HostStage &st = g_thread.stage;
    HIP_TRY(hipMemcpyAsync(st.dev, x_host, bytes, hipMemcpyHostToDevice, st.stream));
    if (int rc = jitnn_hip_llama_prefill_dev(m, (const float *)st.dev, pos0, tokens, logits_host ? m->logits : nullptr, st.stream)) return rc;
    if (logits_host) HIP_TRY(hipMemcpyAsync(logits_host, m->logits, (size_t)m->vocab * 4, hipMemcpyDeviceToHost, st.stream));
    hipError_t e = hipStreamSynchronize(st.stream);
    if (e != hipSuccess) return fail(JITNN_HIP_EDEVICE, "the prefill step failed: %s", hipGetErrorString(e));
    return JITNN_HIP_OK;
}

int jitnn_hip_llama_decode(jitnn_hip_llama *m, const float *x_host, int pos, float *logits_host) {
    if (int rc = check_model(m)) return rc;
    if (!x_host || !logits_host) return fail(JITNN_HIP_EINVAL, "input or output is NULL");
    HIP_TRY(hipMemcpy(m->xin, x_host, (size_t)m->d * 4, hipMemcpyHostToDevice));
    if (int rc = jitnn_hip_llama_decode_dev(m, m->xin, pos, m->logits, nullptr)) return rc;
    HIP_TRY(hipMemcpy(logits_host, m->logits, (size_t)m->vocab * 4, hipMemcpyDeviceToHost));
    return JITNN_HIP_OK;
}

}  // extern "C"
