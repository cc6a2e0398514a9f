// Token operators: host side of ptq8_quantize_rows, ptq8_linear and ptq8_linear_grouped
// (argument checks, kernel choice, launches) and their extern "C" boundary.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <iterator>
#include <mutex>
#include <new>

#include "ptq8.h"
#include "ptq8_linear.cuh"
#include "ptq8_linear_few.cuh"
#include "ptq8_linear_tc.cuh"
#include "ptq8_rows.cuh"

using namespace ptq8;

// what the Python mirror packs
static_assert(sizeof(ptq8_rows_args) == 72 && sizeof(ptq8_linear_args) == 120, "argument structs");

struct ptq8_ops {
    int device = 0;
    int sms = 0;
    int* error = nullptr;       // pinned host word that a kernel whose bounded wait ran out sets (error_word())
    int* error_dev = nullptr;   // its device address
    long long wait_limit = kWaitLimitCycles;
    int stall = 0;
    int variant = -1, split = 1;   // test hook: the tile variant of every product
    PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    char err[512] = "";         // message of the last refusal: a fixed buffer, since refusing must not throw
};

namespace {

int fail(ptq8_ops* o, int status, const char* f, ...) {
    va_list ap;
    va_start(ap, f);
    std::vsnprintf(o->err, sizeof o->err, f, ap);
    va_end(ap);
    return status;
}

// A message for a caller who has no handle yet.
void say(char* err, size_t n, const char* f, const char* more = "") {
    if (err && n) std::snprintf(err, n, f, more);
}

// The device becomes current for the call and is given back: a process may drive several.
struct OnDevice {
    int before = -1;
    cudaError_t rc;
    explicit OnDevice(int device) {
        rc = cudaGetDevice(&before);
        if (rc == cudaSuccess && before != device) rc = cudaSetDevice(device);
        if (before == device) before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// One launch with programmatic stream serialization: the kernel may be scheduled while the kernel
// before it on the stream drains, and waits (griddepcontrol.wait) before it touches global memory.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t stream, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// A handle's error word, zero.  Words come from pinned blocks that stay with the process and no word is used again: a
// kernel of a destroyed handle that is still running, or a graph that holds one, may write its word at any time after.
cudaError_t error_word(int** host, int** dev) {
    constexpr int kWords = 1024;
    static std::mutex lock;
    static int* block = nullptr;
    static int used = kWords;
    std::lock_guard<std::mutex> hold(lock);
    if (used == kWords) {
        int* fresh = nullptr;
        const cudaError_t e = cudaHostAlloc(&fresh, kWords * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable);
        if (e != cudaSuccess) return e;
        std::memset(fresh, 0, kWords * sizeof(int));
        block = fresh;
        used = 0;
    }
    void* at = nullptr;
    const cudaError_t e = cudaHostGetDevicePointer(&at, block, 0);
    if (e != cudaSuccess) return e;
    *host = block + used;
    *dev = static_cast<int*>(at) + used;
    ++used;
    return cudaSuccess;
}

size_t type_size(int t) { return t == PTQ8_F32 ? 4 : 2; }

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// What every call checks first: a wait of an earlier call that ran out, until it is cleared.
int ready(ptq8_ops* o) {
    if (*static_cast<volatile int*>(o->error))
        return fail(o, PTQ8_ERR_TIMEOUT, "a device wait of an earlier call ran out (code %d); its outputs are invalid",
                    *o->error);
    return PTQ8_OK;
}

int cuda_fail(ptq8_ops* o, const char* what, cudaError_t e) {
    cudaGetLastError();   // reported here: the process's next check must not find it again
    return fail(o, PTQ8_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int check_rows(ptq8_ops* o, const ptq8_rows_args& a) {
    const char* w = "quantize_rows";
    if (a.x_type < PTQ8_F32 || a.x_type > PTQ8_BF16) return fail(o, PTQ8_ERR_INVALID, "%s: x_type %d", w, a.x_type);
    if (a.width <= 0 || a.width > PTQ8_MAX_ROW_WIDTH)
        return fail(o, PTQ8_ERR_INVALID, "%s: width %d (1 to %d)", w, a.width, PTQ8_MAX_ROW_WIDTH);
    if (a.x_rows < 0 || a.n_rows < 0 || a.n_rows > 0x7FFFFFFFLL)
        return fail(o, PTQ8_ERR_INVALID, "%s: x_rows %lld, n_rows %lld", w, a.x_rows, a.n_rows);
    if (!a.rows && a.n_rows != a.x_rows)
        return fail(o, PTQ8_ERR_INVALID, "%s: n_rows %lld without a row index, but x has %lld rows", w, a.n_rows, a.x_rows);
    if (a.ldx < a.width && a.x_rows > 1) return fail(o, PTQ8_ERR_INVALID, "%s: ldx %lld < width %d", w, a.ldx, a.width);
    if (a.ldc < a.width && a.n_rows > 1) return fail(o, PTQ8_ERR_INVALID, "%s: ldc %lld < width %d", w, a.ldc, a.width);
    if (a.n_rows == 0) return PTQ8_OK;
    if ((!a.x && a.x_rows) || !a.codes || !a.scale) return fail(o, PTQ8_ERR_INVALID, "%s: null pointer", w);
    if (!aligned(a.x, type_size(a.x_type))) return fail(o, PTQ8_ERR_INVALID, "%s: x is not aligned to its element type", w);
    if (!aligned(a.rows, 4) || !aligned(a.scale, 4)) return fail(o, PTQ8_ERR_INVALID, "%s: rows or scale not aligned to 4 bytes", w);
    return PTQ8_OK;
}

int check_linear(ptq8_ops* o, const ptq8_linear_args& a, bool grouped) {
    const char* w = grouped ? "linear_grouped" : "linear";
    if (a.w_bits != 8 && a.w_bits != 4) return fail(o, PTQ8_ERR_INVALID, "%s: w_bits %d (8 or 4)", w, a.w_bits);
    if (a.epilogue != PTQ8_EPI_NONE && a.epilogue != PTQ8_EPI_SWIGLU)
        return fail(o, PTQ8_ERR_INVALID, "%s: epilogue %d", w, a.epilogue);
    if (a.y_type < PTQ8_F32 || a.y_type > PTQ8_BF16) return fail(o, PTQ8_ERR_INVALID, "%s: y_type %d", w, a.y_type);
    if (a.in_features <= 0 || a.in_features > PTQ8_MAX_IN_FEATURES)
        return fail(o, PTQ8_ERR_INVALID, "%s: in_features %d (1 to %d: int32 sums)", w, a.in_features, PTQ8_MAX_IN_FEATURES);
    if (a.out_features <= 0 || a.out_features > (1 << 24))
        return fail(o, PTQ8_ERR_INVALID, "%s: out_features %d", w, a.out_features);
    if (a.rows < 0 || a.rows > 0x7FFFFF00LL) return fail(o, PTQ8_ERR_INVALID, "%s: rows %lld", w, a.rows);
    const long long wide = a.w_bits == 4 ? (a.in_features + 1) / 2 : a.in_features;
    const long long channels = static_cast<long long>(a.out_features) * (a.epilogue == PTQ8_EPI_SWIGLU ? 2 : 1);
    if (a.ldx < a.in_features && a.rows > 1) return fail(o, PTQ8_ERR_INVALID, "%s: ldx %lld < in_features %d", w, a.ldx, a.in_features);
    if (a.ldw < wide && channels > 1) return fail(o, PTQ8_ERR_INVALID, "%s: ldw %lld < %lld bytes of a weight row", w, a.ldw, wide);
    if (a.ldy < a.out_features && a.rows > 1) return fail(o, PTQ8_ERR_INVALID, "%s: ldy %lld < out_features %d", w, a.ldy, a.out_features);
    if (grouped) {
        if (a.groups <= 0 || a.groups > PTQ8_MAX_GROUPS)
            return fail(o, PTQ8_ERR_INVALID, "%s: groups %d (1 to %d)", w, a.groups, PTQ8_MAX_GROUPS);
        if (a.groups > 1 && a.w_group_stride < a.ldw * (channels - 1) + wide)
            return fail(o, PTQ8_ERR_INVALID, "%s: w_group_stride %lld: groups overlap", w, a.w_group_stride);
        if (!a.offsets) return fail(o, PTQ8_ERR_INVALID, "%s: null offsets", w);
    }
    if (a.rows == 0) return PTQ8_OK;
    if (!a.x || !a.x_scale || !a.w || !a.w_scale || !a.y) return fail(o, PTQ8_ERR_INVALID, "%s: null pointer", w);
    if (!aligned(a.y, type_size(a.y_type))) return fail(o, PTQ8_ERR_INVALID, "%s: y is not aligned to its element type", w);
    if (!aligned(a.x_scale, 4) || !aligned(a.w_scale, 4) || !aligned(a.bias, 4) || (grouped && !aligned(a.offsets, 4)))
        return fail(o, PTQ8_ERR_INVALID, "%s: x_scale, w_scale, bias or offsets not aligned to 4 bytes", w);
    return PTQ8_OK;
}

using RowsKernel = void (*)(RowsParams);

struct RowsVariant {
    int tpr;      // threads per row
    int vecs;     // vectors of 16 bytes that they hold (0: any number, read twice)
    RowsKernel plain, any;
};

template <typename T, int TPR, int NV>
RowsVariant rows_variant() {
    return {TPR, TPR * NV, rows_kernel<T, TPR, NV, true>, rows_kernel<T, TPR, NV, false>};
}

// By row length.  With much to read four vectors a thread, which share the row's statistics (16384 rows of
// 2048 f16: 15.8 us, with two vectors a thread 18.8); with less more threads a row, which finish sooner
// (2000 rows of 2048 bf16: 4.5 us, with four vectors 6.1; 300 of 4096: 2.7 and 3.5).
constexpr long long kManyVectors = 1LL << 20;

template <typename T>
const RowsVariant& rows_for(int vecs, bool many) {
    static const RowsVariant most[] = {rows_variant<T, 32, 1>(),  rows_variant<T, 32, 2>(),  rows_variant<T, 32, 4>(),
                                       rows_variant<T, 64, 4>(),  rows_variant<T, 128, 4>(), rows_variant<T, 256, 4>(),
                                       rows_variant<T, 512, 4>(), rows_variant<T, 1024, 4>()};
    static const RowsVariant soon[] = {rows_variant<T, 32, 1>(),  rows_variant<T, 64, 1>(),  rows_variant<T, 128, 1>(),
                                       rows_variant<T, 128, 2>(), rows_variant<T, 256, 2>(), rows_variant<T, 512, 2>()};
    static const RowsVariant any = rows_variant<T, 512, 0>();
    if (!many)
        for (const RowsVariant& v : soon)
            if (vecs <= v.vecs) return v;
    for (const RowsVariant& v : most)
        if (vecs <= v.vecs) return v;
    return any;
}

int run_rows(ptq8_ops* o, const ptq8_rows_args& a, cudaStream_t st) {
    const RowsParams p{a.x, a.codes, a.scale, a.rows, static_cast<size_t>(a.ldx), static_cast<size_t>(a.ldc), a.x_rows, a.n_rows, a.width};
    const int size = static_cast<int>(type_size(a.x_type)), vecs = (a.width + 16 / size - 1) / (16 / size);
    const bool many = vecs * a.n_rows >= kManyVectors;
    const RowsVariant& v = a.x_type == PTQ8_F32   ? rows_for<float>(vecs, many)
                           : a.x_type == PTQ8_F16 ? rows_for<__half>(vecs, many)
                                                  : rows_for<__nv_bfloat16>(vecs, many);
    const int lanes = 16 / size;   // elements of a vector
    const bool plain = a.width % lanes == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && (a.x_rows <= 1 || a.ldx % lanes == 0) &&
                       reinterpret_cast<uintptr_t>(a.codes) % lanes == 0 && (a.n_rows <= 1 || a.ldc % lanes == 0);
    const int block = std::max(128, v.tpr), per = block / v.tpr;
    const cudaError_t e = launch(plain ? v.plain : v.any, dim3(static_cast<unsigned>((a.n_rows + per - 1) / per)), dim3(block), 0, 1, st, p);
    return e == cudaSuccess ? PTQ8_OK : cuda_fail(o, "quantize_rows", e);
}

// ---- the tensor-core kernel's variants

using TcKernel = void (*)(const CUtensorMap, const CUtensorMap, const TcParams);

struct Variant {
    int cg, tn;            // CTAs per tile, tokens per tile
    bool w4, gated;
    TcKernel kernel;
    int threads, stage, depth, cols, acc_bufs, a_bufs, turns, x_rows, per_sm;
};

template <int CG, int TN, bool W4, bool GATED>
Variant variant() {
    using Sh = TcShape<CG, TN, W4, GATED>;
    return {CG, TN, W4, GATED, linear_tc_kernel<CG, TN, W4, GATED>, Sh::kThreads, Sh::kStage, 128 * Sh::KD, Sh::kCols, Sh::kAccBufs, Sh::kABufs, Sh::kTurns, Sh::XR, Sh::kPerSm};
}

const Variant kVariants[] = {
    variant<1, 16, false, false>(),  variant<1, 16, false, true>(),  variant<1, 16, true, false>(),  variant<1, 16, true, true>(),
    variant<1, 32, false, false>(),  variant<1, 32, false, true>(),  variant<1, 32, true, false>(),  variant<1, 32, true, true>(),
    variant<1, 64, false, false>(),  variant<1, 64, false, true>(),  variant<1, 64, true, false>(),  variant<1, 64, true, true>(),
    variant<1, 128, false, false>(), variant<1, 128, false, true>(), variant<1, 128, true, false>(), variant<1, 128, true, true>(),
    variant<2, 128, false, false>(), variant<2, 128, false, true>(), variant<2, 128, true, true>(),
    variant<2, 256, false, false>(), variant<2, 256, true, false>(),
};

// Dynamic shared memory of a CTA that shares its SM with another, or not.
constexpr int kSmemTwo = 110 * 1024, kSmemOne = 222 * 1024;

// And at least: TMEM is allocated for as many CTAs as are meant to share an SM, so that a further one's allocation would
// wait, and clusters whose CTAs wait so on two SMs for each other's would wait for good.  78 KB keep a third CTA from two
// that share, 160 KB any other from one that has its SM's columns to itself (the SM's 228 KB hold 1 KB more per CTA).
constexpr int kLeastTwo = 78 * 1024, kLeastOne = 160 * 1024;

// Shared memory beside the stages: their alignment, the tile list, a split's partial sums.
int smem_beside(const Variant& v, int split, int list_bytes) { return 1024 + list_bytes + (split > 1 ? v.cols * 128 * 4 : 0); }

// Unpacking sets take turns at the blocks, and a barrier's parity tells two phases apart: each set has to wait for
// every phase of the stages that it waits for.  So the stages are a multiple of the turns, which gives each stage
// one set.  (Otherwise a set could ask for a stage while the load before, another set's, is still on its way, and
// take the phase before that for the one it asks for.)
int stages_of(const Variant& v, int split, int list_bytes) {
    const int most = std::min(kMaxLinStages, ((v.per_sm == 2 ? kSmemTwo : kSmemOne) - smem_beside(v, split, list_bytes)) / v.stage);
    return most / v.turns * v.turns;
}

int smem_of(const Variant& v, int split, int list_bytes) {
    return std::max(v.per_sm == 2 ? kLeastTwo : kLeastOne, smem_beside(v, split, list_bytes) + stages_of(v, split, list_bytes) * v.stage);
}

int list_bytes_of(const ptq8_linear_args& a, bool listed) { return listed ? ((a.groups + 1) * 8 + 127) / 128 * 128 : 0; }

// A launch's time in cycles, up to what all variants share.  Per stage a CTA takes the longest of its chain (the
// MMAs and the wait before them) and, for the CTAs that share an SM, their MMAs, their loads at what an SM draws
// from L2, and the widening of int4 weights.  Few tiles are worth a cluster each: a split pays for sending and
// joining its sums, and clusters of 4 and 8 do not fill every GPC.
//
// How well it chooses: 902 calls (1 to 8192 tokens, 512 to 16384 features, 1 to 64 groups; int8 and int4, with and
// without SwiGLU) were timed as every variant and split not far too long for them, 6711 in all, each with operands from DRAM,
// with operands in L2, and called from Python in a loop.  The choice is 2.5, 2.3 and 2.8 % slower than the fastest
// variant on average, 14 to 19 % at the 95th percentile, and 64 % at most: tiles of 64 tokens with SwiGLU, which hold two
// stages, are rated too well where the weights come from DRAM (128 tokens, 4096 -> 2 x 4096 int8: 25.7 us, a pair of 128
// tokens 16.4).  Constants fitted to half of the calls did no better on the other half than these.
float estimate(int sms, const ptq8_linear_args& a, int groups, const Variant& v, int split) {
    constexpr float kMma = 77.5f, kMmaTmem = 104;    // least cycles of an MMA, M operand in shared memory or TMEM
    constexpr float kMmaTmemPair = 102;              // the latter for a pair: 4096 x 4096 x 4096 gated 102 us, one CTA a tile 107
    constexpr float kWait = 144, kWaitTwo = 47;      // wait of the MMA warp per block (two blocks a stage)
    constexpr float kLoad = 61;                      // bytes per cycle into an SM
    constexpr float kWiden = 225;                    // int4: cycles of an SM per tile of 128 x 128 codes
    constexpr float kColumn = 12, kPush = 54;        // epilogue per accumulator column; sending one to a peer
    constexpr float kSplit = 645, kWave = 1055;      // a split tile's joining; a further wave of clusters
    constexpr float kCluster = 430;                  // start of a launch with clusters
    constexpr float kRagged = 0.62f;                 // part of a row tile that uneven groups waste each
    constexpr float kFill4 = 0.96f, kFill8 = 0.82f;  // share of the SMs that clusters of 4 and of 8 can take
    constexpr float kPacked = 0.47f;                 // CTAs per SM from which two come to share one
    const float h = v.gated ? 2 : 1, rows = static_cast<float>(a.rows);
    const float used = static_cast<float>(std::min<long long>(groups, a.rows)), mean = rows / used;
    const float row_tiles = groups > 1 ? std::max(used, std::ceil(used * (mean / v.tn + kRagged))) : std::ceil(rows / v.tn);
    const float tiles = row_tiles * static_cast<float>((a.out_features + 128 * v.cg - 1) / (128 * v.cg));
    const float blocks = std::ceil(std::ceil(a.in_features / 128.0f) / split);
    const float columns = std::min<float>(v.tn, std::ceil(std::ceil(mean) / (16 * v.cg)) * (16 * v.cg));
    const float share = v.per_sm == 2 && tiles * v.cg * split > kPacked * sms ? 2 : 1;
    const float mma = 4 * h * std::max(!v.w4 ? kMma : v.cg == 2 ? kMmaTmemPair : kMmaTmem, columns / 2);
    const float load = (h * 128 * (v.w4 ? 64 : 128) + v.x_rows * 128) / kLoad;
    const float block = std::max({mma + (v.depth > 128 ? kWaitTwo : kWait), share * mma, share * load, share * (v.w4 ? kWiden * h : 0)});
    const float fill = split == 8 ? kFill8 : split == 4 ? kFill4 : 1;
    const float slots = std::max(1.0f, std::floor(std::floor(sms * v.per_sm * fill) / (v.cg * split)));
    const float waves = std::ceil(tiles / slots);
    float out = kColumn * columns * h / (v.tn >= 128 ? 2 : 1);
    if (split > 1) out += kSplit + kPush * columns * h;
    const float start = v.cg * split > 1 ? kCluster : 0;
    if (split == 1 && waves > 1) return start + waves * std::max(blocks * block, out) + out;
    return start + waves * (blocks * block + out + (split > 1 ? kWave : 0));
}

// Whether a call can run as variant v with the sum over input features split s ways.
bool serves(const ptq8_linear_args& a, bool listed, const Variant& v, int s) {
    if (v.w4 != (a.w_bits == 4) || v.gated != (a.epilogue == PTQ8_EPI_SWIGLU)) return false;
    if (s < 1 || s > (v.cg == 2 ? 1 : 8) || (s & (s - 1)) || static_cast<long long>(s - 1) * v.depth >= a.in_features) return false;
    // the operand tile of a block is free when its stage is; a split's sums leave from the stages' memory
    const int stages = stages_of(v, s, list_bytes_of(a, listed));
    return stages >= std::max(2, v.a_bufs) && (s == 1 || stages * v.stage >= v.cols * 128 * 4);
}

// The variant of the least estimate, among tiles not much longer than the rows of a group.
const Variant* choose(int sms, const ptq8_linear_args& a, bool listed, int& split) {
    const int groups = listed ? a.groups : 1;
    const float mean = static_cast<float>(a.rows) / std::min<long long>(groups, a.rows);
    const Variant* best = nullptr;
    float least = 0;
    for (const Variant& v : kVariants) {
        if (v.tn > 16 && v.tn >= 4 * v.cg * mean) continue;
        for (int s = 1; s <= 8; s *= 2) {
            if (!serves(a, listed, v, s)) continue;
            const float t = estimate(sms, a, groups, v, s);
            if (!best || t < least) best = &v, split = s, least = t;
        }
    }
    return best;
}

bool aligned16(long long v) { return v % 16 == 0; }

// What TMA and 16-byte loads need of the operands' layout (a pitch that no second row uses does not count).
bool vector_layout(const ptq8_linear_args& a, bool grouped) {
    return aligned16(reinterpret_cast<uintptr_t>(a.x)) && aligned16(reinterpret_cast<uintptr_t>(a.w)) &&
           (aligned16(a.ldx) || a.rows == 1) && (aligned16(a.ldw) || a.out_features == 1 && a.epilogue == PTQ8_EPI_NONE) &&
           (!grouped || a.groups == 1 || (aligned16(a.w_group_stride) && a.w_group_stride < (1LL << 39))) && a.ldx < (1LL << 39) && a.ldw < (1LL << 39);
}

int encode(ptq8_ops* o, CUtensorMap* m, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
           const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
    const cuuint32_t one[3] = {1, 1, 1};
    const CUresult r = o->encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, one,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? PTQ8_OK : fail(o, PTQ8_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
}

int run_tc(ptq8_ops* o, const ptq8_linear_args& a, const LinearParams& l, cudaStream_t st) {
    const bool gated = a.epilogue == PTQ8_EPI_SWIGLU, w4 = a.w_bits == 4;
    int split = 1;
    const Variant* v = nullptr;
    if (o->variant < 0)
        v = choose(o->sms, a, l.offsets != nullptr, split);
    else if (serves(a, l.offsets != nullptr, kVariants[o->variant], o->split))
        v = &kVariants[o->variant], split = o->split;
    if (!v) return fail(o, PTQ8_ERR_INVALID, "linear: variant %d with split %d does not serve this call", o->variant, o->split);
    const long long channels = static_cast<long long>(a.out_features) * (gated ? 2 : 1);
    const int wide = w4 ? (a.in_features + 1) / 2 : a.in_features;
    CUtensorMap mx, mw;
    {
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.in_features), static_cast<cuuint64_t>(a.rows)};
        const cuuint64_t pitch[1] = {static_cast<cuuint64_t>(a.rows > 1 ? a.ldx : (a.in_features + 15) / 16 * 16)};
        const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(v->x_rows)};
        if (const int rc = encode(o, &mx, 2, a.x, dims, pitch, box, CU_TENSOR_MAP_SWIZZLE_128B)) return rc;
    }
    {
        const cuuint64_t ldw = channels > 1 ? a.ldw : (wide + 15) / 16 * 16;
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(wide), static_cast<cuuint64_t>(channels), static_cast<cuuint64_t>(l.groups)};
        const cuuint64_t pitch[2] = {ldw, l.groups > 1 ? static_cast<cuuint64_t>(l.gstride) : ldw};
        const cuuint32_t box[3] = {w4 ? 64u : 128u, 128, 1};
        if (const int rc = encode(o, &mw, 3, a.w, dims, pitch, box, w4 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B))
            return rc;
    }
    TcParams p{};
    p.l = l;
    p.kblocks = (a.in_features + v->depth - 1) / v->depth;
    p.split = split;
    p.ctiles = (a.out_features + 128 * v->cg - 1) / (128 * v->cg);
    p.list_bytes = list_bytes_of(a, l.offsets != nullptr);
    p.acc_bufs = split > 1 ? 1 : v->acc_bufs;
    p.tmem_cols = 32;
    while (static_cast<int>(p.tmem_cols) < v->cols * p.acc_bufs) p.tmem_cols *= 2;
    if (w4) p.tmem_cols = 512 / v->per_sm;
    p.wait_limit = o->wait_limit;
    p.err = o->error_dev;
    p.stall = o->stall;
    p.stages = stages_of(*v, split, p.list_bytes);
    const int smem = smem_of(*v, split, p.list_bytes);
    // tiles at most: each group's last tile may be partly filled
    const long long row_tiles = l.offsets ? a.rows / v->tn + std::min<long long>(l.groups, a.rows) : (a.rows + v->tn - 1) / v->tn;
    const long long tiles = row_tiles * p.ctiles;
    if (tiles > 0x3FFFFFFF / 8) return fail(o, PTQ8_ERR_INVALID, "linear: %lld tiles", tiles);
    const int per = v->cg * split, slots = o->sms * v->per_sm / per;
    const long long clusters = split > 1 ? tiles : std::min<long long>(tiles, slots);
    const cudaError_t e = launch(v->kernel, dim3(static_cast<unsigned>(clusters * per)), dim3(v->threads), smem, per, st, mx, mw, p);
    return e == cudaSuccess ? PTQ8_OK : cuda_fail(o, "linear", e);
}

using FewKernel = void (*)(FewParams);

template <int MT>
FewKernel few_kernel(bool w4, bool gated) {
    return w4 ? (gated ? linear_few_kernel<MT, true, true> : linear_few_kernel<MT, true, false>)
              : (gated ? linear_few_kernel<MT, false, true> : linear_few_kernel<MT, false, false>);
}

// Up to four tokens, or one a group on average, while the weights that they read stay small.  Weights from DRAM, us here
// and as the best tensor-core tile of 16:
//   tokens x 4096 x channels     4096 int8   4608 int8   5120 int8    6144 int8   8192 int4   10240 int4   12288 int4
//   1                            5.2   5.9   5.9   6.8   9.7    7.2   10.2  7.5   5.9   7.5   7.2    9.6   7.4   10.0
//   2                            6.0   5.9   6.7   6.8   11.0   7.2   11.5  7.5   8.5   7.6   9.4    9.6   9.3   10.0
//   4                            5.9   6.0   6.6   7.0   8.8    7.4   9.0   7.5   7.6   7.7   11.4   9.8   12.1  10.0
// Above 18 MB rows are no longer shared by two warps, so that a few blocks more than there are SMs make a second turn, and
// bulk copies into shared memory keep more bytes in flight (2048 x 10240 int8, one token, is the other way: 6.6 and 7.4 us).
// One token on int4 codes goes further, since its tiles wait for the unpacking.
// Rows that are not whole vectors of 16 bytes of weights go to the tensor cores too: at 2001 x 1270 joining single bytes
// made four tokens 1.2 (int4 1.6) times slower than a tile.
// The host does not know how ragged groups are.  64 rows of 64 experts, 1024 -> 256: one each or at random 5.8 us (a tile 8.4),
// half of them in one group 20 us (7.2), all of them 34 us (6.7): a group's rows pass over its weights two at a time.
bool few_rows(const ptq8_linear_args& a, int groups) {
    const long long most = a.w_bits == 4 && a.rows == 1 ? 24LL << 20 : 18LL << 20;
    const long long channels = static_cast<long long>(a.out_features) * (a.epilogue == PTQ8_EPI_SWIGLU ? 2 : 1);
    const long long bytes = std::min<long long>(groups, a.rows) * channels * a.in_features * a.w_bits / 8;
    return (groups > 1 ? a.rows <= groups : a.rows <= 4) && bytes <= most && a.in_features % (a.w_bits == 4 ? 32 : 16) == 0;
}

int run_few(ptq8_ops* o, const ptq8_linear_args& a, const LinearParams& l, cudaStream_t st) {
    const bool gated = a.epilogue == PTQ8_EPI_SWIGLU, w4 = a.w_bits == 4;
    const int channels = kFewRows / (gated ? 2 : 1);   // of a warp
    const long long sets = (static_cast<long long>(a.out_features) + channels - 1) / channels;
    const long long used = std::min<long long>(l.groups, a.rows);
    FewParams p{l, 1};
    while (p.ks < kFewWarps && sets * used * p.ks < 1LL * kFewWarps * o->sms) p.ks *= 2;
    // groups differ in their rows: room for two of them at least
    const long long rows = l.groups > 1 ? std::max(2LL, a.rows / used) : a.rows;
    const FewKernel kernel = rows == 1 ? few_kernel<1>(w4, gated) : rows == 2 ? few_kernel<2>(w4, gated) : few_kernel<4>(w4, gated);
    const int per = kFewWarps / p.ks;
    const cudaError_t e = launch(kernel, dim3(static_cast<unsigned>((sets + per - 1) / per), static_cast<unsigned>(l.groups)),
                                 dim3(32 * kFewWarps), 0, 1, st, p);
    return e == cudaSuccess ? PTQ8_OK : cuda_fail(o, "linear", e);
}

int run_linear(ptq8_ops* o, const ptq8_linear_args& a, bool grouped, cudaStream_t st) {
    LinearParams p{};
    p.x = a.x;
    p.w = static_cast<const uint8_t*>(a.w);
    p.xs = a.x_scale;
    p.ws = a.w_scale;
    p.bias = a.bias;
    p.y = a.y;
    p.offsets = grouped ? a.offsets : nullptr;
    p.ldx = a.ldx;
    p.ldw = a.ldw;
    p.gstride = grouped ? a.w_group_stride : 0;
    p.ldy = a.ldy;
    p.rows = a.rows;
    p.k = a.in_features;
    p.n = a.out_features;
    p.groups = grouped ? a.groups : 1;
    p.y_type = a.y_type;
    const bool gated = a.epilogue == PTQ8_EPI_SWIGLU, w4 = a.w_bits == 4;
    const bool vectors = vector_layout(a, grouped);
    if (o->variant >= 0 && !vectors) return fail(o, PTQ8_ERR_INVALID, "linear: variant %d does not serve this layout", o->variant);
    if (vectors) return few_rows(a, p.groups) && o->variant < 0 ? run_few(o, a, p, st) : run_tc(o, a, p, st);
    const long long row_tiles = (a.rows + kAnyTile - 1) / kAnyTile;
    // blocks stride over the channel tiles (x) and over a group's row tiles (y)
    const dim3 grid(static_cast<unsigned>((a.out_features + kAnyTile - 1) / kAnyTile),
                    static_cast<unsigned>(std::min<long long>(row_tiles, grouped ? 64 : 65535)), static_cast<unsigned>(p.groups));
    auto kernel = w4 ? (gated ? linear_any_kernel<true, true> : linear_any_kernel<true, false>)
                     : (gated ? linear_any_kernel<false, true> : linear_any_kernel<false, false>);
    const cudaError_t e = launch(kernel, grid, dim3(256), 0, 1, st, p);
    return e == cudaSuccess ? PTQ8_OK : cuda_fail(o, "linear", e);
}

int product(ptq8_ops* o, const ptq8_linear_args* a, bool grouped, void* stream) {
    if (!o) return PTQ8_ERR_INVALID;
    if (!a) return fail(o, PTQ8_ERR_INVALID, "null arguments");
    if (const int rc = check_linear(o, *a, grouped)) return rc;
    if (const int rc = ready(o)) return rc;
    if (a->rows == 0) return PTQ8_OK;
    OnDevice on(o->device);
    if (on.rc != cudaSuccess) return cuda_fail(o, "cudaSetDevice", on.rc);
    return run_linear(o, *a, grouped, static_cast<cudaStream_t>(stream));
}

// ptq8_linear_choose and ptq8_linear_choose_as (variant >= 0).
int choice_of(int sms, const ptq8_linear_args* args, bool grouped, int variant, int split, ptq8_linear_choice* c) {
    ptq8_ops none;   // takes the message of a refusal
    if (!args || !c || sms < 1 || variant >= static_cast<int>(std::size(kVariants))) return PTQ8_ERR_INVALID;
    const ptq8_linear_args& a = *args;
    if (const int rc = check_linear(&none, a, grouped)) return rc;
    if (a.rows == 0) return PTQ8_ERR_INVALID;   // runs on no kernel
    *c = ptq8_linear_choice{};
    const bool vectors = vector_layout(a, grouped);
    if (variant < 0 && (!vectors || few_rows(a, grouped ? a.groups : 1))) {
        c->kernel = vectors ? PTQ8_KERNEL_FEW : PTQ8_KERNEL_ANY;
        return PTQ8_OK;
    }
    const Variant* v = variant < 0 ? choose(sms, a, grouped, split) : &kVariants[variant];
    if (!vectors || !serves(a, grouped, *v, split)) return PTQ8_ERR_INVALID;
    const int list = list_bytes_of(a, grouped), stages = stages_of(*v, split, list);
    *c = {PTQ8_KERNEL_TILES, static_cast<int>(v - kVariants), v->cg, v->tn, a.w_bits, a.epilogue, split, stages, v->turns, v->a_bufs,
          smem_of(*v, split, list)};
    return PTQ8_OK;
}

}  // namespace

extern "C" {

ptq8_ops* ptq8_ops_create(int device, char* err, size_t errlen) {
    try {
        cudaDeviceProp prop;
        cudaError_t e = cudaGetDeviceProperties(&prop, device);
        if (e == cudaSuccess && prop.major != 10) {
            say(err, errlen, "device is not sm_100: %s", prop.name);
            return nullptr;
        }
        OnDevice on(device);
        if (e == cudaSuccess) e = on.rc;
        void* encode = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSuccess;
        if (e == cudaSuccess) e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &encode, cudaEnableDefault, &q);
        if (e == cudaSuccess && q != cudaDriverEntryPointSuccess) e = cudaErrorNotSupported;
        for (const Variant& v : kVariants)
            if (e == cudaSuccess)
                e = cudaFuncSetAttribute(reinterpret_cast<const void*>(v.kernel), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         v.per_sm == 2 ? kSmemTwo : kSmemOne);
        int* host = nullptr;
        int* dev = nullptr;
        if (e == cudaSuccess) e = error_word(&host, &dev);
        if (e != cudaSuccess) {
            cudaGetLastError();   // reported here: the process's next check must not find it again
            say(err, errlen, "ptq8_ops_create: %s", cudaGetErrorString(e));
            return nullptr;
        }
        auto* o = new (std::nothrow) ptq8_ops();
        if (!o) {
            say(err, errlen, "ptq8_ops_create: out of host memory");
            return nullptr;
        }
        o->device = device;
        o->sms = prop.multiProcessorCount;
        o->error = host;
        o->error_dev = dev;
        o->encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(encode);
        say(err, errlen, "");
        return o;
    } catch (...) {   // std::mutex may throw
        say(err, errlen, "ptq8_ops_create: a host lock failed");
        return nullptr;
    }
}

void ptq8_ops_destroy(ptq8_ops* o) { delete o; }

const char* ptq8_ops_last_error(const ptq8_ops* o) { return o ? o->err : "null handle"; }

int ptq8_ops_check_device_error(ptq8_ops* o, void* stream) {
    if (!o) return PTQ8_ERR_INVALID;
    OnDevice on(o->device);
    cudaError_t e = on.rc;
    if (e == cudaSuccess) e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return cuda_fail(o, "cudaStreamSynchronize", e);
    const int rc = ready(o);
    *static_cast<volatile int*>(o->error) = 0;
    return rc;
}

int ptq8_ops_set_wait_test(ptq8_ops* o, long long wait_limit_cycles, int stall_first_load) {
    if (!o) return PTQ8_ERR_INVALID;
    o->wait_limit = wait_limit_cycles > 0 ? wait_limit_cycles : kWaitLimitCycles;
    o->stall = stall_first_load != 0;
    return PTQ8_OK;
}

int ptq8_linear_variants(void) { return static_cast<int>(std::size(kVariants)); }

int ptq8_linear_choose(int sms, const ptq8_linear_args* a, int grouped, ptq8_linear_choice* c) {
    return choice_of(sms, a, grouped != 0, -1, 1, c);
}

int ptq8_linear_choose_as(int sms, const ptq8_linear_args* a, int grouped, int variant, int split, ptq8_linear_choice* c) {
    return variant < 0 ? PTQ8_ERR_INVALID : choice_of(sms, a, grouped != 0, variant, split, c);
}

int ptq8_ops_set_choice_test(ptq8_ops* o, int variant, int split) {
    if (!o) return PTQ8_ERR_INVALID;
    if (variant >= ptq8_linear_variants()) return fail(o, PTQ8_ERR_INVALID, "variant %d of %d", variant, ptq8_linear_variants());
    o->variant = variant < 0 ? -1 : variant;
    o->split = split;
    return PTQ8_OK;
}

int ptq8_quantize_rows(ptq8_ops* o, const ptq8_rows_args* a, void* stream) {
    if (!o) return PTQ8_ERR_INVALID;
    if (!a) return fail(o, PTQ8_ERR_INVALID, "null arguments");
    if (const int rc = check_rows(o, *a)) return rc;
    if (const int rc = ready(o)) return rc;
    if (a->n_rows == 0) return PTQ8_OK;
    OnDevice on(o->device);
    if (on.rc != cudaSuccess) return cuda_fail(o, "cudaSetDevice", on.rc);
    return run_rows(o, *a, static_cast<cudaStream_t>(stream));
}

int ptq8_linear(ptq8_ops* o, const ptq8_linear_args* a, void* stream) { return product(o, a, false, stream); }

int ptq8_linear_grouped(ptq8_ops* o, const ptq8_linear_args* a, void* stream) { return product(o, a, true, stream); }

}  // extern "C"
