// Token operators: host side of ptq8_linear_w4 (argument checks, kernel choice, launch) and its extern "C" boundary.

#include <algorithm>

#include "ptq8_ops.cuh"
#include "ptq8_w4.cuh"

using namespace ptq8;

// what the Python mirror packs
static_assert(sizeof(ptq8_linear_w4_args) == 112, "argument struct");

namespace {

int check_w4(ptq8_ops* o, const ptq8_linear_w4_args& a) {
    const char* w = "linear_w4";
    if (a.epilogue != PTQ8_EPI_NONE && a.epilogue != PTQ8_EPI_SWIGLU) return fail(o, PTQ8_ERR_INVALID, "%s: epilogue %d", w, a.epilogue);
    const struct {
        int type;
        const char* name;
    } types[] = {{a.x_type, "x_type"}, {a.scale_type, "scale_type"}, {a.y_type, "y_type"}};
    for (const auto& t : types)
        if (t.type < PTQ8_F32 || t.type > PTQ8_BF16) return fail(o, PTQ8_ERR_INVALID, "%s: %s %d", w, t.name, t.type);
    if (a.in_features <= 0 || a.in_features > (1 << 24)) return fail(o, PTQ8_ERR_INVALID, "%s: in_features %d", w, a.in_features);
    if (a.out_features <= 0 || a.out_features > (1 << 24)) return fail(o, PTQ8_ERR_INVALID, "%s: out_features %d", w, a.out_features);
    if (a.group <= 0) return fail(o, PTQ8_ERR_INVALID, "%s: group %d", w, a.group);
    if (a.rows < 0 || a.rows > 0x7FFFFF00LL) return fail(o, PTQ8_ERR_INVALID, "%s: rows %lld", w, a.rows);
    const long long wide = (a.in_features + 1) / 2, groups = (a.in_features - 1) / a.group + 1;
    const long long channels = static_cast<long long>(a.out_features) * (a.epilogue == PTQ8_EPI_SWIGLU ? 2 : 1);
    if (a.ldx < a.in_features && a.rows > 1) return fail(o, PTQ8_ERR_INVALID, "%s: ldx %lld < in_features %d", w, a.ldx, a.in_features);
    if (a.ldw < wide && channels > 1) return fail(o, PTQ8_ERR_INVALID, "%s: ldw %lld < %lld bytes of a weight row", w, a.ldw, wide);
    if (a.lds < groups && channels > 1) return fail(o, PTQ8_ERR_INVALID, "%s: lds %lld < %lld groups", w, a.lds, groups);
    if (a.ldy < a.out_features && a.rows > 1) return fail(o, PTQ8_ERR_INVALID, "%s: ldy %lld < out_features %d", w, a.ldy, a.out_features);
    if (a.rows == 0) return PTQ8_OK;
    if (!a.x || !a.w || !a.w_scale || !a.y) return fail(o, PTQ8_ERR_INVALID, "%s: null pointer", w);
    if (!aligned(a.x, type_size(a.x_type)) || !aligned(a.w_scale, type_size(a.scale_type)) || !aligned(a.y, type_size(a.y_type)) || !aligned(a.bias, 4))
        return fail(o, PTQ8_ERR_INVALID, "%s: x, w_scale, bias or y is not aligned to its element type", w);
    return PTQ8_OK;
}

constexpr int kW4Segment = 16;   // chunks

struct W4Variant {
    int type, vb, nt;   // of the activations; bytes that a lane takes at once; tiles of eight columns
    void (*kernel)(W4Params, W4Plan, const CUtensorMap);
    void (*exact)(W4Params, W4Plan, const CUtensorMap);   // for outputs of 32 bits
    int sums, beside;
    int (*frag)(int columns);
};

template <typename XT, int TYPE, int VB, int NT>
W4Variant w4_variant() {
    using Sh = W4Shape<XT, VB, NT>;
    static_assert(NT > 1 || kW4Smem - 1024 - Sh::kSums - kW4Segment * (Sh::frag(8) + Sh::kBeside) >= kW4Warps * kW4Box, "a segment fits beside a stage");
    return {TYPE, VB, NT, linear_w4_kernel<XT, VB, NT, false>, linear_w4_kernel<XT, VB, NT, true>, Sh::kSums, Sh::kBeside, Sh::frag};
}

#define W4_TILES(XT, TYPE, VB) w4_variant<XT, TYPE, VB, 1>(), w4_variant<XT, TYPE, VB, 2>(), w4_variant<XT, TYPE, VB, 4>()
#define W4_TYPE(XT, TYPE) W4_TILES(XT, TYPE, 4), W4_TILES(XT, TYPE, 8), W4_TILES(XT, TYPE, 16)

const W4Variant kW4Variants[] = {W4_TYPE(float, PTQ8_F32), W4_TYPE(__half, PTQ8_F16), W4_TYPE(__nv_bfloat16, PTQ8_BF16)};

using W4Few = void (*)(W4Params, int);
template <typename XT>
struct W4FewOf {
    static constexpr W4Few kKernels[2] = {linear_w4_few_kernel<XT, 1>, linear_w4_few_kernel<XT, 2>};
};
const W4Few* const kW4Few[] = {W4FewOf<float>::kKernels, W4FewOf<__half>::kKernels, W4FewOf<__nv_bfloat16>::kKernels};   // by type

// One or two tokens while the weights are small.  us here and on the tensor cores, tokens x in -> out:
//                  1024 -> 1024   4096 -> 1024   4096 -> 4096   4096 -> 14336
//   1 x bf16       2.0   4.3      2.6   6.1      4.9    6.3     14.5   12.8
//   2 x bf16       4.1   4.6      5.2   6.3      8.4    6.5     25.3   12.8
//   1 x f32        2.4   4.3      3.3   6.7      7.5    7.1     23.4   13.9
//   2 x f32        4.4   4.3      6.1   7.1      13.3   7.3     42.5   14.1
// (The activations are read again for every four weight rows, which is what large weights make it wait for.)  Rows of whole vectors.
bool few_rows(const ptq8_linear_w4_args& a, bool vectors) {
    const bool gated = a.epilogue == PTQ8_EPI_SWIGLU;
    const long long bytes = static_cast<long long>(a.out_features) * (gated ? 2 : 1) * a.in_features / 2;
    return a.rows <= 2 && bytes <= (a.rows == 1 ? 12LL << 20 : 4LL << 20) && vectors && a.in_features % 32 == 0 && aligned(a.w, 16) &&
           (a.ldw % 16 == 0 || (a.out_features == 1 && !gated));
}

int run_w4(ptq8_ops* o, const ptq8_linear_w4_args& a, cudaStream_t st) {
    W4Params p{};
    p.x = a.x;
    p.w = static_cast<const uint8_t*>(a.w);
    p.s = a.w_scale;
    p.bias = a.bias;
    p.y = a.y;
    p.ldx = a.ldx, p.ldw = a.ldw, p.lds = a.lds, p.ldy = a.ldy;
    p.rows = a.rows;
    p.k = a.in_features, p.n = a.out_features, p.group = a.group;
    p.gated = a.epilogue == PTQ8_EPI_SWIGLU;
    p.x_type = a.x_type, p.s_type = a.scale_type, p.y_type = a.y_type;
    const long long lanes = 16 / static_cast<long long>(type_size(a.x_type));
    p.vec_x = aligned(a.x, 16) && (a.rows == 1 || a.ldx % lanes == 0);
    p.wait_limit = o->wait_limit;
    p.err = o->error_dev;
    p.stall = o->stall;
    p.shift = -1;
    if ((a.group & (a.group - 1)) == 0)
        while ((1LL << ++p.shift) < a.group) {
        }
    // bytes that a lane takes at once: four lanes' stay within a group
    const int vb = a.group % 128 == 0 || a.group >= a.in_features ? 16 : a.group % 64 == 0 ? 8 : a.group % 32 == 0 ? 4 : 0;
    cudaError_t e;
    if (few_rows(a, vb && p.vec_x)) {
        const long long sets = (a.out_features - 1LL) / (p.gated ? 2 : 4) + 1;
        int ks = 1;
        while (ks < kW4FewWarps && sets * ks < 1LL * kW4FewWarps * o->sms) ks *= 2;
        const int per = kW4FewWarps / ks;
        e = launch(kW4Few[a.x_type][a.rows - 1], dim3(static_cast<unsigned>((sets + per - 1) / per)), dim3(32 * kW4FewWarps), 0, 1, st, p, ks);
    } else if (vb && a.lds < (1 << 28) && aligned(a.w, 16) && (a.ldw % 16 == 0 || (a.out_features == 1 && !p.gated)) && a.ldw < (1LL << 39)) {
        const int per_tile = a.x_type == PTQ8_F32 ? 4 : 8;   // tokens
        const int chunks = (a.in_features + kW4Chunk - 1) / kW4Chunk;
        const long long pairs = (a.out_features - 1LL) / (p.gated ? 16 : 32) + 1;   // of tiles
        // The fewest columns that take all tokens in a pass, fewer where all chunks' activations do not fit beside a stage of weights;
        // then as many stages as fit.  Not even with eight columns: a segment of kW4Segment chunks at a time.
        const W4Variant* v = nullptr;
        W4Plan plan{};
        long long passes = 0;
        for (int nt = a.rows <= per_tile ? 1 : a.rows <= 2 * per_tile ? 2 : 4; !plan.stages; nt /= 2) {
            const bool segments = nt == 0;
            for (v = kW4Variants; v->type != a.x_type || v->vb != vb || v->nt != std::max(nt, 1);) ++v;
            passes = (a.rows + v->nt * per_tile - 1) / (v->nt * per_tile);
            plan = {8, segments ? kW4Segment : chunks, segments ? (chunks + kW4Segment - 1) / kW4Segment : 1, 0, static_cast<int>(pairs), 1, 0, static_cast<int>(passes)};
            if (v->nt == 1) plan.columns = static_cast<int>(std::min<long long>(8, a.rows * (a.x_type == PTQ8_F32 ? 2 : 1)));
            // warps a pair: as many as leave the device's warps one each, if that many
            while (1 << plan.split_log < std::min(kW4Warps, plan.held) && (pairs * passes << plan.split_log) * 2 <= static_cast<long long>(kW4Warps) * o->sms) ++plan.split_log;
            const long long left = kW4Smem - 1024 - v->sums - static_cast<long long>(plan.held) * (v->frag(plan.columns) + v->beside);
            plan.stages = static_cast<int>(std::max(0LL, std::min<long long>(kW4MostStages, left / (kW4Warps * kW4Box))));
        }
        const int slots = kW4Warps >> plan.split_log, smem = v->sums + plan.held * (v->frag(plan.columns) + v->beside) + kW4Warps * plan.stages * kW4Box + 1024;
        const long long groups = (pairs + slots - 1) / slots;
        const long long x = std::min<long long>(groups, std::max<long long>(1, o->sms / passes)), y = std::min<long long>(passes, std::max<long long>(1, o->sms / x));
        plan.rounds = static_cast<int>((groups + x - 1) / x);
        const long long channels = static_cast<long long>(a.out_features) * (p.gated ? 2 : 1);
        const int wide = (a.in_features + 1) / 2;
        CUtensorMap map;
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(wide), static_cast<cuuint64_t>(channels)}, pitch[1] = {static_cast<cuuint64_t>(channels > 1 ? a.ldw : (wide + 15) / 16 * 16)};
        const cuuint32_t box[2] = {128, p.gated ? 16u : 32u}, one[2] = {1, 1};
        const CUresult r = o->encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(a.w), dims, pitch, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return fail(o, PTQ8_ERR_CUDA, "linear_w4: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
        e = launch(a.y_type == PTQ8_F32 ? v->exact : v->kernel, dim3(static_cast<unsigned>(x), static_cast<unsigned>(y)), dim3(kW4Threads), smem, 1, st, p, plan, map);
    } else {
        const long long blocks = (a.rows + kW4AnyTokens - 1) / kW4AnyTokens;
        e = launch(linear_w4_any_kernel, dim3((a.out_features + 7) / 8, static_cast<unsigned>(std::min<long long>(blocks, 65535))), dim3(256), 0, 1, st, p);
    }
    return e == cudaSuccess ? PTQ8_OK : cuda_fail(o, "linear_w4", e);
}

}  // namespace

namespace ptq8 {

cudaError_t w4_attributes() {
    for (const W4Variant& v : kW4Variants)
        for (const auto kernel : {v.kernel, v.exact}) {
            const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kW4Smem);
            if (e != cudaSuccess) return e;
        }
    return cudaSuccess;
}

}  // namespace ptq8

extern "C" {

int ptq8_linear_w4(ptq8_ops* o, const ptq8_linear_w4_args* a, void* stream) {
    if (!o) return PTQ8_ERR_INVALID;
    if (!a) return fail(o, PTQ8_ERR_INVALID, "null arguments");
    if (const int rc = check_w4(o, *a)) return rc;
    if (const int rc = ready(o)) return rc;
    if (a->rows == 0) return PTQ8_OK;
    OnDevice on(o->device);
    if (on.rc != cudaSuccess) return cuda_fail(o, "cudaSetDevice", on.rc);
    return run_w4(o, *a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
