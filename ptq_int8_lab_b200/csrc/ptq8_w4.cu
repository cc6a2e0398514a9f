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

using W4Kernel = void (*)(W4Params);

template <typename XT, int VB>
W4Kernel w4_kernel(int rt, int nt) {
    if (nt == 1) return rt == 1 ? linear_w4_kernel<XT, VB, 1, 1> : rt == 2 ? linear_w4_kernel<XT, VB, 2, 1> : linear_w4_kernel<XT, VB, 4, 1>;
    return nt == 2 ? linear_w4_kernel<XT, VB, 2, 2> : linear_w4_kernel<XT, VB, 2, 4>;
}
template <typename XT>
W4Kernel w4_kernel(int vb, int rt, int nt) {
    return vb == 16 ? w4_kernel<XT, 16>(rt, nt) : vb == 8 ? w4_kernel<XT, 8>(rt, nt) : w4_kernel<XT, 4>(rt, nt);
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
    // bytes that a lane takes at once: four lanes' stay within a group
    const int vb = a.group % 128 == 0 || a.group >= a.in_features ? 16 : a.group % 64 == 0 ? 8 : a.group % 32 == 0 ? 4 : 0;
    cudaError_t e;
    if (vb && aligned(a.w, vb) && a.ldw % vb == 0) {
        const int per_tile = a.x_type == PTQ8_F32 ? 4 : 8;   // tokens
        const int nt = a.rows <= per_tile ? 1 : a.rows <= 2 * per_tile ? 2 : 4;
        const long long tiles = (a.out_features + (p.gated ? 8 : 16) - 1LL) / (p.gated ? 8 : 16);
        const int rt = nt > 1 ? 2 : tiles <= 3LL * o->sms ? 1 : tiles <= 8LL * o->sms ? 2 : 4;
        const W4Kernel kernel = a.x_type == PTQ8_F32   ? w4_kernel<float>(vb, rt, nt)
                                : a.x_type == PTQ8_F16 ? w4_kernel<__half>(vb, rt, nt)
                                                       : w4_kernel<__nv_bfloat16>(vb, rt, nt);
        const long long blocks = (a.rows + nt * per_tile - 1) / (nt * per_tile);
        e = launch(kernel, dim3(static_cast<unsigned>((tiles + rt - 1) / rt), static_cast<unsigned>(std::min<long long>(blocks, 65535))), dim3(32 * kW4Warps),
                   static_cast<size_t>(kW4Warps) * rt * nt * 128 * 4, 1, st, p);
    } else {
        const long long blocks = (a.rows + kW4AnyTokens - 1) / kW4AnyTokens;
        e = launch(linear_w4_any_kernel, dim3((a.out_features + 7) / 8, static_cast<unsigned>(std::min<long long>(blocks, 65535))), dim3(256), 0, 1, st, p);
    }
    return e == cudaSuccess ? PTQ8_OK : cuda_fail(o, "linear_w4", e);
}

}  // namespace

namespace ptq8 {

cudaError_t w4_attributes() { return cudaSuccess; }

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
