// Token operators: host side of the 4-bit cache (ptq8_cache_write, ptq8_cache_read, ptq8_cache_attention) and its
// extern "C" boundary.

#include <algorithm>
#include <cmath>

#include "ptq8_attention_tc.cuh"
#include "ptq8_ops.cuh"

using namespace ptq8;

// what the Python mirror packs
static_assert(sizeof(ptq8_cache) == 160 && sizeof(ptq8_cache_rows_args) == 224 && sizeof(ptq8_cache_attention_args) == 248, "argument structs");

namespace {

int check_cache(ptq8_ops* o, const ptq8_cache& c, long long tokens, const char* w) {
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256)
        return fail(o, PTQ8_ERR_INVALID, "%s: head_dim %d (64, 128 or 256)", w, c.head_dim);
    if (c.kv_heads <= 0 || c.kv_heads > 1024) return fail(o, PTQ8_ERR_INVALID, "%s: kv_heads %d (1 to 1024)", w, c.kv_heads);
    if (c.page < 16 || c.page > 4096 || (c.page & (c.page - 1)))
        return fail(o, PTQ8_ERR_INVALID, "%s: page %d (a power of two from 16 to 4096)", w, c.page);
    if (c.pages < 0 || c.pages > 0x7FFFFFFFLL) return fail(o, PTQ8_ERR_INVALID, "%s: pages %lld", w, c.pages);
    if (c.sequences < 0 || c.sequences > PTQ8_MAX_SEQUENCES)
        return fail(o, PTQ8_ERR_INVALID, "%s: sequences %d (up to %d)", w, c.sequences, PTQ8_MAX_SEQUENCES);
    if (c.table_width < 0 || static_cast<long long>(c.table_width) * c.page > 0x7FFFFF00LL)
        return fail(o, PTQ8_ERR_INVALID, "%s: table_width %d of pages of %d", w, c.table_width, c.page);
    if (c.table_pitch < c.table_width && c.sequences > 1)
        return fail(o, PTQ8_ERR_INVALID, "%s: table_pitch %lld < table_width %d", w, c.table_pitch, c.table_width);
    if (tokens < 0 || tokens > 0x7FFFFFFFLL / (2LL * c.kv_heads)) return fail(o, PTQ8_ERR_INVALID, "%s: tokens %lld", w, tokens);
    if (!c.starts && tokens != c.sequences)
        return fail(o, PTQ8_ERR_INVALID, "%s: tokens %lld without starts, but %d sequences", w, tokens, c.sequences);
    const long long codes = static_cast<long long>(c.page) * c.head_dim / 2, pairs = c.page * 4LL;
    const struct {
        const void* at;
        long long page, head, bytes;
        const char* name;
    } parts[] = {{c.k, c.k_page, c.k_head, codes, "k"}, {c.v, c.v_page, c.v_head, codes, "v"},
                 {c.k_scale, c.k_scale_page, c.k_scale_head, pairs, "k_scale"}, {c.v_scale, c.v_scale_page, c.v_scale_head, pairs, "v_scale"}};
    for (const auto& p : parts) {
        if (!aligned(p.at, 16) || (c.pages > 1 && p.page % 16) || (c.kv_heads > 1 && p.head % 16))
            return fail(o, PTQ8_ERR_INVALID, "%s: cache %s: address or strides are not multiples of 16 bytes", w, p.name);
        // pages and heads at any stride, in either order, but not over one another
        const bool heads_in = p.head >= p.bytes && p.page >= (c.kv_heads - 1) * p.head + p.bytes;
        const bool pages_in = p.page >= p.bytes && p.head >= (c.pages - 1) * p.page + p.bytes;
        if ((c.pages > 1 && c.kv_heads > 1 && !heads_in && !pages_in) || (c.pages > 1 && p.page < p.bytes) || (c.kv_heads > 1 && p.head < p.bytes))
            return fail(o, PTQ8_ERR_INVALID, "%s: cache %s: strides %lld, %lld: rows overlap", w, p.name, p.page, p.head);
    }
    if (tokens == 0 || c.sequences == 0) return PTQ8_OK;
    if (!c.lengths || (c.table_width && !c.table)) return fail(o, PTQ8_ERR_INVALID, "%s: null lengths or table", w);
    if (!aligned(c.lengths, 4) || !aligned(c.table, 4) || !aligned(c.starts, 4))
        return fail(o, PTQ8_ERR_INVALID, "%s: table, lengths or starts not aligned to 4 bytes", w);
    if (c.pages && (!c.k || !c.v || !c.k_scale || !c.v_scale)) return fail(o, PTQ8_ERR_INVALID, "%s: null cache", w);
    return PTQ8_OK;
}

CacheView view(const ptq8_cache& c, long long tokens) {
    CacheView v{};
    v.k = c.k;
    v.v = c.v;
    v.ks = reinterpret_cast<uint8_t*>(c.k_scale);
    v.vs = reinterpret_cast<uint8_t*>(c.v_scale);
    v.k_page = c.k_page, v.k_head = c.k_head, v.v_page = c.v_page, v.v_head = c.v_head;
    v.ks_page = c.k_scale_page, v.ks_head = c.k_scale_head, v.vs_page = c.v_scale_page, v.vs_head = c.v_scale_head;
    v.table = c.table;
    v.table_pitch = c.table_pitch;
    v.lengths = c.lengths;
    v.starts = c.starts;
    v.pages = c.pages;
    v.tokens = tokens;
    v.width = c.table_width;
    v.page = c.page;
    while ((1 << v.shift) < c.page) ++v.shift;
    v.heads = c.kv_heads;
    v.seqs = c.sequences;
    return v;
}

// Whether rows of floats [tokens][heads][dim] start at multiples of 16 bytes.
bool vectors(const void* p, long long token, long long head, int type) {
    const long long lanes = 16 / static_cast<long long>(type_size(type));
    return aligned(p, 16) && token % lanes == 0 && head % lanes == 0;
}

// Rows of floats that two (token, head) pairs share would be written twice.
bool apart(long long tokens, long long token, int heads, long long head, int dim) {
    const bool heads_in = head >= dim && token >= (heads - 1) * head + dim, tokens_in = token >= dim && head >= (tokens - 1) * token + dim;
    if (tokens > 1 && heads > 1) return heads_in || tokens_in;
    return (tokens <= 1 || token >= dim) && (heads <= 1 || head >= dim);
}

using CacheKernel = void (*)(CacheRowsParams);

template <typename T, int D, int U>
CacheKernel rows_kernel_of(bool write, bool vec) {
    return write ? (vec ? cache_write_kernel<T, D, true, U> : cache_write_kernel<T, D, false, U>) : (vec ? cache_read_kernel<T, D, true, U> : cache_read_kernel<T, D, false, U>);
}
template <typename T>
CacheKernel rows_kernel_of(int dim, bool write, bool vec, bool four) {
    if (four) return dim == 64 ? rows_kernel_of<T, 64, 4>(write, vec) : dim == 128 ? rows_kernel_of<T, 128, 4>(write, vec) : rows_kernel_of<T, 256, 4>(write, vec);
    return dim == 64 ? rows_kernel_of<T, 64, 1>(write, vec) : dim == 128 ? rows_kernel_of<T, 128, 1>(write, vec) : rows_kernel_of<T, 256, 1>(write, vec);
}

int rows_call(ptq8_ops* o, const ptq8_cache_rows_args* args, bool write, void* stream) {
    if (!o) return PTQ8_ERR_INVALID;
    if (!args) return fail(o, PTQ8_ERR_INVALID, "null arguments");
    const ptq8_cache_rows_args& a = *args;
    const char* w = write ? "cache_write" : "cache_read";
    if (a.type < PTQ8_F32 || a.type > PTQ8_BF16) return fail(o, PTQ8_ERR_INVALID, "%s: type %d", w, a.type);
    if (const int rc = check_cache(o, a.cache, a.tokens, w)) return rc;
    const ptq8_cache& c = a.cache;
    if (!write && (!apart(a.tokens, a.k_token, c.kv_heads, a.k_head, c.head_dim) || !apart(a.tokens, a.v_token, c.kv_heads, a.v_head, c.head_dim)))
        return fail(o, PTQ8_ERR_INVALID, "%s: rows of k or v overlap", w);
    if (a.k_token < 0 || a.k_head < 0 || a.v_token < 0 || a.v_head < 0) return fail(o, PTQ8_ERR_INVALID, "%s: negative strides", w);
    if (const int rc = ready(o)) return rc;
    if (a.tokens == 0 || c.sequences == 0) return PTQ8_OK;
    if (!a.k || !a.v) return fail(o, PTQ8_ERR_INVALID, "%s: null pointer", w);
    if (!aligned(a.k, type_size(a.type)) || !aligned(a.v, type_size(a.type)))
        return fail(o, PTQ8_ERR_INVALID, "%s: k or v is not aligned to its element type", w);
    OnDevice on(o->device);
    if (on.rc != cudaSuccess) return cuda_fail(o, "cudaSetDevice", on.rc);
    // A warp has 32 / (head_dim / 8) rows of a token at a time.  While there are few, that is all it has; then four times that,
    // whose loads overlap (and, writing, whose lanes share the work on four rows' steps): 18 k tokens written and read back 80 us, row by row 92.
    const long long steps = (2 * c.kv_heads * (c.head_dim / 8) + 31) / 32;
    const bool four = steps >= 4 && a.tokens * steps > 64LL * o->sms;
    const long long run = !four ? 1 : (steps + std::max<long long>(1, 64LL * o->sms / a.tokens) * 4 - 1) / (std::max<long long>(1, 64LL * o->sms / a.tokens) * 4) * 4;
    const long long parts = (steps + run - 1) / run;
    const CacheRowsParams p{view(c, a.tokens), a.k, a.v, a.k_token, a.k_head, a.v_token, a.v_head, static_cast<int>(parts), static_cast<int>(run)};
    const bool vec = vectors(a.k, a.k_token, a.k_head, a.type) && vectors(a.v, a.v_token, a.v_head, a.type);
    const CacheKernel kernel = a.type == PTQ8_F32   ? rows_kernel_of<float>(c.head_dim, write, vec, four)
                               : a.type == PTQ8_F16 ? rows_kernel_of<__half>(c.head_dim, write, vec, four)
                                                    : rows_kernel_of<__nv_bfloat16>(c.head_dim, write, vec, four);
    const long long blocks = (a.tokens * parts + kCacheThreads / 32 - 1) / (kCacheThreads / 32);
    const size_t smem = c.starts ? (c.sequences + 1) * sizeof(int) : 0;
    const cudaError_t e = launch(kernel, dim3(static_cast<unsigned>(std::min<long long>(blocks, 8LL * o->sms))), dim3(kCacheThreads), smem, 1,
                                 static_cast<cudaStream_t>(stream), p);
    return e == cudaSuccess ? PTQ8_OK : cuda_fail(o, w, e);
}

using AttKernel = void (*)(AttParams);

struct AttVariant {
    int dim, rows;   // query rows of a tile
    AttKernel kernel;
    int per_sm, smem;   // of PTQ8_MAX_SEQUENCES
    int (*smem_of)(int seqs);
    int threads;
    long long work;   // query rows x tokens that a table has room for, from which on it is taken
};

template <int D, int NT, int RW>
AttVariant att_variant() {
    using Sh = AttShape<D, NT, RW>;
    return {D, Sh::R, cache_attention_kernel<D, NT, RW>, Sh::kPerSm, Sh::smem(PTQ8_MAX_SEQUENCES), Sh::smem, kAttThreads, 0};
}

template <int D>
AttVariant att_tiles_variant() {
    using Sh = TcAttShape<D>;
    return {D, kTcRows, cache_attention_tiles_kernel<D>, 1, Sh::smem(PTQ8_MAX_SEQUENCES), Sh::smem, kTcThreads, D == 128 ? 1 << 24 : 1 << 25};
}

const AttVariant kAttVariants[] = {
    att_variant<64, 1, 1>(),  att_variant<64, 2, 1>(),  att_variant<64, 2, 2>(),  att_variant<64, 2, 4>(), att_tiles_variant<64>(),
    att_variant<128, 1, 1>(), att_variant<128, 2, 1>(), att_variant<128, 2, 2>(), att_variant<128, 2, 4>(), att_tiles_variant<128>(),
    att_variant<256, 1, 1>(), att_variant<256, 1, 2>(), att_variant<256, 1, 4>(),
};

using AttJoin = void (*)(AttParams, int);
constexpr int kAttJoinSmem = 60 * 1024;   // none of it is used (see cache_attributes)
const AttJoin kAttJoins[3][2] = {{cache_attention_join_kernel<64, 1>, cache_attention_join_kernel<64, kAttJoinWide>},
                                 {cache_attention_join_kernel<128, 1>, cache_attention_join_kernel<128, kAttJoinWide>},
                                 {cache_attention_join_kernel<256, 1>, cache_attention_join_kernel<256, kAttJoinWide>}};

// The smallest tile that takes a sequence's query rows of a key head on average, or the largest.  Tiles of 256 rows while there is enough
// to do: their blocks take some us more to begin and to join.  us with them and without, 8 key heads, bf16, sequences x
// query rows of a key head x positions:
//              1 x 512 x 500   1 x 384 x 4000   1 x 512 x 4000   1 x 1024 x 4000   8 x 68 x 4000   8 x 136 x 4000   8 x 512 x 4000
//   D = 64     26   19         37   34          41   40          57   63           65   62         79   86          152   201
//   D = 128    34   26         47   48          51   59          75   98           81   97         99   137         183   332
// (The last but four are 16.5 M rows x tokens, just below the limit of 128 dimensions: a limit that took them would take 1 x 384 x 4000 and
// wider tables of shorter sequences with them.)  The host knows only what the table has room for: a table much wider than its
// sequences are long takes tiles early.  It goes by the mean of the sequences: pieces beside many single tokens may stay on narrow tiles.
const AttVariant& att_choose(const ptq8_cache_attention_args& a, long long room) {
    const long long rows = (a.tokens * (a.heads / a.cache.kv_heads) + a.cache.sequences - 1) / a.cache.sequences;
    const AttVariant* best = nullptr;
    for (const AttVariant& v : kAttVariants)
        if (v.dim == a.cache.head_dim && (!best || best->rows < rows) && a.tokens * a.heads * room >= v.work) best = &v;
    return *best;
}

// Row tiles at most: each sequence's last may be partly filled.
long long att_items(const ptq8_cache_attention_args& a, const AttVariant& v) {
    const long long per = a.heads / a.cache.kv_heads, n = std::min<long long>(a.cache.sequences, a.tokens);
    const long long tiles = a.cache.starts ? a.tokens * per / v.rows + n : n * ((per + v.rows - 1) / v.rows);
    return tiles * a.cache.kv_heads;
}

// Many row tiles keep the SMs busy one CTA each; fewer are cut into equal shares.  (So are more units than an int counts.)
bool att_by_item(const ptq8_ops* o, const ptq8_cache_attention_args& a, const AttVariant& v, int table_width) {
    const long long most = static_cast<long long>(table_width) * a.cache.page / kAttTile + 1 + kAttOver, items = att_items(a, v);
    if (items > kAttUnits / most) return true;
    return a.cache.starts && a.tokens * (a.heads / a.cache.kv_heads) / v.rows * a.cache.kv_heads >= 8LL * o->sms * v.per_sm;
}

int check_attention(ptq8_ops* o, const ptq8_cache_attention_args& a) {
    const char* w = "cache_attention";
    if (a.type != PTQ8_F16 && a.type != PTQ8_BF16) return fail(o, PTQ8_ERR_INVALID, "%s: type %d (f16 or bf16)", w, a.type);
    if (const int rc = check_cache(o, a.cache, a.tokens, w)) return rc;
    if (a.heads <= 0 || a.heads > 4096 || a.heads % a.cache.kv_heads)
        return fail(o, PTQ8_ERR_INVALID, "%s: heads %d for %d key heads", w, a.heads, a.cache.kv_heads);
    if (a.tokens > 0x7FFFFF00LL / a.heads) return fail(o, PTQ8_ERR_INVALID, "%s: tokens %lld", w, a.tokens);
    if (!std::isfinite(a.scale)) return fail(o, PTQ8_ERR_INVALID, "%s: scale %g", w, static_cast<double>(a.scale));
    if (a.q_token < 0 || a.q_head < 0) return fail(o, PTQ8_ERR_INVALID, "%s: negative strides", w);
    if (!apart(a.tokens, a.out_token, a.heads, a.out_head, a.cache.head_dim)) return fail(o, PTQ8_ERR_INVALID, "%s: rows of out overlap", w);
    return PTQ8_OK;
}

long long workspace_of(const ptq8_ops* o, const ptq8_cache_attention_args& a) {
    if (a.tokens == 0 || a.cache.sequences == 0) return 0;
    long long need = 0;
    for (const long long room : {0LL, 1LL << 31}) {   // whatever the table's width
        const AttVariant& v = att_choose(a, room);
        const long long n = static_cast<long long>(o->sms) * v.per_sm;
        if (!att_by_item(o, a, v, 0)) need = std::max(need, 2 * n * v.rows * (v.dim + 2) * 4 + n * static_cast<long long>(sizeof(AttDesc)));
    }
    return need;
}

int attention_call(ptq8_ops* o, const ptq8_cache_attention_args& a, cudaStream_t st) {
    const AttVariant& v = att_choose(a, static_cast<long long>(a.cache.table_width) * a.cache.page);
    AttParams p{};
    p.c = view(a.cache, a.tokens);
    p.q = a.q;
    p.out = a.out;
    p.q_token = a.q_token, p.q_head = a.q_head, p.o_token = a.out_token, p.o_head = a.out_head;
    int power = 0;
    const double fraction = std::frexp(a.scale * 1.4426950408889634, &power);
    const int held = std::min(std::max(power, -126), 1);   // (with what takes the largest queries' products back, a power of two that is a float)
    p.key_scale = fraction == 0.0 ? std::ldexp(1.0f, -kAttKeys) : static_cast<float>(std::ldexp(fraction, power - held - kAttKeys));
    p.score_scale = fraction == 0.0 ? 0.0f : std::ldexp(1.0f, held);
    p.per = a.heads / a.cache.kv_heads;
    p.by_item = att_by_item(o, a, v, a.cache.table_width);
    p.type = a.type;
    p.vec_q = vectors(a.q, a.q_token, a.q_head, a.type);
    p.vec_o = vectors(a.out, a.out_token, a.out_head, a.type);
    p.wait_limit = o->wait_limit;
    p.err = o->error_dev;
    p.stall = o->stall;
    const long long items = att_items(a, v);
    long long n = static_cast<long long>(o->sms) * v.per_sm;
    if (p.by_item) {
        n = items;
    } else {
        p.part = static_cast<float*>(a.workspace);
        p.stat = p.part + 2 * n * v.rows * v.dim;
        p.desc = reinterpret_cast<AttDesc*>(p.stat + 2 * n * v.rows * 2);
        p.listed = !a.cache.starts && items <= n;
    }
    cudaError_t e = launch(v.kernel, dim3(static_cast<unsigned>(n)), dim3(v.threads), v.smem_of(a.cache.sequences), 1, st, p);
    if (e == cudaSuccess && !p.by_item) {
        // few row tiles have many parts each: eight warps a row; else a warp a row
        const bool wide = p.listed && 4 * items <= n;
        const int rows = p.listed ? std::min(v.rows, p.per) : v.rows;
        e = launch(kAttJoins[v.dim == 64 ? 0 : v.dim == 128 ? 1 : 2][wide], dim3(static_cast<unsigned>(p.listed ? items : n), wide ? rows : (rows + 7) / 8), dim3(256), kAttJoinSmem, 1, st, p, v.rows);
    }
    return e == cudaSuccess ? PTQ8_OK : cuda_fail(o, "cache_attention", e);
}

}  // namespace

namespace ptq8 {

static cudaError_t most_shared(const void* kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
}

cudaError_t cache_attributes() {
    for (const AttVariant& v : kAttVariants) {
        const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(v.kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem);
        if (e != cudaSuccess) return e;
    }
    // An SM divides its memory anew between L1 and shared memory only when it is empty.  The kernels that run beside attention's
    // under programmatic launch therefore ask for its division (one token over 2000 positions: 8.3 us a call instead of 8.8).
    for (const auto& pair : kAttJoins)
        for (const AttJoin join : pair)
        {
            if (const cudaError_t e = most_shared(reinterpret_cast<const void*>(join)); e != cudaSuccess) return e;
            if (const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(join), cudaFuncAttributeMaxDynamicSharedMemorySize, kAttJoinSmem); e != cudaSuccess) return e;
        }
    for (const int dim : {64, 128, 256})
        for (const bool write : {false, true})
            for (const int i : {0, 1, 2, 3})
                for (const CacheKernel k : {rows_kernel_of<float>(dim, write, i & 1, i & 2), rows_kernel_of<__half>(dim, write, i & 1, i & 2), rows_kernel_of<__nv_bfloat16>(dim, write, i & 1, i & 2)})
                    if (const cudaError_t e = most_shared(reinterpret_cast<const void*>(k)); e != cudaSuccess) return e;
    return cudaSuccess;
}

}  // namespace ptq8

extern "C" {

int ptq8_cache_write(ptq8_ops* o, const ptq8_cache_rows_args* a, void* stream) { return rows_call(o, a, true, stream); }

int ptq8_cache_read(ptq8_ops* o, const ptq8_cache_rows_args* a, void* stream) { return rows_call(o, a, false, stream); }

long long ptq8_cache_attention_workspace(ptq8_ops* o, const ptq8_cache_attention_args* a) {
    if (!o) return -1;
    if (!a) return fail(o, -1, "null arguments");
    ptq8_cache_attention_args shape = *a;   // the tensors do not count
    ptq8_cache& c = shape.cache;
    c.k = c.v = nullptr;
    c.k_scale = c.v_scale = nullptr;
    c.pages = 0;
    c.table_width = 0;
    static const int none = 0;
    c.lengths = &none;
    if (c.starts) c.starts = &none;
    if (check_attention(o, shape)) return -1;
    return workspace_of(o, shape);
}

int ptq8_cache_attention(ptq8_ops* o, const ptq8_cache_attention_args* args, void* stream) {
    if (!o) return PTQ8_ERR_INVALID;
    if (!args) return fail(o, PTQ8_ERR_INVALID, "null arguments");
    const ptq8_cache_attention_args& a = *args;
    if (const int rc = check_attention(o, a)) return rc;
    if (const int rc = ready(o)) return rc;
    if (a.tokens == 0 || a.cache.sequences == 0) return PTQ8_OK;
    const char* w = "cache_attention";
    if (!a.q || !a.out) return fail(o, PTQ8_ERR_INVALID, "%s: null pointer", w);
    if (!aligned(a.q, 2) || !aligned(a.out, 2)) return fail(o, PTQ8_ERR_INVALID, "%s: q or out is not aligned to its element type", w);
    const long long need = workspace_of(o, a);
    if (a.workspace_bytes < need || (need && !a.workspace))
        return fail(o, PTQ8_ERR_INVALID, "%s: workspace of %lld bytes, %lld are wanted", w, a.workspace_bytes, need);
    if (need && !aligned(a.workspace, 16)) return fail(o, PTQ8_ERR_INVALID, "%s: workspace not aligned to 16 bytes", w);
    OnDevice on(o->device);
    if (on.rc != cudaSuccess) return cuda_fail(o, "cudaSetDevice", on.rc);
    return attention_call(o, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
