// C entries of the edge attention (include/dedf.h: dedf_edge_segments, dedf_edge_attention, dedf_edge_attention_backward)
#include "../../include/dedf.h"
#include "dedf_attn.h"
#include <algorithm>
#include <cmath>

using namespace dedf::attn;

// the launches for one element type: each type is a compilation of its own (DEDF_ELEMENT 0, 1, 2), the entries another (none)
namespace dedf {
namespace attn {

struct Plan { Args a; int mode, nv, ga; size_t record, lds_forward, lds_backward; int blocks; };

struct Forward {
    const Plan& p; void* out; float* out32; double* norm; int64_t* rng_used; void* records; hipStream_t st;
    template <class T, int MODE, int NV, int GA> int run() {
        if (p.lds_forward > 65536 && hipFuncSetAttribute((const void*)k_attn_forward<T, MODE, NV, GA>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds_forward) != hipSuccess) return DEDF_ERR_RUNTIME;
        const int empty_blocks = (int)(((int64_t)p.a.n_dst + 64 * kWaves - 1) / (64 * kWaves));
        hipLaunchKernelGGL((k_attn_forward<T, MODE, NV, GA>), dim3(p.blocks + empty_blocks), dim3(256), p.lds_forward, st, p.a, (T*)out, out32, norm, records, rng_used);
        if (p.a.n_waves > 1) hipLaunchKernelGGL((k_attn_merge<T, MODE, NV>), dim3((p.a.n_waves - 1 + merge_waves<NV>() - 1) / merge_waves<NV>()), dim3(1024 / NV), 0, st, p.a, (T*)out, out32, norm, (const void*)records);
        return hipGetLastError() == hipSuccess ? DEDF_OK : DEDF_ERR_RUNTIME;
    }
};
struct Backward {
    const Plan& p; BackArgs b; const float* out32; float* delta; float* d_alpha_dot; float* d_table; hipStream_t st;
    template <class T, int MODE, int NV, int GA> int run() {
        if (p.lds_backward > 65536 && hipFuncSetAttribute((const void*)k_attn_backward<T, MODE, NV, GA>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds_backward) != hipSuccess) return DEDF_ERR_RUNTIME;
        const Args& a = p.a;
        const int64_t pairs = (int64_t)a.n_dst * a.heads;          // (a launch has fewer than 2^32 threads: 16 a pair pass that at 2^28 pairs)
        hipLaunchKernelGGL((k_attn_delta<T>), dim3((unsigned)std::min<int64_t>((pairs + 15) / 16, 1 << 23)), dim3(256), 0, st, pairs, a.d, (const T*)b.grad, out32, delta);
        hipLaunchKernelGGL((k_attn_backward<T, MODE, NV, GA>), dim3(p.blocks), dim3(256), p.lds_backward, st, a, b);
        if (b.param_rows) {
            const int n_w = a.heads * a.k, columns = n_w + a.heads * a.n_buckets;
            hipLaunchKernelGGL(k_column_sums, dim3((columns + 15) / 16), dim3(1024), 0, st, (const float*)b.param_rows, p.blocks, columns, d_alpha_dot, n_w, d_table);
        }
        return hipGetLastError() == hipSuccess ? DEDF_OK : DEDF_ERR_RUNTIME;
    }
};

template <class T, int MODE, class F> int by_width(int nv, int ga, F& f) {
    if constexpr (MODE == kHeads) if (ga == 2) return f.template run<T, MODE, 4, 2>();          // (aligned features have at most 64 quads)
    if (nv == 4) return f.template run<T, MODE, 4, 4>();
    if (nv == 2) return ga == 16 ? f.template run<T, MODE, 2, 16>() : ga == 8 ? f.template run<T, MODE, 2, 8>() : f.template run<T, MODE, 2, 4>();
    return ga == 16 ? f.template run<T, MODE, 1, 16>() : f.template run<T, MODE, 1, 8>();
}
template <class T, class F> int launch(int mode, int nv, int ga, F f) {
    if (mode != kElements) return mode == kAligned ? by_width<T, kAligned>(nv, ga, f) : by_width<T, kHeads>(nv, ga, f);
    if (ga == 2) return f.template run<T, kElements, 4, 2>();          // (at most 16 value quads)
    return ga == 16 ? f.template run<T, kElements, 1, 16>() : ga == 8 ? f.template run<T, kElements, 1, 8>() : f.template run<T, kElements, 2, 4>();
}

#define DEDF_LAUNCHES(T, PREFIX) PREFIX template int launch<T, Forward>(int, int, int, Forward); PREFIX template int launch<T, Backward>(int, int, int, Backward);
#ifndef DEDF_ELEMENT
DEDF_LAUNCHES(float, extern) DEDF_LAUNCHES(_Float16, extern) DEDF_LAUNCHES(__bf16, extern)
#elif DEDF_ELEMENT == 0
DEDF_LAUNCHES(float, )
#elif DEDF_ELEMENT == 1
DEDF_LAUNCHES(_Float16, )
#else
DEDF_LAUNCHES(__bf16, )
#endif

}  // namespace attn
}  // namespace dedf

#ifndef DEDF_ELEMENT
namespace {

constexpr int kSimds = 1024;          // 256 CUs of 4
constexpr size_t kMostLds = 160 * 1024;

size_t element(int type) { return type == DEDF_F32 ? 4 : 2; }
bool whole_quads(const void* p, int64_t stride, int type) {
    const size_t quad = 4 * element(type);
    return (reinterpret_cast<uintptr_t>(p) % quad) == 0 && stride % 4 == 0;
}

// `tensors`: the call's other tensors of (edges or rows, heads, k or d) in the element type
int make_plan(const dedf_edge_attn* x, bool backward, Plan& p, std::initializer_list<const void*> tensors) {
    if (!x || x->n_edges < 0 || x->n_dst < 0 || x->heads < 1 || x->k < 1 || x->d < 1 || x->n_buckets < 0) return DEDF_ERR_INVALID;
    if (x->type != DEDF_F32 && x->type != DEDF_F16 && x->type != DEDF_BF16) return DEDF_ERR_UNSUPPORTED;
    if (x->n_edges >= (int64_t)1 << 31 || x->heads > 16 || x->k > 256 || x->d > 1024 || x->heads * x->k > 256 || row_quads(x->heads, x->d) > 256) return DEDF_ERR_UNSUPPORTED;
    if (x->n_buckets > 1024 || x->n_buckets * x->heads > 2048) return DEDF_ERR_UNSUPPORTED;
    if (x->n_edges > 0 && (!x->alpha || !x->value || !x->alpha_dot || !x->dst)) return DEDF_ERR_INVALID;
    if (x->n_dst > 0 && !x->rowptr) return DEDF_ERR_INVALID;
    if (x->n_dst == 0 && x->n_edges > 0) return DEDF_ERR_INVALID;
    if (x->n_buckets > 0 && (!x->bias_table || (x->n_edges > 0 && !x->edge_length) || (x->n_buckets > 1 && !x->bias_boundaries))) return DEDF_ERR_INVALID;
    if (!(x->dropout >= 0.0 && x->dropout < 1.0) || (x->dropout > 0.0 && !x->rng)) return DEDF_ERR_INVALID;
    if (x->alpha_stride < 0 || x->value_stride < 0) return DEDF_ERR_INVALID;
    Args& a = p.a;
    a = Args{};
    a.n_edges = x->n_edges; a.n_dst = x->n_dst; a.heads = x->heads; a.k = x->k; a.d = x->d;
    a.a = x->alpha; a.v = x->value; a.w = x->alpha_dot; a.a_stride = x->alpha_stride; a.v_stride = x->value_stride;
    a.dst = x->dst; a.rowptr = x->rowptr; a.logits = x->edge_logits; a.length = x->edge_length; a.bounds = x->bias_boundaries; a.table = x->bias_table;
    a.n_buckets = x->n_buckets;
    a.threshold = (uint32_t)std::floor(x->dropout * 4294967296.0);
    a.keep_scale = (float)(1.0 / (1.0 - x->dropout)); a.rng = x->rng;
    bool whole = a.k % 4 == 0 && a.d % 4 == 0 && whole_quads(a.a, a.a_stride, x->type) && whole_quads(a.v, a.v_stride, x->type);
    for (const void* t : tensors) whole = whole && whole_quads(t, 0, x->type);
    p.mode = whole ? kAligned : a.d >= 4 ? kHeads : kElements;
    const int qa = row_quads(a.heads, a.k), qv = row_quads(a.heads, a.d);          // (qa <= 75: 15 heads of 17)
    // as many edges a group as four feature quads a lane hold: with 8 heads of 3 + 33 channels (400 000 float32 edges, training) groups of 16 0.40 ms, of 8 0.43
    p.ga = qa > 64 ? 2 : qv > 128 || qa > 32 ? 4 : qa > 16 ? 8 : 16;
    p.nv = qv > 128 || p.ga == 2 ? 4 : qv > 64 || p.ga == 4 ? 2 : 1;
    const int bytes = (int)element(x->type), most = kSimds * (backward ? backward_waves(p.nv, bytes) : forward_waves(p.nv, bytes));
    const int64_t even = (a.n_edges + most - 1) / most;
    a.range = (int)std::max<int64_t>(kBatch, (even + kBatch - 1) / kBatch * kBatch);
    a.n_waves = (int)((a.n_edges + a.range - 1) / a.range);
    p.blocks = (a.n_waves + kWaves - 1) / kWaves;
    p.record = (size_t)(p.nv * 28 + 15) / 16 * 16 * 64 * 2;
    static_assert(sizeof(Record<1>) == 32 && sizeof(Record<2>) == 64 && sizeof(Record<4>) == 112, "records are as large as computed here");
    const size_t own = Wave<float, kAligned, 1, 16>::wave_bytes(a.heads);          // (whatever the type, mode and width)
    const int BH = a.n_buckets * a.heads;
    const size_t shared = Wave<float, kAligned, 1, 16>::shared_bytes(qa, a.heads, a.n_buckets);
    p.lds_forward = shared + kWaves * (own + (size_t)kBatch * a.heads * 8);
    p.lds_backward = shared + kWaves * ((own + (size_t)kBatch * a.heads * 4 + (size_t)((BH + 1) & ~1) * 4 + 15) & ~(size_t)15);
    if (p.lds_forward > kMostLds || p.lds_backward > kMostLds) return DEDF_ERR_UNSUPPORTED;
    return DEDF_OK;
}
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }
size_t forward_bytes(const Plan& p) { return (size_t)p.blocks * kWaves * p.record; }
template <class F> int by_shape(int type, const Plan& p, F f) {
    return type == DEDF_F32 ? launch<float>(p.mode, p.nv, p.ga, f) : type == DEDF_F16 ? launch<_Float16>(p.mode, p.nv, p.ga, f) : launch<__bf16>(p.mode, p.nv, p.ga, f);
}
size_t backward_bytes(const Plan& p) {
    return up16((size_t)p.a.n_dst * p.a.heads * 4) + (size_t)p.blocks * (p.a.heads * (p.a.k + p.a.n_buckets)) * 4;
}

}  // namespace

extern "C" {

int dedf_edge_segments(const int64_t* edge_dst, int64_t n_edges, int n_dst, int32_t* dst, int32_t* rowptr, int32_t* bad, void* stream) {
    if (n_edges < 0 || n_dst < 0 || !rowptr || !bad || (n_edges > 0 && (!edge_dst || !dst || n_dst == 0))) return DEDF_ERR_INVALID;
    if (n_edges >= (int64_t)1 << 31) return DEDF_ERR_UNSUPPORTED;
    const int64_t n = std::max<int64_t>(n_edges, (int64_t)n_dst + 1);
    hipLaunchKernelGGL(k_edge_segments, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, static_cast<hipStream_t>(stream), edge_dst, n_edges, n_dst, dst, rowptr, bad);
    return hipGetLastError() == hipSuccess ? DEDF_OK : DEDF_ERR_RUNTIME;
}

size_t dedf_edge_attention_scratch_bytes(const dedf_edge_attn* x, int backward) {
    Plan p;
    if (make_plan(x, backward != 0, p, {}) != DEDF_OK) return 0;
    if (backward) return backward_bytes(p);
    return forward_bytes(p);
}

int dedf_edge_attention(const dedf_edge_attn* x, void* out, float* out_f, double* norm, int64_t* rng_used, void* scratch, size_t scratch_bytes, void* stream) {
    Plan p;
    const int rc = make_plan(x, false, p, {out, out_f});
    if (rc != DEDF_OK) return rc;
    if (p.a.n_dst == 0) return DEDF_OK;
    if (!out || scratch_bytes < forward_bytes(p) || (forward_bytes(p) > 0 && !scratch) || (reinterpret_cast<uintptr_t>(scratch) & 15)) return DEDF_ERR_INVALID;
    Forward f{p, out, out_f, norm, rng_used, scratch, static_cast<hipStream_t>(stream)};
    return by_shape(x->type, p, f);
}

int dedf_edge_attention_backward(const dedf_edge_attn* x, const double* norm, const float* out_f, const void* grad_out, void* d_alpha, void* d_value,
                                 float* d_alpha_dot, float* d_edge_logits, float* d_bias_table, void* scratch, size_t scratch_bytes, void* stream) {
    Plan p;
    const int rc = make_plan(x, true, p, {grad_out, d_alpha, d_value});
    if (rc != DEDF_OK) return rc;
    if (p.a.n_dst > 0 && (!norm || !out_f || !grad_out)) return DEDF_ERR_INVALID;
    if (scratch_bytes < backward_bytes(p) || (backward_bytes(p) > 0 && !scratch) || (reinterpret_cast<uintptr_t>(scratch) & 15)) return DEDF_ERR_INVALID;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int n_w = p.a.heads * p.a.k, columns = n_w + p.a.heads * p.a.n_buckets;
    if (p.a.n_edges == 0) {          // no edge: the parameters' gradients are zero (a sum over no rows)
        hipLaunchKernelGGL(k_column_sums, dim3((columns + 15) / 16), dim3(1024), 0, st, (const float*)nullptr, 0, columns, d_alpha_dot, n_w, d_bias_table);
        return hipGetLastError() == hipSuccess ? DEDF_OK : DEDF_ERR_RUNTIME;
    }
    BackArgs b{norm, (const float*)scratch, grad_out, d_alpha, d_value, d_edge_logits,
               d_alpha_dot || d_bias_table ? (float*)((char*)scratch + up16((size_t)p.a.n_dst * p.a.heads * 4)) : nullptr};
    Backward f{p, b, out_f, (float*)scratch, d_alpha_dot, d_bias_table, st};
    return by_shape(x->type, p, f);
}

}  // extern "C"
#endif
