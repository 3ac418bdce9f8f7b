// C entries of the row operators (include/dedf.h: dedf_norm_gate_residual, dedf_norm_gate_residual_backward, dedf_channel_dropout)
#include "../../include/dedf.h"
#include "dedf_rows.h"
#include <algorithm>
#include <cmath>

using namespace dedf::rows;

namespace {

constexpr int kMostWidth = 2048;
constexpr int kCus = 256, kDropoutBlocks = 2048;
int quads(int width) { return width <= 256 || (width > 512 && width <= 1024) ? 1 : 2; }          // of a lane, as by_width
int norm_blocks(bool backward, int width) { return kCus * (backward ? backward_waves(quads(width)) : forward_waves(quads(width))); }          // (a workgroup has a wave on each SIMD)

size_t element(int type) { return type == DEDF_F32 ? 4 : 2; }
bool shared_rows(int width) { return width > 512; }          // a row has the whole workgroup

template <class T, bool FAST, class F> int by_width(int width, F& f) {
    return width <= 256 ? f.template run<T, 1, FAST, 1>() : width <= 512 ? f.template run<T, 2, FAST, 1>()
         : width <= 1024 ? f.template run<T, 1, FAST, 4>() : f.template run<T, 2, FAST, 4>();
}

// `whole`: blocks start on whole quads
int make_shape(int n_blocks, const int* mul, const int* degree, Shape& s, bool& whole) {
    if (n_blocks < 1 || !mul || !degree) return DEDF_ERR_INVALID;
    if (n_blocks > kMostBlocks) return DEDF_ERR_UNSUPPORTED;
    s = Shape{};
    s.n_blocks = n_blocks;
    whole = true;
    int64_t width = 0, channels = 0;
    for (int b = 0; b < kMostBlocks; ++b) {
        const bool there = b < n_blocks;
        if (there && (mul[b] < 1 || degree[b] < 0 || (b > 0 && degree[b] <= degree[b - 1]))) return DEDF_ERR_INVALID;
        if (there && (mul[b] > kMostWidth || degree[b] > 7)) return DEDF_ERR_UNSUPPORTED;
        const int m = there ? mul[b] : 0, d = there ? 2 * degree[b] + 1 : 1;
        s.start[b] = (int)width; s.first[b] = (int)channels; s.d[b] = d;
        s.divide[b] = (65536 + d - 1) / d;          // (exact for x d < 65536: x < 2048, d <= 15)
        s.inverse[b] = there ? 1.0f / (float)(m * d) : 0.0f;
        width += (int64_t)m * d; channels += m;
        s.start[b + 1] = (int)width;
        whole = whole && width % 4 == 0;
    }
    if (width > kMostWidth) return DEDF_ERR_UNSUPPORTED;
    s.width = (int)width; s.channels = (int)channels; s.scalars = degree[0] == 0 ? mul[0] : 0;
    return DEDF_OK;
}

// groups of rows cut into slices until there is a unit for every wave
void cut(Args& a, int waves) {
    const int64_t rows = a.n_rows / a.groups;          // (sums of two counts pass 32 bits)
    a.slices = (int)std::max<int64_t>(1, std::min<int64_t>(rows, waves / a.groups));
    a.slice_rows = (int)((rows + a.slices - 1) / a.slices);
    a.slices = (int)((rows + a.slice_rows - 1) / a.slice_rows);
}
int grid(const Args& a, int most) {
    const int teams = shared_rows(a.s.width) ? 1 : kWaves;
    return (int)std::min<int64_t>(most, ((int64_t)a.groups * a.slices + teams - 1) / teams);
}

int make_args(const dedf_norm* x, bool backward, Args& a, bool& fast) {
    if (!x || x->n_rows < 0) return DEDF_ERR_INVALID;
    if (x->type != DEDF_F32 && x->type != DEDF_F16 && x->type != DEDF_BF16) return DEDF_ERR_UNSUPPORTED;
    a = Args{};
    const int rc = make_shape(x->n_blocks, x->mul, x->degree, a.s, fast);
    if (rc != DEDF_OK) return rc;
    const int groups = x->gate ? x->groups : 1;
    if (x->n_rows > 0 && (!x->x || groups < 1 || groups > x->n_rows || x->n_rows % groups != 0)) return DEDF_ERR_INVALID;
    if (x->n_rows > 0 && !x->y && (x->gate || x->post_weight || x->dropout != 0.0)) return DEDF_ERR_INVALID;
    if (a.s.scalars > 0 && ((x->post_weight && !x->post_bias) || (x->next_weight && !x->next_bias))) return DEDF_ERR_INVALID;
    if (!(x->dropout >= 0.0 && x->dropout < 1.0) || (x->dropout > 0.0 && !x->rng) || !(x->eps >= 1e-30f)) return DEDF_ERR_INVALID;
    a.n_rows = x->n_rows; a.groups = std::max(1, groups);
    a.x = x->x; a.y = x->y; a.gate = x->gate; a.gate_f32 = x->type == DEDF_F32 || x->gate_f;
    a.post_w = x->post_weight; a.post_b = x->post_bias; a.next_w = x->next_weight; a.next_b = x->next_bias;
    a.scale = x->scale; a.eps = x->eps;
    a.threshold = (uint32_t)std::floor(x->dropout * 4294967296.0); a.keep_scale = (float)(1.0 / (1.0 - x->dropout)); a.rng = x->rng;
    if (a.n_rows > 0) cut(a, norm_blocks(backward, a.s.width) * (shared_rows(a.s.width) ? 1 : kWaves));
    return DEDF_OK;
}
bool on_quads(int type, std::initializer_list<const void*> all) {
    for (const void* p : all) if (reinterpret_cast<uintptr_t>(p) % (4 * element(type)) != 0) return false;
    return true;
}

size_t lds_bytes(const Args& a) { return shared_rows(a.s.width) ? Row<float, 1, true, 4>::team_bytes(a.s) : kWaves * Row<float, 1, true, 1>::team_bytes(a.s); }

}  // namespace

// the launches of one operator for one element type: each type is a compilation of its own (DEDF_ELEMENT 0, 1, 2), the entries another (none)
namespace dedf {
namespace rows {

struct NormForward {
    const Args& a; hipStream_t st;
    template <class T, int NQ, bool FAST, int WPR> int run() {
        hipLaunchKernelGGL((k_norm_forward<T, NQ, FAST, WPR>), dim3(grid(a, norm_blocks(false, a.s.width))), dim3(256), lds_bytes(a), st, a);
        return hipGetLastError() == hipSuccess ? DEDF_OK : DEDF_ERR_RUNTIME;
    }
};
struct NormBackward {
    const Args& a; hipStream_t st; float* post_w; float* post_b; float* next_w; float* next_b;
    template <class T, int NQ, bool FAST, int WPR> int run() {
        const int blocks = grid(a, norm_blocks(true, a.s.width)), C = a.s.channels;
        hipLaunchKernelGGL((k_norm_backward<T, NQ, FAST, WPR>), dim3(blocks), dim3(256), lds_bytes(a), st, a);
        const int narrow = a.gate_f32 ? 0 : 1;
        if (a.param_rows)
            hipLaunchKernelGGL(k_row_sums<T>, dim3((a.n_params * C + 15) / 16), dim3(1024), 0, st, (const float*)a.param_rows, blocks, a.n_params * C, C,
                               Outputs{{post_w, post_b, next_w, next_b, a.d_gate}, {C, a.s.scalars, C, a.s.scalars, C}, {0, 0, 0, 0, narrow}});
        if (a.gate_rows && a.slices <= 32) {          // (1 000 groups of 5 slices: 21 us with k_row_sums)
            const int64_t sums = (int64_t)a.groups * C;
            hipLaunchKernelGGL(k_few_rows<T>, dim3((unsigned)((sums + 255) / 256)), dim3(256), 0, st, (const float*)a.gate_rows, a.slices, C, sums, narrow ? (T*)a.d_gate : nullptr,
                               narrow ? nullptr : (float*)a.d_gate);
        } else if (a.gate_rows)
            hipLaunchKernelGGL(k_row_sums<T>, dim3((C + 15) / 16, a.groups), dim3(1024), 0, st, (const float*)a.gate_rows, a.slices, C, C, Outputs{{a.d_gate}, {C}, {narrow}});
        return hipGetLastError() == hipSuccess ? DEDF_OK : DEDF_ERR_RUNTIME;
    }
};
struct Dropout {
    const Args& a; hipStream_t st;
    template <class T, int NQ, bool FAST, int WPR> int run() {
        constexpr int teams = kWaves / WPR;
        Args b = a;
        const int64_t rows = a.n_rows;
        b.slice_rows = (int)((rows + kDropoutBlocks * teams - 1) / (kDropoutBlocks * teams));
        const int slices = (int)((rows + b.slice_rows - 1) / b.slice_rows);
        hipLaunchKernelGGL((k_dropout<T, NQ, FAST, WPR>), dim3((slices + teams - 1) / teams), dim3(256), lds_bytes(a), st, b);
        return hipGetLastError() == hipSuccess ? DEDF_OK : DEDF_ERR_RUNTIME;
    }
};
template <class T, class F> int launch(int width, bool fast, F f) { return fast ? by_width<T, true>(width, f) : by_width<T, false>(width, f); }

#define DEDF_LAUNCHES(T, PREFIX) \
    PREFIX template int launch<T, NormForward>(int, bool, NormForward); PREFIX template int launch<T, NormBackward>(int, bool, NormBackward); PREFIX template int launch<T, Dropout>(int, bool, Dropout);
#ifndef DEDF_ELEMENT
DEDF_LAUNCHES(float, extern) DEDF_LAUNCHES(_Float16, extern) DEDF_LAUNCHES(__bf16, extern)
#elif DEDF_ELEMENT == 0
DEDF_LAUNCHES(float, )
#elif DEDF_ELEMENT == 1
DEDF_LAUNCHES(_Float16, )
#else
DEDF_LAUNCHES(__bf16, )
#endif

}  // namespace rows
}  // namespace dedf

#ifndef DEDF_ELEMENT
namespace {

template <class F> int by_shape(int type, int width, bool fast, F f) {
    return type == DEDF_F32 ? launch<float>(width, fast, f) : type == DEDF_F16 ? launch<_Float16>(width, fast, f) : launch<__bf16>(width, fast, f);
}
size_t param_bytes(const Args& a) { return (size_t)grid(a, norm_blocks(true, a.s.width)) * 5 * a.s.channels * 4; }
size_t gate_bytes(const Args& a) { return a.gate && a.groups > 1 && a.slices > 1 ? (size_t)a.groups * a.slices * a.s.channels * 4 : 0; }
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

extern "C" {

int dedf_norm_gate_residual(const dedf_norm* x, void* h, void* z, int64_t* rng_used, void* stream) {
    Args a; bool fast;
    const int rc = make_args(x, false, a, fast);
    if (rc != DEDF_OK) return rc;
    if (a.n_rows == 0) return DEDF_OK;          // (tensors without elements may have no address)
    if ((x->y != nullptr) != (h != nullptr) || (x->next_weight != nullptr) != (z != nullptr) || (!h && !z)) return DEDF_ERR_INVALID;
    a.h = h; a.z = z; a.rng_used = rng_used;
    fast = fast && on_quads(x->type, {a.x, a.y, h, z});
    NormForward f{a, static_cast<hipStream_t>(stream)};
    return by_shape(x->type, a.s.width, fast, f);
}

size_t dedf_norm_scratch_bytes(const dedf_norm* x) {
    Args a; bool fast;
    if (make_args(x, true, a, fast) != DEDF_OK || a.n_rows == 0) return 0;
    return up16(param_bytes(a)) + gate_bytes(a);
}

int dedf_norm_gate_residual_backward(const dedf_norm* x, const void* grad_h, const void* grad_z, void* d_x, void* d_y, void* d_gate,
                                     float* d_post_weight, float* d_post_bias, float* d_next_weight, float* d_next_bias,
                                     void* scratch, size_t scratch_bytes, void* stream) {
    Args a; bool fast;
    const int rc = make_args(x, true, a, fast);
    if (rc != DEDF_OK) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool params = d_post_weight || d_post_bias || d_next_weight || d_next_bias;
    if (a.n_rows == 0) {          // no row: the parameters' gradients are zero (a sum over no rows), those of any number of gate rows too
        const int C = a.s.channels;
        const int64_t sums = (int64_t)x->groups * C;
        if (d_gate && sums > 0)          // (16-bit types share their zero)
            hipLaunchKernelGGL(k_few_rows<_Float16>, dim3((unsigned)std::min<int64_t>((sums + 255) / 256, 1 << 20)), dim3(256), 0, st, (const float*)nullptr, 0, C, sums,
                               a.gate_f32 ? nullptr : (_Float16*)d_gate, a.gate_f32 ? (float*)d_gate : nullptr);
        if (params) hipLaunchKernelGGL(k_row_sums<float>, dim3((4 * C + 15) / 16), dim3(1024), 0, st, (const float*)nullptr, 0, 4 * C, C,
                                       Outputs{{d_post_weight, d_post_bias, d_next_weight, d_next_bias, nullptr}, {C, a.s.scalars, C, a.s.scalars, 0}, {}});
        return hipGetLastError() == hipSuccess ? DEDF_OK : DEDF_ERR_RUNTIME;
    }
    if ((!grad_h && !grad_z) || (grad_z && !x->next_weight) || (d_y && !x->y) || (d_gate && !x->gate)) return DEDF_ERR_INVALID;
    const size_t need = up16(param_bytes(a)) + gate_bytes(a);
    if (!scratch || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15)) return DEDF_ERR_INVALID;
    a.dh = grad_h; a.dz = grad_z; a.dx = d_x; a.dy = d_y; a.d_gate = d_gate;
    const bool shared_gate = d_gate && a.groups == 1;          // a gradient like the norms' weights
    a.gate_rows = d_gate && !shared_gate && a.slices > 1 ? (float*)((char*)scratch + up16(param_bytes(a))) : nullptr;
    a.param_rows = params || shared_gate ? (float*)scratch : nullptr;
    a.n_params = shared_gate ? 5 : 4;
    fast = fast && on_quads(x->type, {a.x, a.y, grad_h, grad_z, d_x, d_y});
    NormBackward f{a, st, d_post_weight, d_post_bias, d_next_weight, d_next_bias};
    return by_shape(x->type, a.s.width, fast, f);
}

int dedf_channel_dropout(int type, int n_rows, int n_blocks, const int* mul, const int* degree, const void* x, double dropout, const int64_t* rng,
                         void* out, int64_t* rng_used, void* stream) {
    Args a{}; bool fast;
    if (type != DEDF_F32 && type != DEDF_F16 && type != DEDF_BF16) return DEDF_ERR_UNSUPPORTED;
    const int rc = make_shape(n_blocks, mul, degree, a.s, fast);
    if (rc != DEDF_OK) return rc;
    if (n_rows < 0 || (n_rows > 0 && (!x || !out)) || !(dropout >= 0.0 && dropout < 1.0) || (dropout > 0.0 && !rng)) return DEDF_ERR_INVALID;
    if (n_rows == 0) return DEDF_OK;
    a.n_rows = n_rows; a.x = x; a.h = out; a.rng_used = rng_used;
    a.threshold = (uint32_t)std::floor(dropout * 4294967296.0); a.keep_scale = (float)(1.0 / (1.0 - dropout)); a.rng = rng;
    fast = fast && on_quads(type, {x, out});
    Dropout f{a, static_cast<hipStream_t>(stream)};
    return by_shape(type, a.s.width, fast, f);
}

}  // extern "C"
#endif
