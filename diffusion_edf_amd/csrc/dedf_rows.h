// Row operators on irreps features in their training form: the norms around a block fused with its dropout, gate and residual scale
// (EquivariantLayerNormV2, reference equiformer/layer_norm.py:91-156; skips and projections' dropout, gnn_block.py:164-218), and dropout of whole
// channels (EquivariantDropout, equiformer/drop.py:76-96), each with its backward pass.
//
//   u = post(y)          h = x + scale gate[group, channel] keep[row, channel] u          z = next(h)
//   norm(f)[c] = w[channel] (f[c] - mean) r + bias:  mean over the scalars (degree 0 only), r = (mean of the degree's squares + eps)^-1/2
// backward, p = dz w, n = the normalised value:  df = r (p - n mean(p n)), for the scalars minus its mean; sums over rows give the parameters' gradients
//
// A wave (four for wide rows) owns a row: a lane holds quads of 4 consecutive components in registers, the degree sums go through the wave once each.  Everything a
// row needs is read once and its results written once, so memory bandwidth bounds both directions; the backward pass reads the inputs and computes the
// forward values again instead of storing them.  All sums are in 32 bits over at most 2 048 components; sums over rows are kept per lane, folded per
// workgroup and added in 64 bits in a fixed order.
#pragma once
#include "dedf_philox.h"

namespace dedf {
namespace rows {

constexpr int kWaves = 4, kMostBlocks = 4;          // waves of a workgroup; degrees of a feature row

// Waves a SIMD holds, by registers; a launch of the norms has as many workgroups as are resident at once, which share out the rows evenly
constexpr int forward_waves(int nq) { return nq == 1 ? 6 : 4; }
constexpr int backward_waves(int nq) { return nq == 1 ? 4 : 2; }

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
template <class T> struct Quad;
template <> struct Quad<float> { typedef f4 type; };
template <> struct Quad<_Float16> { typedef h4 type; };
template <> struct Quad<__bf16> { typedef b4 type; };

struct Shape {
    int n_blocks, width, channels, scalars;          // scalars: channels of degree 0 (the first block), 0 if there is none
    int start[kMostBlocks + 1];                      // first component of a block
    int first[kMostBlocks];                          // first channel
    int d[kMostBlocks];                              // components of a channel
    int divide[kMostBlocks];                         // (x divide) >> 16 = x / d for components x of a block
    float inverse[kMostBlocks];                      // 1 / components of a block; 0 and an empty range for a block that is not there
};
struct Args {
    Shape s;
    int n_rows, groups, slices, slice_rows;          // a unit of work: one slice of one group's consecutive rows
    const void* x; const void* y;
    const void* gate; int gate_f32;
    const float* post_w; const float* post_b; const float* next_w; const float* next_b;
    float scale, eps;
    uint32_t threshold; float keep_scale;
    const int64_t* rng;
    // forward
    void* h; void* z; int64_t* rng_used;
    // backward
    const void* dh; const void* dz; void* dx; void* dy;
    void* d_gate; float* gate_rows;                  // a group with one slice writes its gradient, else (unit, channels) sums
    float* param_rows; int n_params;                 // (workgroups, n_params channels): post weight, post bias, next weight, next bias; the gate of one group
};

template <int CTRL> __device__ inline float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// x of the rows of 16 lanes added in pairs, then of the halves of the wave: every lane gets the sum over the lanes with its place in a row
__device__ inline float add_rows(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    x = __builtin_bit_cast(float, (unsigned)a[0]) + __builtin_bit_cast(float, (unsigned)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, (unsigned)b[0]) + __builtin_bit_cast(float, (unsigned)b[1]);
}
// sum over the wave, in every lane
__device__ inline float wave_sum(float x) {
    x += dpp<0xB1>(x);           // neighbours, pairs, halves of a row, rows
    x += dpp<0x4E>(x);
    x += dpp<0x141>(x);
    x += dpp<0x140>(x);
    return add_rows(x);
}
// four sums over the wave at once: lane i gets the sum of v[i % 4].  The first two steps halve the number of values a lane carries instead of adding
// all four in every lane.
__device__ inline float wave_sums4(const float (&v)[4], int lane) {
    const bool odd = lane & 1, upper = lane & 2;
    const float a = (odd ? v[1] : v[0]) + dpp<0xB1>(odd ? v[0] : v[1]);
    const float b = (odd ? v[3] : v[2]) + dpp<0xB1>(odd ? v[2] : v[3]);
    float c = (upper ? b : a) + dpp<0x4E>(upper ? a : b);
    c += dpp<0x124>(c);          // the other quads of a row: rotations by 4 and 8
    c += dpp<0x128>(c);
    return add_rows(c);
}
__device__ inline void wave_sync() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// a lane's components of a row and where they belong.  FAST: blocks start on whole, aligned quads, so a quad has one degree and is one access.  WPR:
// waves that share a row (1; 4, the whole workgroup, for rows over 512 components).  One wave with four quads a lane spills 329 registers in the backward kernel (bfloat16, two waves a
// SIMD); with three, for up to 768 components, that kernel keeps its 246 and the forward one spills 121 at its four waves a SIMD: not timed.  Lanes behind the row's end repeat its last quad;
// they belong to no block and are not stored.  Rows off whole quads are read element by element: 100 000 float32 rows of 33x0e+17x1e, post-norm to next norm, 65 us forward and
// 142 backward, of 32x0e+16x1e 40 and 83 (bfloat16: 72 and 167, 36 and 82).
template <class T, int NQ, bool FAST, int WPR> struct Row {
    typedef typename Quad<T>::type Raw;
    const Shape& s; int lane;             // of the row's WPR x 64
    float* own; float* exchange; int turn;
    int64_t held;                         // row whose dropout words LDS holds (and the next one's, where two rows fit)
    int block[NQ][FAST ? 1 : 4];          // -1: no component
    int channel[NQ][4];
    float inverse[NQ][FAST ? 1 : 4];      // 1 / components of the block
    __device__ Row(const Shape& shape, char* lds, int team) : s(shape), lane(threadIdx.x & (64 * WPR - 1)), turn(0), held(-2) {
        own = (float*)(lds + team * team_bytes(shape));
        exchange = own + own_floats(shape);
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int c = 4 * (j * 64 * WPR + lane) + i;
                int b = -1, ch = 0;
                float inv = 0.0f;
#pragma unroll
                for (int k = 0; k < kMostBlocks; ++k) {
                    const bool in = (c >= s.start[k]) & (c < s.start[k + 1]);
                    b = in ? k : b;
                    inv = in ? s.inverse[k] : inv;
                    ch = in ? s.first[k] + (((c - s.start[k]) * s.divide[k]) >> 16) : ch;
                }
                channel[j][i] = ch;
                if (!FAST || i == 0) { block[j][FAST ? 0 : i] = b; inverse[j][FAST ? 0 : i] = inv; }
            }
    }
    __device__ int of(int j, int i) const { return block[j][FAST ? 0 : i]; }
    __device__ void load(f4 (&f)[NQ], const void* p, int64_t row) const {
        const T* at = (const T*)p + row * s.width;
        if constexpr (FAST) {
            Raw raw[NQ];
#pragma unroll
            for (int j = 0; j < NQ; ++j) raw[j] = *(const Raw*)(at + min(4 * (j * 64 * WPR + lane), s.width - 4));
#pragma unroll
            for (int j = 0; j < NQ; ++j) f[j] = f4{(float)raw[j][0], (float)raw[j][1], (float)raw[j][2], (float)raw[j][3]};
        } else {
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) { const int c = 4 * (j * 64 * WPR + lane) + i; f[j][i] = c < s.width ? (float)at[c] : 0.0f; }
        }
    }
    __device__ void store(void* p, int64_t row, const f4 (&f)[NQ]) const {
        T* at = (T*)p + row * s.width;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            const int c = 4 * (j * 64 * WPR + lane);
            if constexpr (FAST) { if (c < s.width) *(Raw*)(at + c) = Raw{(T)f[j][0], (T)f[j][1], (T)f[j][2], (T)f[j][3]}; }
            else {
#pragma unroll
                for (int i = 0; i < 4; ++i) if (c + i < s.width) at[c + i] = (T)f[j][i];
            }
        }
    }
    // a channel's value on each of its components; channels from n on have 0
    __device__ void spread(f4 (&f)[NQ], const float* values, int n) const {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            f[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (n > 0)
#pragma unroll
                for (int i = 0; i < 4; ++i) { const float x = values[min(channel[j][i], n - 1)]; f[j][i] = channel[j][i] < n ? x : 0.0f; }
        }
    }
    __device__ void sync() const { if constexpr (WPR == 1) wave_sync(); else __syncthreads(); }
    // a lane's share of the sums over each block of f g
    __device__ void block_parts(float (&part)[kMostBlocks], const f4 (&f)[NQ], const f4 (&g)[NQ]) const {
#pragma unroll
        for (int k = 0; k < kMostBlocks; ++k) part[k] = 0.0f;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            if constexpr (FAST) {
                const f4 m = f[j] * g[j];
                const float q = (m[0] + m[1]) + (m[2] + m[3]);
#pragma unroll
                for (int k = 0; k < kMostBlocks; ++k) part[k] += block[j][0] == k ? q : 0.0f;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int k = 0; k < kMostBlocks; ++k) part[k] += of(j, i) == k ? f[j][i] * g[j][i] : 0.0f;
            }
        }
    }
    __device__ float scalar_part(const f4 (&f)[NQ]) const {
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) part += of(j, i) == 0 ? f[j][i] : 0.0f;
        return part;
    }
    typedef float PerQuad[NQ][FAST ? 1 : 4];
    static __device__ float at(const PerQuad& v, int j, int i) { return v[j][FAST ? 0 : i]; }
    // the blocks' sums of parts (by block) and the scalars' sum of one more value: each component's own block's sum, and the latter
    __device__ float sums(PerQuad& own_sum, const float (&part)[kMostBlocks], float scalar) {
        float c = wave_sums4(part, lane);
        scalar = wave_sum(scalar);
        if constexpr (WPR > 1) {          // (two buffers in turn: a wave that is one exchange ahead does not touch what another still reads)
            float* to = exchange + turn * WPR * 8;
            turn ^= 1;
            if ((lane & 63) < 4) to[(lane >> 6) * 8 + (lane & 3)] = c;
            if ((lane & 63) == 4) to[(lane >> 6) * 8 + 4] = scalar;
            __syncthreads();
            scalar = 0.0f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) scalar += to[w * 8 + 4];
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < (FAST ? 1 : 4); ++i) {
                    own_sum[j][i] = 0.0f;
#pragma unroll
                    for (int w = 0; w < WPR; ++w) own_sum[j][i] += to[w * 8 + (block[j][i] & 3)];
                }
        } else {
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < (FAST ? 1 : 4); ++i) own_sum[j][i] = __shfl(c, (lane & ~3) | (block[j][i] & 3));
        }
        return scalar;
    }
    // the sum of one value alone
    __device__ float sum(float x) {
        x = wave_sum(x);
        if constexpr (WPR > 1) {
            float* to = exchange + turn * WPR * 8;
            turn ^= 1;
            if ((lane & 63) == 0) to[(lane >> 6) * 8] = x;
            __syncthreads();
            x = 0.0f;
#pragma unroll
            for (int w = 0; w < WPR; ++w) x += to[w * 8];
        }
        return x;
    }
    // f becomes its normalised value n, r the factor of each component's block
    __device__ void normalise(f4 (&f)[NQ], PerQuad& r, float eps) {
        if (s.scalars) {
            const float mean = sum(scalar_part(f)) * s.inverse[0];
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) f[j][i] -= of(j, i) == 0 ? mean : 0.0f;
        }
        float part[kMostBlocks];
        block_parts(part, f, f);
        sums(r, part, 0.0f);
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < (FAST ? 1 : 4); ++i) r[j][i] = __builtin_amdgcn_rsqf(fmaf(r[j][i], inverse[j][i], eps));
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) f[j][i] *= at(r, j, i);
    }
    // g: gradient of the normalised value n -> gradient of the value before the norm
    __device__ void normalise_back(f4 (&g)[NQ], const f4 (&n)[NQ], const PerQuad& r) {
        float part[kMostBlocks];
        PerQuad dot;
        block_parts(part, g, n);
        const float scalar = sums(dot, part, scalar_part(g)), mean = s.scalars ? scalar * s.inverse[0] : 0.0f;
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) g[j][i] = at(r, j, i) * (g[j][i] - (of(j, i) == 0 ? mean : 0.0f) - n[j][i] * (at(dot, j, i) * at(inverse, j, i)));
    }
    // dropout factors of a row, one word for each channel, through LDS: of this row and the next at once where both fit into the row's lanes
    __device__ void keep(f4 (&f)[NQ], int64_t row, uint64_t offset, uint64_t seed, uint32_t threshold, float scale) {
        const int groups = (s.channels + 3) >> 2, rows = two_rows(s) ? 2 : 1;
        if (row != held && (rows == 1 || row != held + 1)) {
            sync();
            for (int idx = lane; idx < rows * groups; idx += 64 * WPR) {
                const int next = idx >= groups, g = idx - (next ? groups : 0);
                const Words x = dropout_words((uint32_t)(row + next), (1u << 16) + g, offset, seed);
                *(f4*)(own + 4 * idx) = f4{x.w[0] >= threshold ? scale : 0.0f, x.w[1] >= threshold ? scale : 0.0f, x.w[2] >= threshold ? scale : 0.0f, x.w[3] >= threshold ? scale : 0.0f};
            }
            held = row;
            sync();
        }
        const float* at = own + (row == held ? 0 : 4 * groups);
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) f[j][i] = at[channel[j][i]];
    }
    // components to LDS, from which folded() adds up a channel's
    __device__ void fold(const f4 (&f)[NQ]) {
        held = -2;
        sync();
#pragma unroll
        for (int j = 0; j < NQ; ++j) if (4 * (j * 64 * WPR + lane) < s.width) *(f4*)(own + 4 * (j * 64 * WPR + lane)) = f[j];
        sync();
    }
    __device__ float folded(const float* lds, int c) const {
        int b = 0;
        for (int k = 1; k < s.n_blocks; ++k) if (c >= s.first[k]) b = k;
        float sum = 0.0f;
        const int at = s.start[b] + (c - s.first[b]) * s.d[b];
        for (int i = 0; i < s.d[b]; ++i) sum += lds[at + i];
        return sum;
    }
    static __host__ __device__ bool two_rows(const Shape& s) { return s.channels <= 128; }
    static __host__ __device__ int own_floats(const Shape& s) {
        const int c = (s.channels + 3) & ~3, w = (s.width + 3) & ~3, k = two_rows(s) ? 2 * c : c;
        return w > k ? w : k;
    }
    static __host__ __device__ size_t team_bytes(const Shape& s) { return (size_t)own_floats(s) * 4 + (WPR > 1 ? 2 * WPR * 8 * 4 : 0); }
};

template <class T> __device__ inline float gate_at(const void* gate, int f32, int64_t i) { return f32 ? ((const float*)gate)[i] : (float)((const T*)gate)[i]; }

// Reads x and y, writes h and z: 103 000 rows of 240 float32 in 81 us, 4.9 TB/s, a large copy's rate.
template <class T, int NQ, bool FAST, int WPR> __global__ __launch_bounds__(256, forward_waves(NQ)) void k_norm_forward(Args P) {
    extern __shared__ __align__(16) char lds[];
    if (P.rng_used && P.threshold && blockIdx.x == 0 && threadIdx.x < 2) P.rng_used[threadIdx.x] = P.rng[threadIdx.x];
    constexpr int TEAMS = kWaves / WPR;
    const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WPR));          // (known to be uniform: row addresses stay scalar)
    Row<T, NQ, FAST, WPR> R(P.s, lds, team);
    uint64_t seed = 0, offset = 0;
    if (P.threshold) { seed = (uint64_t)P.rng[0]; offset = (uint64_t)P.rng[1]; }
    f4 pw[NQ], pb[NQ], nw[NQ], nb[NQ], gate[NQ];
    if (P.post_w) { R.spread(pw, P.post_w, P.s.channels); R.spread(pb, P.post_b, P.s.scalars); }
    if (P.z) { R.spread(nw, P.next_w, P.s.channels); R.spread(nb, P.next_b, P.s.scalars); }
    // (unsigned: the step behind the last unit and the end of a group's last slice pass 2^31)
    const uint32_t slices = P.slices, slice_rows = P.slice_rows, units = P.groups * slices, group_rows = P.n_rows / P.groups;
    for (uint32_t u = blockIdx.x * TEAMS + team; u < units; u += gridDim.x * TEAMS) {
        const uint32_t g = u / slices, first = (u - g * slices) * slice_rows, last = min(first + slice_rows, group_rows);
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) gate[j][i] = P.scale * (P.gate ? gate_at<T>(P.gate, P.gate_f32, (int64_t)g * P.s.channels + R.channel[j][i]) : 1.0f);
        for (uint32_t k = first; k < last; ++k) {
            const int64_t row = (int64_t)g * group_rows + k;
            f4 h[NQ], y[NQ];
            R.load(h, P.x, row);
            if (P.y) {
                R.load(y, P.y, row);
                if (P.post_w) {
                    typename Row<T, NQ, FAST, WPR>::PerQuad r;
                    R.normalise(y, r, P.eps);
#pragma unroll
                    for (int j = 0; j < NQ; ++j) y[j] = y[j] * pw[j] + pb[j];
                }
                if (P.threshold) {
                    f4 m[NQ];
                    R.keep(m, row, offset, seed, P.threshold, P.keep_scale);
#pragma unroll
                    for (int j = 0; j < NQ; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[j][i] = m[j][i] == 0.0f ? 0.0f : y[j][i] * m[j][i];
                }
#pragma unroll
                for (int j = 0; j < NQ; ++j) h[j] += gate[j] * y[j];
                R.store(P.h, row, h);
            }
            if (P.z) {
                typename Row<T, NQ, FAST, WPR>::PerQuad r;
                R.normalise(h, r, P.eps);
#pragma unroll
                for (int j = 0; j < NQ; ++j) h[j] = h[j] * nw[j] + nb[j];
                R.store(P.z, row, h);
            }
        }
    }
}

// Reads x, y, dh, dz, writes dx, dy: 103 000 rows of 240 float32 in 149 us, 4.0 TB/s; 415 vector instructions a row at 4 waves a SIMD come next to the
// memory.  16 384 rows of lmax 3 in float16 49 us, 1.2 TB/s: the two waves of a SIMD wait in half of their time, for a row's loads
// and then for its sums, and vector instructions issue in 46 % of the cycles: latency.  Summing the four degrees with one value a lane (wave_sums4) instead of four chains, and choosing a degree's sum before its root: 218 us before.
template <class T, int NQ, bool FAST, int WPR> __global__ __launch_bounds__(256, backward_waves(NQ)) void k_norm_backward(Args P) {
    extern __shared__ __align__(16) char lds[];
    typedef Row<T, NQ, FAST, WPR> Rw;
    constexpr int TEAMS = kWaves / WPR;
    const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WPR)), C = P.s.channels;
    Rw R(P.s, lds, team);
    uint64_t seed = 0, offset = 0;
    if (P.threshold) { seed = (uint64_t)P.rng[0]; offset = (uint64_t)P.rng[1]; }
    const bool post = P.post_w != nullptr, next = P.dz != nullptr;
    f4 pw[NQ], pb[NQ], nw[NQ], gate[NQ], d_pw[NQ], d_pb[NQ], d_nw[NQ], d_nb[NQ], d_gate[NQ];
    if (post) { R.spread(pw, P.post_w, C); R.spread(pb, P.post_b, P.s.scalars); }
    if (next) R.spread(nw, P.next_w, C);
#pragma unroll
    for (int j = 0; j < NQ; ++j) d_pw[j] = d_pb[j] = d_nw[j] = d_nb[j] = d_gate[j] = f4{0, 0, 0, 0};
    // (unsigned: as in the forward pass)
    const uint32_t slices = P.slices, slice_rows = P.slice_rows, units = P.groups * slices, group_rows = P.n_rows / P.groups;
    for (uint32_t u = blockIdx.x * TEAMS + team; u < units; u += gridDim.x * TEAMS) {
        const uint32_t g = u / slices, first = (u - g * slices) * slice_rows, last = min(first + slice_rows, group_rows);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            if (P.n_params < 5) d_gate[j] = f4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) gate[j][i] = P.gate ? gate_at<T>(P.gate, P.gate_f32, (int64_t)g * C + R.channel[j][i]) : 1.0f;
        }
        for (uint32_t k = first; k < last; ++k) {
            const int64_t row = (int64_t)g * group_rows + k;
            f4 h[NQ], n[NQ], y[NQ], m[NQ], up[NQ];
            typename Rw::PerQuad ry;
            R.load(h, P.x, row);
            if (P.y) R.load(y, P.y, row);
            if (P.dh) R.load(up, P.dh, row);
            else
#pragma unroll
                for (int j = 0; j < NQ; ++j) up[j] = f4{0, 0, 0, 0};
            if (P.y) {
                if (post) R.normalise(y, ry, P.eps);
                if (P.threshold) R.keep(m, row, offset, seed, P.threshold, P.keep_scale);
#pragma unroll
                for (int j = 0; j < NQ; ++j) {
                    if (!P.threshold) m[j] = f4{1.0f, 1.0f, 1.0f, 1.0f};
                    m[j] *= P.scale;
                    const f4 un = post ? y[j] * pw[j] + pb[j] : y[j];
#pragma unroll
                    for (int i = 0; i < 4; ++i) h[j][i] += m[j][i] == 0.0f ? 0.0f : gate[j][i] * m[j][i] * un[i];
                }
            }
            if (next) {
                f4 dz[NQ];
                typename Rw::PerQuad r;
                R.load(dz, P.dz, row);
#pragma unroll
                for (int j = 0; j < NQ; ++j) n[j] = h[j];
                R.normalise(n, r, P.eps);
#pragma unroll
                for (int j = 0; j < NQ; ++j) {
                    d_nw[j] += dz[j] * n[j];
                    d_nb[j] += dz[j];
                    dz[j] *= nw[j];
                }
                R.normalise_back(dz, n, r);
#pragma unroll
                for (int j = 0; j < NQ; ++j) up[j] += dz[j];
            }
            if (P.dx) R.store(P.dx, row, up);
            if (!P.y) continue;
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                const f4 un = post ? y[j] * pw[j] + pb[j] : y[j];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float t = m[j][i] == 0.0f ? 0.0f : m[j][i] * up[j][i];
                    d_gate[j][i] += t == 0.0f ? 0.0f : t * un[i];
                    up[j][i] = t * gate[j][i];
                }
                if (post) {
                    d_pw[j] += up[j] * y[j];
                    d_pb[j] += up[j];
                    up[j] *= pw[j];
                }
            }
            if (!P.dy) continue;
            if (post) R.normalise_back(up, y, ry);
            R.store(P.dy, row, up);
        }
        if (P.n_params < 5 && (P.d_gate || P.gate_rows)) {
            R.fold(d_gate);
            for (int c = R.lane; c < C; c += 64 * WPR) {
                const float s = R.folded(R.own, c);
                if (P.gate_rows) P.gate_rows[(int64_t)u * C + c] = s;
                else if (P.gate_f32) ((float*)P.d_gate)[(int64_t)u * C + c] = s;
                else ((T*)P.d_gate)[(int64_t)u * C + c] = (T)s;
            }
        }
    }
    if (!P.param_rows) return;
    // the workgroup's sums, a parameter at a time
#pragma unroll 1
    for (int which = 0; which < P.n_params; ++which) {
        f4 d[NQ];
#pragma unroll
        for (int j = 0; j < NQ; ++j) d[j] = which == 0 ? d_pw[j] : which == 1 ? d_pb[j] : which == 2 ? d_nw[j] : which == 3 ? d_nb[j] : d_gate[j];
        __syncthreads();
        R.fold(d);
        __syncthreads();
        for (int c = threadIdx.x; c < C; c += 256) {
            float s = 0.0f;
            for (int x = 0; x < TEAMS; ++x) s += R.folded((const float*)(lds + x * Rw::team_bytes(P.s)), c);
            P.param_rows[((int64_t)blockIdx.x * P.n_params + which) * C + c] = s;
        }
    }
}

// x keep: forward and backward are the same map; 103 000 rows of 240 float32 in 43 us, 4.6 TB/s
template <class T, int NQ, bool FAST, int WPR> __global__ __launch_bounds__(256) void k_dropout(Args P) {
    extern __shared__ __align__(16) char lds[];
    if (P.rng_used && P.threshold && blockIdx.x == 0 && threadIdx.x < 2) P.rng_used[threadIdx.x] = P.rng[threadIdx.x];
    constexpr int TEAMS = kWaves / WPR;
    const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * WPR));          // (known to be uniform: row addresses stay scalar)
    Row<T, NQ, FAST, WPR> R(P.s, lds, team);
    uint64_t seed = 0, offset = 0;
    if (P.threshold) { seed = (uint64_t)P.rng[0]; offset = (uint64_t)P.rng[1]; }
    const int64_t first = ((int64_t)blockIdx.x * TEAMS + team) * P.slice_rows, last = min(first + P.slice_rows, (int64_t)P.n_rows);
    for (int64_t row = first; row < last; ++row) {
        f4 x[NQ], m[NQ];
        R.load(x, P.x, row);
        if (P.threshold) {
            R.keep(m, row, offset, seed, P.threshold, P.keep_scale);
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[j][i] = m[j][i] == 0.0f ? 0.0f : x[j][i] * m[j][i];
        }
        R.store(P.h, row, x);
    }
}

// sums over `rows` rows of (rows, columns) in 64 bits, in a fixed order; 16 columns a workgroup, one of blockIdx.y matrices.  Column c is element
// c % width of output c / width: its first n elements are written, as 32 bits or as T.
struct Outputs { void* to[5]; int n[5]; int narrow[5]; };
template <class T> __global__ __launch_bounds__(1024) void k_row_sums(const float* x, int rows, int columns, int width, Outputs out) {
    __shared__ double share[64][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), r0 = threadIdx.x >> 4;
    const float* m = x + (size_t)blockIdx.y * rows * columns + c;
    double s = 0.0;
    if (c < columns) {
        int r = r0;
        for (; r + 3 * 64 < rows; r += 4 * 64) {
            const float a = m[(size_t)r * columns], b = m[(size_t)(r + 64) * columns], d = m[(size_t)(r + 128) * columns], e = m[(size_t)(r + 192) * columns];
            s += ((double)a + (double)b) + ((double)d + (double)e);
        }
        for (; r < rows; r += 64) s += (double)m[(size_t)r * columns];
    }
    share[r0][threadIdx.x & 15] = s;
    for (int half = 32; half >= 1; half >>= 1) {
        __syncthreads();
        if (r0 < half) share[r0][threadIdx.x & 15] += share[r0 + half][threadIdx.x & 15];
    }
    if (r0 != 0 || c >= columns) return;
    const int which = c / width, at = c - which * width;
    if (!out.to[which] || at >= out.n[which]) return;
    const float v = (float)share[0][threadIdx.x & 15];
    const size_t to = (size_t)blockIdx.y * out.n[which] + at;
    if (out.narrow[which]) ((T*)out.to[which])[to] = (T)v; else ((float*)out.to[which])[to] = v;
}

// the same for many matrices of a few rows: a thread a sum
template <class T> __global__ __launch_bounds__(256) void k_few_rows(const float* x, int rows, int columns, int64_t sums, T* narrow, float* wide) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < sums; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / columns;
        const float* at = x + m * rows * columns + (i - m * columns);
        double s = 0.0;
        for (int r = 0; r < rows; ++r) s += (double)at[(int64_t)r * columns];
        if (narrow) narrow[i] = (T)(float)s; else wide[i] = (float)s;
    }
}

}  // namespace rows
}  // namespace dedf
