// Attention over a sorted edge list in its training form: the last part of GraphAttentionMLP2 (reference graph_attention.py:237-273) with gradients.
//
//   s[e,h] = sum_k act(a[e,h,k]) w[h,k]           act(x) = c x (0.2 + 0.8 sigma(x)), SmoothLeakyReLU(0.2) under normalize2mom
//   t[e,h] = s + l[e] + T[bucket(len[e]), h]      bucket(x) = number of boundaries <= x
//   p      = softmax of t over the edges of a destination; an edge and head with t = -inf takes no part
//   P      = p m / (1 - q)                        m from Philox4x32-10, key = seed, counter = (edge, head / 4, offset), word head % 4
//   out[n,h,:] = sum_e P v[e,h,:]
// backward, from a logit M near a row and head's largest and 1 / Z, Z = sum exp(t - M), alone (the probabilities are recomputed, the mask is drawn again):
//   p = exp(t - M) / Z   dP = m/(1-q) (dout . v)   delta = dout . out   dt = p (dP - delta)
//   dv = P dout   dl = sum_h dt   dT[b,h] = sum dt   dw = sum_e dt act(a)   da = dt w act'(a)
//
// Both directions stream the per-edge rows once, so memory bandwidth bounds them.  A wave owns a contiguous RANGE of edges whatever the rows are:
// the load is even for any degree distribution, from one edge per row to one row with every edge.  It walks its range in batches of 16 edges; a lane
// holds 4 consecutive channels of one head (a "quad") of every row, 8 rows in flight.  Rows that lie inside a range are finished by its wave; a row
// that crosses ranges leaves one record per range, or per workgroup of ranges (running maximum, sum, weighted sum), which k_attn_merge joins in order: no
// atomics, and the result depends on the sizes alone.  Logits and maxima are held in 64 bits (with masks of a type's lowest value in edge_logits, t loses s in 32), and M and Z
// apart: beside such a mask log Z would be lost in 64.
#pragma once
#include "dedf_philox.h"

// products are fused into sums where it says so, not where the compiler likes: a result does not depend on the instantiation that alignment picks
#pragma clang fp contract(off)

namespace dedf {
namespace attn {

constexpr int kBatch = 16;                 // edges per step of a wave
constexpr int kWaves = 4;                  // waves per workgroup
enum { kElements = 0, kHeads = 1, kAligned = 2 };          // how a row is cut into quads: see load_quad
// Waves a SIMD holds, by the registers of each instantiation; a launch has as many waves as are resident at once, each with one range of edges.  More
// waves than that run in two rounds, of which the second is half empty: 1.97 M edges, float32, a training pass with two waves a SIMD
// in the backward kernel 1.65 ms, with three 1.83 ms.
constexpr int forward_waves(int nv, int bytes) { return nv == 4 ? 2 : nv == 1 && bytes == 2 ? 4 : 3; }
constexpr int backward_waves(int nv, int bytes) { return bytes == 2 && nv <= 2 ? 3 : 2; }          // (499 979 edges, lmax 3, bfloat16: 0.46 ms with 3, 0.52 with 2)
constexpr float kActNorm = 1.531320475574866f;
constexpr double kLog2e = 1.4426950408889634;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef double d2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
template <class T> struct Quad;
template <> struct Quad<float> { typedef f4 type; };
template <> struct Quad<_Float16> { typedef h4 type; };
template <> struct Quad<__bf16> { typedef b4 type; };

struct Args {
    int64_t n_edges;
    int n_dst, heads, k, d;
    const void* a; const void* v; const float* w;
    int64_t a_stride, v_stride;            // elements between the rows of two edges
    const int* dst; const int* rowptr;
    const float* logits; const float* length; const float* bounds; const float* table;
    int n_buckets;
    uint32_t threshold; float keep_scale;  // dropout: kept iff word >= threshold; threshold 0 = none
    const int64_t* rng;
    int range, n_waves;                    // edges per wave, waves
};

// How a row of H heads is cut into quads (MODE).  A quad lies inside one head.
//   kAligned   head widths are multiples of 4 and every row begins at a whole quad: an aligned access each
//   kHeads     any other head width from 4: the head's last quad ends with the head and so begins inside the one before; an unaligned access each.  What two
//              quads hold is summed by the first of them.
//   kElements  heads narrower than a quad: element by element, the others zero
// 400 000 edges of 3 heads of 17 + 33 channels, a training pass: float32 0.24 ms (quads across the heads, by elements: 0.42), bfloat16 0.20 ms (0.64); 4 aligned
// heads of 16 + 60 0.36 ms in float32, of 16 + 61 0.38 ms.
template <class T, int MODE> __device__ inline typename Quad<T>::type load_quad(const T* p, int width) {
    typename Quad<T>::type r = {(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
    if constexpr (MODE == kAligned) r = *(const typename Quad<T>::type*)p;
    else if constexpr (MODE == kHeads) __builtin_memcpy(&r, p, sizeof(r));
    else {
#pragma unroll
        for (int i = 0; i < 3; ++i) if (i < width) r[i] = p[i];
    }
    return r;
}
template <class T, int MODE> __device__ inline void store_quad(T* p, f4 x, int width) {
    const typename Quad<T>::type r = {(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
    if constexpr (MODE == kAligned) *(typename Quad<T>::type*)p = r;
    else if constexpr (MODE == kHeads) __builtin_memcpy(p, &r, sizeof(r));
    else {
#pragma unroll
        for (int i = 0; i < 3; ++i) if (i < width) p[i] = r[i];
    }
}
// quads of a row of H heads
__host__ __device__ constexpr int row_quads(int H, int width) { return H * ((width + 3) >> 2); }
// first element of the head's quad i, relative to the head, and how many of its elements the quad before holds too
__device__ inline int quad_begin(int i, int width) { return width < 4 ? 0 : min(4 * i, width - 4); }
__device__ inline int quad_shared(int begin) { return -begin & 3; }

// LDS of one wave is written and read by its own lanes only: LDS operations of a wave complete in order, the compiler must keep that order
__device__ inline void wave_sync() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// exp(x) to 1e-7 relative, x = -inf and NaN too: the exponent is split into whole and fraction in 64 bits, so a long way below the maximum loses
// nothing.  x is a logit less one that is at least the largest but for its rounding to float (0.03 at 1e6), or, in the backward pass, up to 24 above: no
// result passes 1.04
__device__ inline float exp_d(double x) {
    if (x < -150.0) return 0.0f;
    const double y = x * kLog2e, n = __builtin_rint(y);
    return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f((float)(y - n)), (int)n);
}
__device__ inline float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }
__device__ inline float act(float x) { return kActNorm * x * fmaf(0.8f, sigmoid(x), 0.2f); }

// number of boundaries <= x in a sorted list
__device__ inline int bucket_of(const float* bounds, int n, float x) {
    int lo = 0, hi = n;
    while (lo < hi) { const int mid = (lo + hi) >> 1; if (bounds[mid] <= x) lo = mid + 1; else hi = mid; }
    return lo;
}

// first element of each of the lane's value quads (the last one where it has none) and its head
template <int NV> __device__ inline void value_places(const Args& P, int lane, int (&begin)[NV], int (&head)[NV]) {
    const int per = (P.d + 3) >> 2;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int q = min(j * 64 + lane, P.heads * per - 1);
        head[j] = q / per;
        begin[j] = head[j] * P.d + quad_begin(q - head[j] * per, P.d);
    }
}

// what both directions share: the wave's place, its LDS, the batch's per-edge values, the logits
//   MODE: how value rows are cut (see load_quad); feature rows are cut that way too, with kHeads and kElements by the width of their own heads
//   NV: quads of a value row a lane holds: 1, 2 or 4 (up to 64, 128, 256 quads)
//   GA: edges whose features are loaded at once: 16 (feature rows of up to 16 quads), 8 (32), 4 (64) or 2 (128)
template <class T, int MODE, int NV, int GA> struct Wave {
    static constexpr int NA = 4;                                             // GA edges x feature quads fill NA loads of a wave
    static constexpr int rows(int quads) { return quads / NV < GA ? quads / NV : GA; }
    static constexpr int R = rows(8), RF = rows(NV > 1 && sizeof(T) == 2 ? 16 : 8);        // value rows in flight: backward, forward
    static constexpr int kPart = 256 * NA;                                   // floats of the partial-sum buffer
    const Args& P;
    int lane, wave, H, K, D, HK, HD, per_a, qa, qv;                          // (per_a: feature quads of a head)
    int begin_v[NV], head_v[NV];                                             // of the lane's value quads (the last one where it has none): first element, its head
    uint32_t inv_h, inv_qa, inv_per_a;
    int64_t e0, e1;
    float* part; double* t; float* keep; const float* w; const float* bounds; const float* table;
    uint64_t seed, offset;
    int64_t base; int n;                                                     // the batch: edges base .. base + n - 1, n <= 16
    uint32_t starts;                                                         // bit e: its edge e begins a row (or the batch)
    int* e_dst; int* e_bucket; float* e_logit;                               // its edges' destination, length bucket, edge logit

    static __host__ __device__ size_t wave_bytes(int H) { return (size_t)kPart * 4 + (size_t)kBatch * (H * 16 + 12); }
    static __host__ __device__ size_t shared_bytes(int qa, int H, int B) { return ((4 * (size_t)qa + (B ? B + (size_t)B * H : 0)) * 4 + 15) & ~(size_t)15; }

    __device__ Wave(const Args& p, char* lds, size_t own_bytes) : P(p) {
        lane = threadIdx.x & 63; wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);          // (known to be uniform: row addresses stay scalar)
        H = p.heads; K = p.k; D = p.d; HK = H * K; HD = H * D;
        per_a = (K + 3) >> 2; qa = row_quads(H, K); qv = row_quads(H, D);
        inv_h = (65536 + H - 1) / H; inv_qa = (65536 + qa - 1) / qa; inv_per_a = (65536 + per_a - 1) / per_a;
        value_places(P, lane, begin_v, head_v);
        float* s = (float*)lds;          // (filled by stage())
        const int hk4 = 4 * qa, B = p.n_buckets;
        w = s; bounds = s + hk4; table = s + hk4 + B;
        char* mine = lds + shared_bytes(qa, H, B) + wave * own_bytes;
        t = (double*)mine; part = (float*)(mine + (size_t)kBatch * H * 8); keep = part + kPart;
        e_logit = keep + 2 * kBatch * H; e_dst = (int*)(e_logit + kBatch); e_bucket = e_dst + kBatch;
        seed = offset = 0;
        if (p.threshold) { seed = (uint64_t)p.rng[0]; offset = (uint64_t)p.rng[1]; }
        const int64_t id = (int64_t)blockIdx.x * kWaves + wave;
        e0 = min(id * p.range, p.n_edges); e1 = min(e0 + p.range, p.n_edges);
    }
    // the call's parameters into LDS: for every wave of the workgroup, behind its first loads of edges
    __device__ void stage(char* lds) const {
        float* s = (float*)lds;
        const int hk4 = 4 * qa, B = P.n_buckets;
        for (int i = threadIdx.x; i < hk4; i += blockDim.x) { int h; const int c = begin_a(i >> 2, h) + (i & 3); s[i] = (i & 3) < K ? P.w[c] : 0.0f; }
        for (int i = threadIdx.x; i < B - 1; i += blockDim.x) s[hk4 + i] = P.bounds[i];
        for (int i = threadIdx.x; i < B * H; i += blockDim.x) s[hk4 + B + i] = P.table[i];
        __syncthreads();
    }
    // per-edge values of the batch at b: requested early (into registers of the first 16 lanes), put into LDS when the batch begins
    struct Edge { int dst; float logit, length; };
    __device__ Edge request(int64_t b) const {
        const int64_t e = min(b + (lane & (kBatch - 1)), e1 - 1);          // (places behind the last edge repeat it)
        return Edge{P.dst[e], P.logits ? P.logits[e] : 0.0f, P.n_buckets ? P.length[e] : 0.0f};
    }
    __device__ void begin(int64_t b, const Edge& x) {
        base = b; n = (int)min((int64_t)kBatch, e1 - b);
        if (lane < kBatch) {
            e_dst[lane] = x.dst;
            e_logit[lane] = x.logit;
            e_bucket[lane] = P.n_buckets ? bucket_of(bounds, P.n_buckets - 1, x.length) : 0;
        }
        const int before = __shfl_up(x.dst, 1);
        starts = (uint32_t)__ballot(lane < n && (lane == 0 || x.dst != before));
    }
    // first element of feature quad q and its head
    __device__ int begin_a(int q, int& h) const {
        h = (int)((q * inv_per_a) >> 16);
        return MODE == kAligned ? 4 * q : h * K + quad_begin(q - h * per_a, K);
    }
    // feature quad i of the edges e_first .. e_first + GA - 1: its edge (relative to e_first) and quad; false if there is none
    __device__ bool a_place(int i, int e_first, int& e, int& q) const {
        const int idx = i * 64 + lane;
        e = (int)((idx * inv_qa) >> 16); q = idx - e * qa;
        return e < GA && e_first + e < n;
    }
    // Loads go out unconditionally (places that do not exist repeat an edge or the row's last quad): a branch around each would make the wave wait
    // for one row at a time.
    typedef typename Quad<T>::type Raw;
    __device__ void load_a(Raw (&a)[NA], int64_t base, int n, int e_first) const {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            int h;
            const int idx = i * 64 + lane, e = (int)((idx * inv_qa) >> 16), q = idx - e * qa, c = begin_a(q, h);
            const T* p = (const T*)P.a + (base + min(e_first + e, n - 1)) * P.a_stride + c;
            if (MODE == kAligned) a[i] = load_quad<T, kAligned>(p, 4);
            else a[i] = K < 4 ? load_quad<T, kElements>(p, K) : load_quad<T, kHeads>(p, 4);
        }
    }
    // the lane's quads of a row of H D elements
    __device__ void load_row(Raw (&v)[NV], const T* row) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            v[j] = load_quad<T, MODE>(row + begin_v[j], D);
        }
    }
    __device__ const T* value_row(int64_t e) const { return (const T*)P.v + min(e, e1 - 1) * P.v_stride; }
    __device__ float dropped(int64_t edge, int h) const {
        if (!P.threshold) return 1.0f;
        const Words x = dropout_words((uint32_t)edge, (uint32_t)(h >> 2), offset, seed);
        const uint32_t lo = h & 1 ? x.w[1] : x.w[0], hi = h & 1 ? x.w[3] : x.w[2];
        return (h & 2 ? hi : lo) >= P.threshold ? P.keep_scale : 0.0f;
    }
    // sums over a quad of act(a) w for the edges e_first .. e_first + GA - 1, into LDS
    __device__ void partial_logits(const Raw (&a)[NA], int e_first) {
        wave_sync();
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            int e, q, h;
            if (!a_place(i, e_first, e, q)) continue;
            f4 wq = *(const f4*)(w + 4 * q), x;
            const int begin = begin_a(q, h), shared = MODE == kAligned ? 0 : quad_shared(begin - h * K);
#pragma unroll
            for (int j = 0; j < 4; ++j) { x[j] = j < shared ? 0.0f : act((float)a[i][j]); wq[j] = j < shared ? 0.0f : wq[j]; }          // (0 where the head has no such element)
            part[e * qa + q] = fmaf(x[3], wq[3], fmaf(x[2], wq[2], fmaf(x[1], wq[1], x[0] * wq[0])));
        }
        wave_sync();
    }
    // t of edge e_first + e and head h
    __device__ double logit(int e_first, int e, int h) const {
        const int eb = e_first + e;
        float s = 0.0f;
        for (int i = 0; i < per_a; ++i) s += part[e * qa + h * per_a + i];
        const float l = e_logit[eb];
        double x = (double)s + (double)l;
        if (P.n_buckets) { const float b = table[e_bucket[eb] * H + h]; x = b == -__builtin_inff() ? (double)b : x + (double)b; }
        if (l == -__builtin_inff()) x = -__builtin_inf();          // a masked edge takes no part whatever its features hold
        return x == __builtin_inf() ? __builtin_nan("") : x;
    }
};

// a value of another lane of the row of 16: rotations by 4 (0x124) and 8, the neighbour (0xB1), the other pair (0x4E), the mirrored half (0x141), the mirrored row (0x140)
template <int CTRL> __device__ inline float ror(float x) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true)); }

// ---- forward --------------------------------------------------------------------------------------------------------------------------------

// running softmax of one row in a lane: its quads' weighted sums, and a maximum and sum for the head of each
template <int NV> struct Row {
    f4 acc[NV]; double m[NV]; float sum[NV];
    __device__ void clear() {
        for (int j = 0; j < NV; ++j) { acc[j] = f4{0, 0, 0, 0}; m[j] = -__builtin_inf(); sum[j] = 0.0f; }
    }
    // a sum relative to x comes in (x = -inf: an empty one): factors of the old sum and of the new one
    __device__ static void weights(double& m, double x, float& w_old, float& w_new) {
        if (x == -__builtin_inf()) w_old = w_new = 1.0f;          // nothing (or NaN, which its sum holds)
        else if (x > m) { w_old = m == -__builtin_inf() ? 0.0f : exp_d(m - x); w_new = 1.0f; m = x; }
        else { w_old = 1.0f; w_new = exp_d(x - m); }
    }
    template <class X> __device__ void join(const X& x) {          // with the sums of edges behind
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float w_old, w_new;
            weights(m[j], x.m[j], w_old, w_new);
            sum[j] = fmaf(x.sum[j], w_new, sum[j] * w_old);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(x.acc[j][i], w_new, acc[j][i] * w_old);
        }
    }
    template <class X> __device__ void put(X& x) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) { x.acc[j] = acc[j]; x.m[j] = m[j]; x.sum[j] = sum[j]; }
    }
};

// Record of a row that crosses ranges, for each lane of the walk: [NV] quads, a 64-bit maximum and a sum for each.  Slot 0 of a wave holds its first row, slot 1
// its last one.  Where a row begins before the ranges of a workgroup and ends behind them, the workgroup leaves one record, in slot 0 of its first wave (the
// partial-sum buffers hold the others' for up to two quads a lane): 7 rows of 300 007 edges are joined in 11 us instead of 29
template <int NV> struct Record { f4 acc[NV]; double m[NV]; float sum[NV]; };
template <int NV> constexpr int joined_waves() { return NV <= 2 ? kWaves : 1; }

template <class T, int MODE, int NV> __device__ inline void
finish_row(const Args& P, int row, const Row<NV>& r, int lane, int qv, const int (&begin_v)[NV], const int (&head_v)[NV], T* out, float* out32, double* norm) {
    const int HD = P.heads * P.d;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (j * 64 + lane >= qv) continue;
        const float inv = r.sum[j] == 0.0f ? 0.0f : 1.0f / r.sum[j];          // (no edge takes part: 0)
        const f4 o = {r.acc[j][0] * inv, r.acc[j][1] * inv, r.acc[j][2] * inv, r.acc[j][3] * inv};
        if (norm && begin_v[j] == head_v[j] * P.d) *(d2*)(norm + 2 * ((int64_t)row * P.heads + head_v[j])) = d2{r.m[j], (double)inv};
        store_quad<T, MODE>(out + (int64_t)row * HD + begin_v[j], o, P.d);
        if (out32) store_quad<float, MODE>(out32 + (int64_t)row * HD + begin_v[j], o, P.d);
    }
}

// Read of the per-edge rows once; bandwidth bounds it, in 16 bits nearly as much the 46 vector instructions of an edge.  1.97 M edges of 64 + 240 channels:
// float32 0.57 ms (4.4 TB/s), float16 0.30 ms (4.2 TB/s), where a large copy reaches 4.8.  A logit's 16 products are summed per quad by the lanes that
// loaded it and finished by one lane for each edge and head, which also draws the dropout word: the walk then needs one share per edge and lane.  (Running
// maxima per edge and lane instead: 0.69 ms in float16.)  At lmax 3 (296 channels, 76 quads) a lane holds two quads, the second one mostly idle: 0.124 ms for
// 499 979 bfloat16 edges, 2.9 TB/s, vector instructions in half of all cycles (a fourth wave a SIMD and half the rows in flight: 0.127).
template <class T, int MODE, int NV, int GA> __global__ __launch_bounds__(256, forward_waves(NV, sizeof(T)))
void k_attn_forward(Args P, T* out, float* out32, double* norm, void* records, int64_t* rng_used) {
    typedef Wave<T, MODE, NV, GA> W;
    extern __shared__ __align__(16) char lds[];
    if (rng_used && P.threshold && blockIdx.x == 0 && threadIdx.x < 2) rng_used[threadIdx.x] = P.rng[threadIdx.x];
    const int edge_blocks = (P.n_waves + kWaves - 1) / kWaves;
    if ((int)blockIdx.x >= edge_blocks) {
        // rows without edges: 64 rows a wave
        const int H = P.heads, HD = H * P.d, lane = threadIdx.x & 63;
        const int64_t first = (((int64_t)blockIdx.x - edge_blocks) * kWaves + (threadIdx.x >> 6)) * 64, row = first + lane;
        uint64_t empty = __ballot(row < P.n_dst && P.rowptr[min(row, (int64_t)P.n_dst - 1)] == P.rowptr[min(row, (int64_t)P.n_dst - 1) + 1]);
        while (empty) {
            const int64_t r = first + __builtin_ctzll(empty);
            empty &= empty - 1;
            for (int i = lane; i < HD; i += 64) { out[r * HD + i] = (T)0.0f; if (out32) out32[r * HD + i] = 0.0f; }
            if (norm && lane < H) *(d2*)(norm + 2 * (r * H + lane)) = d2{-__builtin_inf(), 0.0};
        }
        return;
    }
    const size_t own = W::wave_bytes(P.heads) + (size_t)kBatch * P.heads * 8;
    W w(P, lds, own);
    if (w.e0 >= w.e1) { w.stage(lds); return; }
    const int lane = w.lane, H = w.H, qv = w.qv;
    // R value rows are always in flight: a row's registers are loaded again, R edges ahead, as soon as it has been added
    constexpr int R = W::RF;
    typename W::Edge edge = w.request(w.e0);
    typename W::Raw a[W::NA], v[R][NV];
    w.load_a(a, w.e0, (int)min((int64_t)kBatch, w.e1 - w.e0), 0);
#pragma unroll
    for (int i = 0; i < R; ++i) w.load_row(v[i], w.value_row(w.e0 + i));
    const int before = P.dst[max(w.e0 - 1, (int64_t)0)], behind = P.dst[min(w.e1, P.n_edges - 1)];
    w.stage(lds);
    Row<NV> r;
    r.clear();
    int cur = __builtin_amdgcn_readfirstlane(edge.dst);
    const bool open_front = w.e0 > 0 && before == cur;
    bool first_row = true;
    Record<NV>* rec = (Record<NV>*)records + ((int64_t)blockIdx.x * kWaves + w.wave) * 2 * 64 + lane;
    auto flush = [&](bool open_back) {
        if ((first_row && open_front) || open_back) {
            Record<NV> x;
            r.put(x);
            rec[first_row ? 0 : 64] = x;
        } else finish_row<T, MODE>(P, cur, r, lane, qv, w.begin_v, w.head_v, out, out32, norm);
    };
    float2* share = (float2*)w.keep;                       // [16][H] share of the piece, and that share times the dropout factor
    double* top = (double*)(w.e_bucket + kBatch);          // [16][H] logit that the shares are relative to
    for (int64_t base = w.e0; base < w.e1; base += kBatch) {
        w.begin(base, edge);
        edge = w.request(min(base + kBatch, w.e1 - 1));
        int g = 0;
        do {          // (at least once: a load from before the loop has its later ones to count, and no wait for everything in flight)
            w.partial_logits(a, g);
            // the next features are on their way while this group is summed up
            if (g + GA < kBatch && g + GA < w.n) w.load_a(a, base, w.n, g + GA);
            else if (base + kBatch < w.e1) w.load_a(a, base + kBatch, (int)min((int64_t)kBatch, w.e1 - base - kBatch), 0);
            // A "piece" is what one row has in this group.  Shares are relative to a logit that every lane of a head agrees on: the group's largest, if it is
            // at most 24 above the smallest (shares of 4e-11 and more keep full precision for any values above 1e-27), else the piece's own largest.
            // (8 heads of 32 + 77 channels, 400 000 bfloat16 edges, forward: 0.275 ms, with the pieces' own 0.291.)
            const uint32_t starts = (w.starts >> g) | 1u;
            const int live = min(GA, w.n - g);
            bool near = false;
            constexpr int NH = 64 / GA;            // lanes for each edge
            constexpr uint64_t kEdgeBits = ~(uint64_t)0 / (((uint64_t)1 << NH) - 1);          // bit NH e for every edge e
            uint64_t some = ~(uint64_t)0;          // bit NH e: edge e takes part somewhere
            bool select = true;                    // an edge may take part in one head and not in another
            if (H <= NH) {
                // one edge and head a lane: the largest and smallest logits of the group, through the wave
                const int e = lane / NH, h = lane % NH;
                const bool there = h < H;
                const double x = there ? w.logit(g, e, h) : -__builtin_inf();
                const bool in = e < live && x != -__builtin_inf();
                float most = in ? (float)x : -__builtin_inff(), least = in ? (float)x : __builtin_inff();
                if (NH <= 4) { most = fmaxf(most, ror<0x124>(most)); least = fminf(least, ror<0x124>(least)); }
                if (NH <= 8) { most = fmaxf(most, ror<0x128>(most)); least = fminf(least, ror<0x128>(least)); }
                if (NH <= 16) { most = fmaxf(most, __shfl_xor(most, 16)); least = fminf(least, __shfl_xor(least, 16)); }
                most = fmaxf(most, __shfl_xor(most, 32)); least = fminf(least, __shfl_xor(least, 32));
                // (no edge of the head takes part: -inf and +inf.  Logits beyond float's range, as two masks of its lowest value make together, leave a difference of NaN
                // or infinity: not near)
                near = __ballot(!(most == -__builtin_inff() && least == __builtin_inff()) && !(most - least <= 24.0f && fabsf(most) <= 1e6f)) == 0;
                if (near) {
                    const float p = in ? exp_d(x - (double)most) : 0.0f;
                    uint64_t all = __ballot(in || !there);
                    some = __ballot(in);
                    if (there) {
                        share[(g + e) * H + h] = float2{p, in ? p * w.dropped(base + g + e, h) : 0.0f};
                        top[(g + e) * H + h] = (double)most;
                    }
                    // The walk reads this where a piece begins.  A piece of which no edge takes part leaves its row's maximum alone: the largest logit here is another
                    // row's and may lie so far above this row's that the sum would end as zero.  Bits 0, NH, 2 NH ... of kEdgeBits: the piece's edges from e on
                    if (there && ~all) {
                        const uint32_t after = starts & ~((2u << e) - 1u);
                        const int to = min(after ? __builtin_ctz(after) : GA, GA);
                        const uint64_t piece = (kEdgeBits & ~(uint64_t)0 >> (64 - NH * (to - e))) << lane;
                        if (!(some & piece)) top[(g + e) * H + h] = -__builtin_inf();
                    }
#pragma unroll
                    for (int i = 1; i < NH; i *= 2) { some |= some >> i; all &= all >> i; }
                    select = ((some ^ all) & kEdgeBits) != 0;
                } else if (there) w.t[(g + e) * H + h] = x;
            } else {
                for (int idx = lane; idx < GA * H; idx += 64) {
                    const int e = (int)((idx * w.inv_h) >> 16), h = idx - e * H;
                    w.t[(g + e) * H + h] = w.logit(g, e, h);
                }
            }
            wave_sync();
            if (!near) {          // relative to the piece's own largest logit
#pragma unroll 1
                for (int idx = lane; idx < GA * H; idx += 64) {
                    const int e = (int)((idx * w.inv_h) >> 16), h = idx - e * H;
                    const uint32_t upto = starts & ((2u << e) - 1u), after = starts & ~((2u << e) - 1u);
                    const int from = 31 - __builtin_clz(upto), to = min(after ? __builtin_ctz(after) : GA, live);
                    double most = -__builtin_inf();
                    for (int k = from; k < to; ++k) most = __builtin_fmax(most, w.t[(g + k) * H + h]);
                    const double x = w.t[(g + e) * H + h];
                    const float p = e >= live || x == -__builtin_inf() ? 0.0f : exp_d(x - most);
                    share[(g + e) * H + h] = float2{p, e < live ? p * w.dropped(base + g + e, h) : 0.0f};
                    top[(g + e) * H + h] = most;
                }
                wave_sync();
            }
            float scale[NV];
#pragma unroll 1
            for (int s = 0; s < GA; s += R)
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int e = s + i;
                if (e < live) {
                    if ((starts >> e) & 1u) {
                        const int d = __builtin_amdgcn_readfirstlane(w.e_dst[g + e]);
                        if (d != cur) { flush(false); cur = d; first_row = false; r.clear(); }
#pragma unroll
                        for (int j = 0; j < NV; ++j) {
                            float w_old;
                            Row<NV>::weights(r.m[j], top[(g + e) * H + w.head_v[j]], w_old, scale[j]);
                            r.sum[j] *= w_old;
#pragma unroll
                            for (int c = 0; c < 4; ++c) r.acc[j][c] *= w_old;
                        }
                    }
                    if ((some >> (NH * e)) & 1)
#pragma unroll
                    for (int j = 0; j < NV; ++j) {
                        const float2 f = share[(g + e) * H + w.head_v[j]];
                        const float k = f.y * scale[j];
                        r.sum[j] = fmaf(f.x, scale[j], r.sum[j]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            // (what a head does not look at may be NaN)
                            const float x = select && f.x == 0.0f ? 0.0f : (float)v[i][j][c];
                            r.acc[j][c] = fmaf(k, x, r.acc[j][c]);
                        }
                    }
                }
                w.load_row(v[i], w.value_row(base + g + e + R));
            }
            wave_sync();
        } while ((g += GA) < kBatch && g < w.n);
    }
    constexpr int JOIN = joined_waves<NV>();
    if (JOIN > 1) {
        const int64_t first = (int64_t)blockIdx.x * kWaves * P.range, end = first + (int64_t)kWaves * P.range;
        if (first > 0 && end < P.n_edges && P.dst[first - 1] == P.dst[end]) {          // (the same for the whole workgroup) one row holds all its ranges
            static_assert(JOIN == 1 || sizeof(Record<NV>) * 64 <= W::kPart * 4, "a record fits into the partial-sum buffer");
            if (w.wave > 0) r.put(((Record<NV>*)w.part)[lane]);
            __syncthreads();
            if (w.wave > 0) return;
#pragma unroll 1
            for (int x = 1; x < kWaves; ++x) r.join(((const Record<NV>*)((const char*)w.part + x * own))[lane]);
            flush(true);
            return;
        }
    }
    flush(w.e1 < P.n_edges && behind == cur);
}

// Rows that cross ranges.  Few bytes, all waiting: 3 000 ranges 7.5 us.  A wave looks at one border between two ranges and takes a row whose first crossing that is: it joins up to 8 records by itself;
// a longer row is joined by the whole workgroup, every wave a share of the records, then the waves' results in order.
template <int NV> constexpr int merge_waves() { return 16 / NV; }
template <class T, int MODE, int NV> __global__ __launch_bounds__(1024 / NV)
void k_attn_merge(Args P, T* out, float* out32, double* norm, const void* records) {
    constexpr int WAVES = merge_waves<NV>();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qv = row_quads(P.heads, P.d);
    int begin_v[NV], head_v[NV];
    value_places(P, lane, begin_v, head_v);
    __shared__ Record<NV> share[WAVES - 1][64];
    __shared__ int long_row[WAVES], long_first[WAVES];
    const Record<NV>* rec = (const Record<NV>*)records + lane;
    Row<NV> r;
    // The records of a row that begins at edge `begin` in range w0 and ends in range `last`: those of the ranges of w0's workgroup, one for each workgroup between,
    // those of the last one's.  Item k of them, and how many:
    constexpr int JOIN = joined_waves<NV>();
    auto record = [&](int64_t k, int64_t w0, int64_t begin, int64_t last) {
        const int64_t front = min(last, w0 | (JOIN - 1)) - w0 + 1, blocks = max(last / JOIN - w0 / JOIN - 1, (int64_t)0);
        const int64_t x = k < front ? w0 + k : k < front + blocks ? (w0 / JOIN + 1 + k - front) * JOIN : last / JOIN * JOIN + k - front - blocks;
        return rec + (x * 2 + (x == w0 && begin > w0 * P.range ? 1 : 0)) * 64;
    };
    auto records_of = [&](int64_t w0, int64_t last) {
        if (last / JOIN == w0 / JOIN) return last - w0 + 1;
        return (w0 | (JOIN - 1)) - w0 + 1 + (last / JOIN - w0 / JOIN - 1) + (last & (JOIN - 1)) + 1;
    };
    auto join_records = [&](int64_t w0, int64_t begin, int64_t last, int64_t first, int64_t n, int step) {
        r.clear();
#pragma unroll 4
        for (int64_t k = first; k < n; k += step) { const Record<NV> o = *record(k, w0, begin, last); r.join(o); }
    };
    const int64_t mine = (int64_t)blockIdx.x * WAVES + wave, border = min((mine + 1) * P.range, P.n_edges - 1);
    const int before = __builtin_amdgcn_readfirstlane(P.dst[border - 1]), row = __builtin_amdgcn_readfirstlane(P.dst[border]);          // (two ranges at least)
    if (lane == 0) long_row[wave] = -1;
    if ((mine + 1) * P.range < P.n_edges && before == row) {
        const int64_t begin = P.rowptr[row], last = ((int64_t)P.rowptr[row + 1] - 1) / P.range;
        if (begin >= mine * P.range) {                              // (else an earlier border is its first)
            const int64_t n = records_of(mine, last);
            if (n <= 8) { join_records(mine, begin, last, 0, n, 1); finish_row<T, MODE>(P, row, r, lane, qv, begin_v, head_v, out, out32, norm); }
            else if (lane == 0) { long_row[wave] = row; long_first[wave] = (int)mine; }
        }
    }
    __syncthreads();
    for (int i = 0; i < WAVES; ++i) {
        const int row = long_row[i];
        if (row < 0) continue;
        const int64_t w0 = long_first[i], begin = P.rowptr[row], last = ((int64_t)P.rowptr[row + 1] - 1) / P.range;
        join_records(w0, begin, last, wave, records_of(w0, last), WAVES);
        if (wave > 0) r.put(share[wave - 1][lane]);
        __syncthreads();
        if (wave == 0) {
            for (int o = 0; o < WAVES - 1; ++o) r.join(share[o][lane]);
            finish_row<T, MODE>(P, row, r, lane, qv, begin_v, head_v, out, out32, norm);
        }
        __syncthreads();
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------------------------------

// delta[n,h] = sum_c dout out32: 16 lanes for each row and head, a quad at a time; two reads of (rows, H D).  103 000 rows of
// 240 float32 36 us, 5.5 TB/s with what the caches still hold (a wave for each row, 64 lanes for a head of 60 channels: 57 us)
template <class T> __global__ __launch_bounds__(256)
void k_attn_delta(int64_t n_pairs, int D, const T* grad, const float* out32, float* delta) {
    const int l = threadIdx.x & 15, quads = (D + 3) >> 2;
    for (int64_t pair = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); pair < n_pairs; pair += (int64_t)gridDim.x * 16) {          // (one each up to 2^27 pairs)
        const T* g = grad + pair * D; const float* o = out32 + pair * D;
        float s = 0.0f;
        for (int q = l; q < quads; q += 16) {
            const int c = quad_begin(q, D), shared = quad_shared(c);
            const typename Quad<T>::type x = D < 4 ? load_quad<T, kElements>(g, D) : load_quad<T, kHeads>(g + c, 4);
            const f4 y = D < 4 ? load_quad<float, kElements>(o, D) : load_quad<float, kHeads>(o + c, 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) s = i < shared ? s : fmaf((float)x[i], y[i], s);
        }
        s += ror<0xB1>(s); s += ror<0x4E>(s); s += ror<0x141>(s); s += ror<0x140>(s);
        if (l == 0) delta[pair] = s;
    }
}

struct BackArgs {
    const double* norm; const float* delta; const void* grad;
    void* da; void* dv; float* dl;          // any of them may be null
    float* param_rows;                      // (workgroups, H K + B H) sums of dw and dT, or null
};

// Reads the per-edge rows once and writes their gradients; the rows of dout come from the caches, read again for each edge rather than kept while a row
// lasts, so nothing waits where rows are short.  1.97 M edges of 64 + 240 float32 channels: 1.01 ms, 4.8 TB/s, the rate of a large copy; 499 979 bfloat16 edges
// of lmax 3 0.213 ms, 3.4 TB/s and 135 vector instructions an edge in 53 % of all cycles, neither unit full (with a fourth wave a SIMD, which spills, 0.25).  The dot of a value row with dout goes through LDS (a partial sum for each
// quad part), since a head's quads are not a power of two of lanes.
template <class T, int MODE, int NV, int GA> __global__ __launch_bounds__(256, backward_waves(NV, sizeof(T)))
void k_attn_backward(Args P, BackArgs B) {
    typedef Wave<T, MODE, NV, GA> W;
    constexpr int NA = W::NA, R = W::R;
    extern __shared__ __align__(16) char lds[];
    const int BH = P.n_buckets * P.heads;
    const size_t own = W::wave_bytes(P.heads) + (size_t)kBatch * P.heads * 4 + (size_t)((BH + 1) & ~1) * 4;
    W w(P, lds, (own + 15) & ~(size_t)15);
    const int lane = w.lane, H = w.H, HD = w.HD, HK = w.HK, qv = w.qv, per_head = (P.d + 3) >> 2;
    float2* share = (float2*)w.keep;                    // [16][H] probability and dropout factor
    float* weight = (float*)w.t;                        // [16][H] their product
    float* delta = weight + kBatch * H;                 // [16][H] the row's delta
    float* dt = (float*)(w.e_bucket + kBatch);          // [16][H]
    float* bins = dt + kBatch * H;                      // [buckets][H]
    for (int i = lane; i < BH; i += 64) bins[i] = 0.0f;
    int shared_v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) shared_v[j] = quad_shared(w.begin_v[j] - w.head_v[j] * P.d);
    int lanes = 0;          // 2^lanes lanes sum the dot of an edge and head
    while (lanes < 3 && (2 * R * H << lanes) <= 64) ++lanes;
    f4 dw[NA];
    int head_a[NA];          // of the lane's feature quads
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        int e, q;
        w.a_place(i, 0, e, q);
        dw[i] = f4{0, 0, 0, 0};
        w.begin_a(q, head_a[i]);
    }

    if (w.e0 >= w.e1) w.stage(lds);
    else {
        // value rows and the upper gradient at their destinations, R edges ahead; a batch's per-edge values and features one batch ahead
        // (destinations two batches ahead, so that they are there when this one asks for the next one's rows)
        auto request_dst = [&](int64_t b) { return P.dst[min(b + (lane & (kBatch - 1)), w.e1 - 1)]; };
        typename W::Edge edge = w.request(w.e0);
        int dst_next = request_dst(w.e0 + kBatch);
        typename W::Raw a[NA], a_next[NA], v[R][NV], up[R][NV];
        w.load_a(a_next, w.e0, (int)min((int64_t)kBatch, w.e1 - w.e0), 0);
        // What the rows of the next group's first 64 edges and heads keep (of all of them for up to 4 heads), on its way before the last value rows of this one:
        // loads return in order, so a load issued where it is used would wait for every row in flight.  499 979 bfloat16 edges of lmax 3 0.216 ms
        // (loads where they are used 0.253)
        struct Kept { d2 norm; float delta; } kept;
        auto request_kept = [&](int dst, int first, int n) {          // of a batch of these destinations, its edges first .. first + n - 1
            const int k = min(lane, n * H - 1), e = (int)((k * w.inv_h) >> 16);
            const int64_t at = (int64_t)__shfl(dst, first + e) * H + k - e * H;
            kept.norm = *(const d2*)(B.norm + 2 * at);
            kept.delta = B.delta[at];
        };
        // waits for it: left to the head of a loop, the wait would be for the fewest loads that any way there has issued since, which is everything in flight
        auto arrived = [](Kept& x) { double m = x.norm[0], z = x.norm[1]; asm volatile("" : "+v"(m), "+v"(z), "+v"(x.delta)); x.norm = d2{m, z}; };
        request_kept(edge.dst, 0, (int)min((int64_t)GA, w.e1 - w.e0));
#pragma unroll
        for (int i = 0; i < R; ++i) {
            w.load_row(v[i], w.value_row(w.e0 + i));
            w.load_row(up[i], (const T*)B.grad + (int64_t)__builtin_amdgcn_readlane(edge.dst, i) * HD);
        }
        w.stage(lds);
        arrived(kept);
        for (int64_t base = w.e0; base < w.e1; base += kBatch) {
            w.begin(base, edge);
            const typename W::Edge next = w.request(min(base + kBatch, w.e1 - 1));
            const int dst_after = request_dst(base + 2 * kBatch);
            wave_sync();
            int g = 0;
#pragma unroll 1
            do {
#pragma unroll
                for (int i = 0; i < NA; ++i) a[i] = a_next[i];
                if (g + GA < kBatch && g + GA < w.n) w.load_a(a_next, base, w.n, g + GA);
                else if (base + kBatch < w.e1) w.load_a(a_next, base + kBatch, (int)min((int64_t)kBatch, w.e1 - base - kBatch), 0);
                const int pairs = min(GA, w.n - g) * H;
                w.partial_logits(a, g);
                arrived(kept);
#pragma unroll 1
                for (int idx = lane; idx < pairs; idx += 64) {
                    const int e = (int)((idx * w.inv_h) >> 16), h = idx - e * H, eb = g + e;
                    const double x = w.logit(g, e, h);
                    const float p = x == -__builtin_inf() ? 0.0f : exp_d(x - kept.norm[0]) * (float)kept.norm[1], k = p == 0.0f ? 0.0f : w.dropped(base + eb, h);
                    share[eb * H + h] = float2{p, k};
                    weight[eb * H + h] = p * k;
                    delta[eb * H + h] = kept.delta;
                    if (idx + 64 < pairs) {
                        const int e = (int)(((idx + 64) * w.inv_h) >> 16);
                        const int64_t row = (int64_t)w.e_dst[g + e] * H + idx + 64 - e * H;
                        kept = Kept{*(const d2*)(B.norm + 2 * row), B.delta[row]};
                        arrived(kept);
                    }
                }
                wave_sync();
                int s = g;
#pragma unroll 1
                do {
                    if (s + R >= g + GA || s + R >= w.n) {
                        if (g + GA < kBatch && g + GA < w.n) request_kept(edge.dst, g + GA, min(GA, w.n - g - GA));
                        else if (base + kBatch < w.e1) request_kept(dst_next, 0, (int)min((int64_t)GA, w.e1 - base - kBatch));
                    }
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        if (s + i < w.n) {
#pragma unroll
                            for (int j = 0; j < NV; ++j) {
                                const int q = j * 64 + lane;
                                const float f = weight[(s + i) * H + w.head_v[j]];
                                f4 o;
                                float dot = 0.0f;
#pragma unroll
                                for (int c = 0; c < 4; ++c) {
                                    o[c] = f * (float)up[i][j][c];
                                    dot = fmaf((float)v[i][j][c], (float)up[i][j][c], dot);
                                    if (MODE == kHeads && c < 3) dot = c < shared_v[j] ? 0.0f : dot;
                                }
                                if (q < qv) {
                                    w.part[i * qv + q] = dot;
                                    if (B.dv) store_quad<T, MODE>((T*)B.dv + (base + s + i) * HD + w.begin_v[j], o, P.d);
                                }
                            }
                        }
                        const int ahead = s + i + R, dst = ahead < kBatch ? __builtin_amdgcn_readlane(edge.dst, ahead) : __builtin_amdgcn_readlane(dst_next, ahead - kBatch);
                        w.load_row(v[i], w.value_row(base + ahead));
                        w.load_row(up[i], (const T*)B.grad + (int64_t)dst * HD);
                    }
                    wave_sync();
                    const int last = min(s + R, w.n) - s;          // edges of this part
                    auto write_dt = [&](int i, int h, float dot) {
                        const float2 f = share[(s + i) * H + h];
                        // (a masked edge's value may be NaN)
                        dt[(s + i) * H + h] = f.x == 0.0f ? 0.0f : f.x * ((f.y == 0.0f ? 0.0f : f.y * dot) - delta[(s + i) * H + h]);
                    };
                    for (int k = lane >> lanes; k < last * H; k += 64 >> lanes) {
                        const int i = (int)((k * w.inv_h) >> 16), h = k - i * H, l = lane & ((1 << lanes) - 1);
                        float dot = 0.0f;
                        for (int c = l; c < per_head; c += 1 << lanes) dot += w.part[i * qv + h * per_head + c];
                        if (lanes > 0) dot += ror<0xB1>(dot);
                        if (lanes > 1) dot += ror<0x4E>(dot);
                        if (lanes > 2) dot += ror<0x141>(dot);
                        if (l == 0) write_dt(i, h, dot);
                    }
                    wave_sync();
                } while ((s += R) < g + GA && s < w.n);
                if (B.dl && lane < GA && g + lane < w.n) {
                    float s = 0.0f;
                    for (int h = 0; h < H; ++h) s += dt[(g + lane) * H + h];
                    B.dl[base + g + lane] = s;
                }
#pragma unroll
                for (int i = 0; i < NA; ++i) {
                    int e, q;
                    if (!w.a_place(i, g, e, q)) continue;
                    const f4 wq = *(const f4*)(w.w + 4 * q);
                    const float f = dt[(g + e) * H + head_a[i]];
                    f4 o;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float x = (float)a[i][j], sg = sigmoid(x);
                        const float slope = kActNorm * fmaf(0.8f * sg, fmaf(x, 1.0f - sg, 1.0f), 0.2f);
                        o[j] = f == 0.0f ? 0.0f : f * wq[j] * slope;
                        dw[i][j] = f == 0.0f ? dw[i][j] : fmaf(f, kActNorm * x * fmaf(0.8f, sg, 0.2f), dw[i][j]);
                    }
                    int h;
                    const int c = w.begin_a(q, h);
                    if (B.da) {
                        T* p = (T*)B.da + (base + g + e) * HK + c;
                        if (MODE == kAligned) store_quad<T, kAligned>(p, o, 4);
                        else if (P.k < 4) store_quad<T, kElements>(p, o, P.k);
                        else store_quad<T, kHeads>(p, o, 4);
                    }
                }
                if (BH && B.param_rows && lane < H)          // in the edges' order: lane h alone adds to the sums of its head
                    for (int e = 0; e < GA && g + e < w.n; ++e) bins[w.e_bucket[g + e] * H + lane] += dt[(g + e) * H + lane];
                wave_sync();
            } while ((g += GA) < kBatch && g < w.n);
            edge = typename W::Edge{dst_next, next.logit, next.length};
            dst_next = dst_after;
        }
    }
    if (!B.param_rows) return;
    // the workgroup's sums: each wave folds its feature quads by place, then the four waves are added in order
    wave_sync();
#pragma unroll
    for (int i = 0; i < NA; ++i) *(f4*)(w.part + 4 * (i * 64 + lane)) = dw[i];
    __syncthreads();
    const size_t stride = (own + 15) & ~(size_t)15;
    for (int c = threadIdx.x; c < HK; c += 256) {
        int at = c;          // its place among the feature quads' elements
        if (MODE != kAligned) { const int h = c / P.k, x = c - h * P.k; at = 4 * (h * w.per_a + (x >> 2)) + x - quad_begin(x >> 2, P.k); }
        float s = 0.0f;
        for (int x = 0; x < kWaves; ++x) {
            const float* part = (const float*)((const char*)w.part + ((ptrdiff_t)x - w.wave) * (ptrdiff_t)stride);
            for (int i = at >> 2; i < GA * w.qa; i += w.qa) s += part[4 * i + (at & 3)];
        }
        B.param_rows[(size_t)blockIdx.x * (HK + BH) + c] = s;
    }
    for (int c = threadIdx.x; c < BH; c += 256) {
        float s = 0.0f;
        for (int x = 0; x < kWaves; ++x) s += *(const float*)((const char*)(bins + c) + ((ptrdiff_t)x - w.wave) * (ptrdiff_t)stride);
        B.param_rows[(size_t)blockIdx.x * (HK + BH) + HK + c] = s;
    }
}

// column sums of (rows, columns) in 64 bits, in a fixed order: 16 columns a workgroup; the first n_first go to `first`, the rest to `second`
static __global__ __launch_bounds__(1024) void k_column_sums(const float* x, int rows, int columns, float* first, int n_first, float* second) {
    __shared__ double share[64][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), r0 = threadIdx.x >> 4;
    const float* m = x + c;
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
    const float v = (float)share[0][threadIdx.x & 15];
    if (c < n_first) { if (first) first[c] = v; }
    else if (second) second[c - n_first] = v;
}

// ---- the sorted edge list -------------------------------------------------------------------------------------------------------------------

// 32-bit copy of the destinations, first edge of each row (rowptr[n_dst] = n_edges); *bad is set where the list is not sorted or leaves [0, n_dst)
static __global__ __launch_bounds__(256) void k_edge_segments(const int64_t* edge_dst, int64_t n_edges, int n_dst, int* dst, int* rowptr, int* bad) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n_edges) {
        const int64_t d = edge_dst[i];
        if (d < 0 || d >= n_dst || (i > 0 && edge_dst[i - 1] > d)) *bad = 1;
        dst[i] = (int)min(max(d, (int64_t)0), (int64_t)n_dst - 1);
    }
    if (i <= n_dst) {
        int64_t lo = 0, hi = n_edges;
        while (lo < hi) { const int64_t mid = (lo + hi) >> 1; if (edge_dst[mid] < i) lo = mid + 1; else hi = mid; }
        rowptr[i] = (int)lo;
    }
}

}  // namespace attn
}  // namespace dedf
