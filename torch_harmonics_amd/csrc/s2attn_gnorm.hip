// Group norm with an activation on channels-last tensors [B, nlat, nlon, C], forward and backward; statistics over the grid and the channels of
// a group, optionally weighted by the quadrature of the latitude rings.
//
//   mean = sum w x / W,  var = sum w (x - mean)^2 / W,  W = sum of w over the points and channels of a group  (w = 1 without weights)
//   z = (x - mean) r gamma + beta,  r = 1 / sqrt(var + eps),  y = act(z)
//   dz = dy act'(z);  per batch entry and channel  s1 = sum dz,  s2 = sum dz xhat,  xhat = (x - mean) r
//   dbeta = sum over the batch of s1,  dgamma = of s2;  A = sum over a group's channels of gamma s1,  E = of gamma s2
//   dx = r (gamma dz - (w / W) (A + xhat E))
// so one pass over x (and dy) for the sums and one for the result; bound by memory.
//
// Sums: a thread's values as (weight, mean, squared deviations) of chunks that it holds in registers, merged pairwise by the exact update for
// two samples' moments (Chan, Golub, LeVeque): no value is squared before a mean close to it is taken off, so an offset or a first
// value far from the others costs nothing.  All sums run in an order that the sizes alone fix: results are the same in every run.

#include "s2attn_internal.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

namespace s2norm {

struct bf16_t {
    unsigned short bits;
};
struct f16_t {
    _Float16 v;
};
__device__ inline float widen(float x) { return x; }
__device__ inline float widen(bf16_t x) { return __uint_as_float((unsigned)x.bits << 16); }
__device__ inline float widen(f16_t x) { return (float)x.v; }
__device__ inline void narrow(float &d, float x) { d = x; }
__device__ inline void narrow(bf16_t &d, float x) { d.bits = __builtin_bit_cast(unsigned short, (__bf16)x); }
__device__ inline void narrow(f16_t &d, float x) { d.v = (_Float16)x; }

// V neighboring channels of a point
template <typename T, int V> struct alignas(sizeof(T) * V) Piece {
    T v[V];
};
template <typename T, int V> __device__ inline void load(float (&x)[V], const T *p)
{
    const Piece<T, V> r = *reinterpret_cast<const Piece<T, V> *>(p);
#pragma unroll
    for (int i = 0; i < V; i++) x[i] = widen(r.v[i]);
}
template <typename T, int V> __device__ inline void store(T *p, const float (&x)[V])
{
    Piece<T, V> r;
#pragma unroll
    for (int i = 0; i < V; i++) narrow(r.v[i], x[i]);
    *reinterpret_cast<Piece<T, V> *>(p) = r;
}
__device__ inline float param(const void *p, int i, int dtype, float absent)
{
    if (!p) return absent;
    if (dtype == S2ATTN_F32) return static_cast<const float *>(p)[i];
    if (dtype == S2ATTN_BF16) return widen(static_cast<const bf16_t *>(p)[i]);
    return widen(static_cast<const f16_t *>(p)[i]);
}
__device__ inline void store_param(void *p, int i, int dtype, float x)
{
    if (!p) return;
    if (dtype == S2ATTN_F32)
        static_cast<float *>(p)[i] = x;
    else if (dtype == S2ATTN_BF16)
        narrow(static_cast<bf16_t *>(p)[i], x);
    else
        narrow(static_cast<f16_t *>(p)[i], x);
}

constexpr float LOG2E = 1.4426950408889634f;
constexpr float INV_SQRT_2PI = 0.39894228040143268f;

__device__ inline float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * z)); }
// The normal distribution function and e = exp(-z^2 / 2).  Its tail at a = |z| is e g(a), g smooth: a polynomial of degree 8 in t = 1 / (1 + 0.3 a),
// fitted to erfcx over 0 <= a < 14.5 with the least largest relative error, 2^-24; evaluated in fp32 the result is off by 1.9e-7.  e is what the
// slope needs as well.  (erff evaluates two branches and an exponential of its own: the sums of the backward pass over 361x720x256 in fp32 took 146 us
// with it, 136 with this.)
struct Normal {
    float below, e;
};
__device__ inline Normal normal(float z)
{
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, fabsf(z), 1.f)), e = __builtin_amdgcn_exp2f(-0.5f * LOG2E * z * z);
    float g = 0.038407109677791595f;
    g = fmaf(g, t, -0.16930623352527618f);
    g = fmaf(g, t, 0.22894950211048126f);
    g = fmaf(g, t, -0.07683734595775604f);
    g = fmaf(g, t, 0.1427638679742813f);
    g = fmaf(g, t, 0.09458639472723007f);
    g = fmaf(g, t, 0.12194514274597168f);
    g = fmaf(g, t, 0.11948422342538834f);
    g = fmaf(g, t, 7.371657375188079e-06f);
    g *= e;
    return {z < 0.f ? g : 1.f - g, e};
}
template <int ACT> __device__ inline float act(float z)
{
    if (ACT == S2ATTN_ACT_RELU) return z < 0.f ? 0.f : z; // (NaN stays)
    if (ACT == S2ATTN_ACT_SILU) return z * sigmoid(z);
    if (ACT == S2ATTN_ACT_GELU) return z * normal(z).below;
    return z;
}
template <int ACT> __device__ inline float slope(float z)
{
    if (ACT == S2ATTN_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    if (ACT == S2ATTN_ACT_SILU) {
        const float s = sigmoid(z);
        return s * fmaf(z, 1.f - s, 1.f);
    }
    if (ACT == S2ATTN_ACT_GELU) {
        const Normal n = normal(z);
        return fmaf(z * INV_SQRT_2PI, n.e, n.below);
    }
    return 1.f;
}

// weight, mean, sum of weighted squared deviations
struct Moments {
    float w, mean, m2;
};
__device__ inline Moments merge(const Moments &a, const Moments &b)
{
    const float w = a.w + b.w, f = w > 0.f ? b.w / w : 0.f, d = b.mean - a.mean;
    return {w, fmaf(d, f, a.mean), a.m2 + b.m2 + d * d * a.w * f};
}
__device__ inline Moments merge_lanes(Moments m, int lanes)
{
    for (int o = lanes / 2; o; o >>= 1) {
        const Moments b = {__shfl_xor(m.w, o), __shfl_xor(m.mean, o), __shfl_xor(m.m2, o)};
        // both lanes of a pair compute the same bits: the lower one's values come first
        m = (threadIdx.x & o) ? merge(b, m) : merge(m, b);
    }
    return m;
}

constexpr int NT = 256; // threads
constexpr int UN = 4;   // rows in flight per thread (those past a slab's end are its last one again: a load under a condition waits its turn)

struct GArgs {
    const void *x, *dy, *weight, *bias;
    void *y, *dx, *dweight, *dbias;
    const float *ring; // weights of the latitude rings, or null
    float *stats;      // [B][groups][3]: mean, 1 / std, 1 / W
    Moments *part;     // forward: [B][slabs][groups]
    float *sums;       // backward: [B][slabs][C][2] partial (s1, s2), then [B][C][2]
    float *sums_all;
    int64_t ldx, lddy; // elements between two points of x and dy
    int64_t N;         // points
    int nlon, C, G, Cg, B;
    int pdtype, slabs;
    int pieces, pieces_pb, rows_pb; // pieces of V channels per point; of them per workgroup; rows a workgroup takes at a time
    int64_t slab_rows;
    float eps;
    int act;
};

// A thread's place: piece (of V channels) and row offset inside a workgroup that covers pieces_pb pieces x rows_pb rows at a time.
struct Place {
    int piece, row;
    bool on;
};
__device__ inline Place place(const GArgs &a, int chunk)
{
    Place p;
    p.row = threadIdx.x / a.pieces_pb;
    p.piece = chunk * a.pieces_pb + threadIdx.x % a.pieces_pb;
    p.on = p.row < a.rows_pb && p.piece < a.pieces;
    return p;
}
// ring weight of a row, rows walked in steps
struct RingWalk {
    int lat, lon;
    __device__ inline void start(int64_t row, int nlon) { lat = (int)(row / nlon), lon = (int)(row - (int64_t)lat * nlon); }
    __device__ inline void step(int rows, int nlon)
    {
        lon += rows;
        while (lon >= nlon) lon -= nlon, lat++;
    }
    __device__ inline void back(int rows, int nlon)
    {
        lon -= rows;
        while (lon < 0) lon += nlon, lat--;
    }
};
// The second pass over the data walks a slab from its end: the rows that the first one read last are still in the last-level cache, and those
// that the forward's second pass read last are the ones that the backward's first begins with.  From their starts on / from their ends on, the second
// passes take 200 / 194 us (721x1440x256 bf16, forward) and 160 / 147 us (361x720x256 fp32, backward), the backward's first 136 / 118 us.
__device__ inline int64_t last_rows(const GArgs &a, int64_t first, int64_t last)
{
    const int64_t by = (int64_t)UN * a.rows_pb;
    return first + max((int64_t)0, last - first - 1) / by * by;
}

// ---- forward: moments of every (slab of rows, group) -------------------------------------------------------------------------
// V divides the channels of a group, so a piece has one group.
template <typename T, int V, bool RING> __global__ __launch_bounds__(NT) void stats_kernel(const GArgs a)
{
    __shared__ Moments red[NT];
    const int slab = blockIdx.x % a.slabs, chunk = (blockIdx.x / a.slabs) % ((a.pieces + a.pieces_pb - 1) / a.pieces_pb);
    const int b = blockIdx.x / a.slabs / ((a.pieces + a.pieces_pb - 1) / a.pieces_pb);
    const Place p = place(a, chunk);
    const int64_t first = (int64_t)slab * a.slab_rows, last = min(a.N, first + a.slab_rows);
    Moments m = {0.f, 0.f, 0.f};
    if (p.on) {
        const T *x = static_cast<const T *>(a.x) + (int64_t)b * a.N * a.ldx + (int64_t)p.piece * V;
        RingWalk ring;
        if (RING) ring.start(first + p.row, a.nlon);
        for (int64_t n = first + p.row; n < last; n += (int64_t)UN * a.rows_pb) {
            float v[UN][V], w[UN];
#pragma unroll
            for (int u = 0; u < UN; u++) {
                const int64_t r = n + (int64_t)u * a.rows_pb;
                load<T, V>(v[u], x + min(r, last - 1) * a.ldx);
                w[u] = r < last ? 1.f : 0.f;
                if (RING && r < last) w[u] = a.ring[ring.lat];
                if (RING) ring.step(a.rows_pb, a.nlon);
            }
            float s = 0.f, q = 0.f, sw = 0.f;
#pragma unroll
            for (int u = 0; u < UN; u++) {
                float t = 0.f;
#pragma unroll
                for (int i = 0; i < V; i++) t += v[u][i];
                if (w[u] != 0.f) s = fmaf(w[u], t, s); // (what weighs nothing is not looked at, also where it is not finite)
                sw += w[u];
            }
            sw *= V;
            const float mean = sw > 0.f ? s / sw : 0.f;
#pragma unroll
            for (int u = 0; u < UN; u++) {
                float t = 0.f;
#pragma unroll
                for (int i = 0; i < V; i++) t = fmaf(v[u][i] - mean, v[u][i] - mean, t);
                if (w[u] != 0.f) q = fmaf(w[u], t, q);
            }
            m = merge(m, {sw, mean, q});
        }
    }
    red[threadIdx.x] = m;
    __syncthreads();
    // groups that start in this chunk's channels share them with no other chunk (pieces_pb holds whole groups, or one group spans chunks)
    const int c0 = chunk * a.pieces_pb * V, c1 = min(a.C, c0 + a.pieces_pb * V);
    const int g0 = c0 / a.Cg, ng = (c1 + a.Cg - 1) / a.Cg - g0;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int i = wave; i < ng; i += NT / 64) {
        const int lo = max(c0, (g0 + i) * a.Cg), hi = min(c1, (g0 + i + 1) * a.Cg);
        const int np = (hi - lo) / V, p0 = (lo - c0) / V, n = np * a.rows_pb;
        Moments t = {0.f, 0.f, 0.f};
        for (int e = lane; e < n; e += 64) t = merge(t, red[(e / np) * a.pieces_pb + p0 + e % np]);
        t = merge_lanes(t, 64);
        if (lane == 0) a.part[((int64_t)(chunk * a.B + b) * a.slabs + slab) * a.G + g0 + i] = t;
    }
}

// mean, 1 / std, 1 / W of a (batch entry, group) from its slabs (and chunks, where a group spans several)
__global__ __launch_bounds__(NT) void stats_finish_kernel(const GArgs a, int chunk_channels)
{
    __shared__ Moments red[NT / 64];
    const int b = blockIdx.x / a.G, g = blockIdx.x % a.G;
    Moments m = {0.f, 0.f, 0.f};
    for (int chunk = g * a.Cg / chunk_channels; chunk <= ((g + 1) * a.Cg - 1) / chunk_channels; chunk++)
        for (int s = threadIdx.x; s < a.slabs; s += NT) m = merge(m, a.part[((int64_t)(chunk * a.B + b) * a.slabs + s) * a.G + g]);
    m = merge_lanes(m, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        m = red[0];
        for (int i = 1; i < NT / 64; i++) m = merge(m, red[i]);
        float *st = a.stats + 3 * (int64_t)blockIdx.x;
        const float var = m.w > 0.f ? m.m2 / m.w : 0.f;
        st[0] = m.mean;
        st[1] = 1.f / sqrtf(var + a.eps);
        st[2] = m.w > 0.f ? 1.f / m.w : 0.f;
    }
}

template <typename T, int V, int ACT> __global__ __launch_bounds__(NT) void apply_kernel(const GArgs a)
{
    const int nchunk = (a.pieces + a.pieces_pb - 1) / a.pieces_pb;
    const int slab = blockIdx.x % a.slabs, chunk = (blockIdx.x / a.slabs) % nchunk, b = blockIdx.x / a.slabs / nchunk;
    const Place p = place(a, chunk);
    const int64_t first = (int64_t)slab * a.slab_rows, last = min(a.N, first + a.slab_rows);
    if (!p.on || first >= last) return;
    const float *st = a.stats + 3 * ((int64_t)b * a.G + p.piece * V / a.Cg);
    const float mean = st[0], r = st[1];
    float ga[V], be[V];
#pragma unroll
    for (int i = 0; i < V; i++) ga[i] = r * param(a.weight, p.piece * V + i, a.pdtype, 1.f), be[i] = param(a.bias, p.piece * V + i, a.pdtype, 0.f);
    const T *x = static_cast<const T *>(a.x) + (int64_t)b * a.N * a.ldx + (int64_t)p.piece * V;
    T *y = static_cast<T *>(a.y) + (int64_t)b * a.N * a.C + (int64_t)p.piece * V;
    for (int64_t n = last_rows(a, first, last) + p.row; n >= first; n -= (int64_t)UN * a.rows_pb) {
        float v[UN][V];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            load<T, V>(v[u], x + min(n + (int64_t)u * a.rows_pb, last - 1) * a.ldx);
        }
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int64_t row = n + (int64_t)u * a.rows_pb;
            if (row < last) {
#pragma unroll
                for (int i = 0; i < V; i++) v[u][i] = act<ACT>(fmaf(v[u][i] - mean, ga[i], be[i]));
                store<T, V>(y + row * a.C, v[u]);
            }
        }
    }
}

// ---- backward: per batch entry, slab and channel, s1 = sum dz and s2 = sum dz xhat ----------------------------------------------
template <typename T, int V, int ACT> __global__ __launch_bounds__(NT) void grad_sums_kernel(const GArgs a)
{
    extern __shared__ float red[]; // [rows_pb][pieces_pb * V][2]
    const int nchunk = (a.pieces + a.pieces_pb - 1) / a.pieces_pb;
    const int slab = blockIdx.x % a.slabs, chunk = (blockIdx.x / a.slabs) % nchunk, b = blockIdx.x / a.slabs / nchunk;
    const Place p = place(a, chunk);
    float s1[V] = {}, s2[V] = {};
    if (p.on) {
        const float *st = a.stats + 3 * ((int64_t)b * a.G + p.piece * V / a.Cg);
        const float mean = st[0], r = st[1];
        float ga[V], be[V];
#pragma unroll
        for (int i = 0; i < V; i++) ga[i] = param(a.weight, p.piece * V + i, a.pdtype, 1.f), be[i] = param(a.bias, p.piece * V + i, a.pdtype, 0.f);
        const T *x = static_cast<const T *>(a.x) + (int64_t)b * a.N * a.ldx + (int64_t)p.piece * V;
        const T *dy = static_cast<const T *>(a.dy) + (int64_t)b * a.N * a.lddy + (int64_t)p.piece * V;
        const int64_t first = (int64_t)slab * a.slab_rows, last = min(a.N, first + a.slab_rows);
        for (int64_t n = first + p.row; n < last; n += (int64_t)UN * a.rows_pb) {
            float v[UN][V], d[UN][V];
#pragma unroll
            for (int u = 0; u < UN; u++) {
                const int64_t row = min(n + (int64_t)u * a.rows_pb, last - 1);
                load<T, V>(v[u], x + row * a.ldx), load<T, V>(d[u], dy + row * a.lddy);
            }
#pragma unroll
            for (int u = 0; u < UN; u++) {
                if (n + (int64_t)u * a.rows_pb < last) {
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float xh = (v[u][i] - mean) * r, dz = d[u][i] * slope<ACT>(fmaf(xh, ga[i], be[i]));
                        s1[i] += dz;
                        s2[i] = fmaf(dz, xh, s2[i]);
                    }
                }
            }
        }
    }
    const int width = a.pieces_pb * V;
    if (p.row < a.rows_pb) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            float *o = red + 2 * (p.row * width + (threadIdx.x % a.pieces_pb) * V + i);
            o[0] = s1[i], o[1] = s2[i];
        }
    }
    __syncthreads();
    float *out = a.sums + 2 * (((int64_t)b * a.slabs + slab) * a.C + (int64_t)chunk * width);
    const int n = 2 * min(width, a.C - chunk * width);
    for (int e = threadIdx.x; e < n; e += NT) {
        float t = 0.f;
        for (int row = 0; row < a.rows_pb; row++) t += red[2 * row * width + e];
        out[e] = t;
    }
}

// sums_all[b][c] = (s1, s2) over the slabs, and dbeta, dgamma over the batch: eight channels (sixteen numbers) per workgroup.  A thread adds up
// every 64th slab, four at a time: a load that waits for the one before it costs a microsecond (1024 slabs by sixteen threads, one after
// another: 21 us, this: 4).
constexpr int NTF = 1024;
__global__ __launch_bounds__(NTF) void grad_finish_kernel(const GArgs a)
{
    __shared__ double red[NTF];
    const int j = threadIdx.x % 16, lane = threadIdx.x / 16, e = 16 * blockIdx.x + j;
    const bool on = e < 2 * a.C;
    double total = 0.0;
    for (int b = 0; b < a.B; b++) {
        double t = 0.0;
        if (on) {
            const float *sums = a.sums + 2 * (int64_t)b * a.slabs * a.C + e;
            for (int s = lane; s < a.slabs; s += 4 * (NTF / 16)) {
                float x[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int r = s + u * (NTF / 16);
                    x[u] = r < a.slabs ? sums[2 * (int64_t)r * a.C] : 0.f;
                }
                t += ((double)x[0] + x[1]) + ((double)x[2] + x[3]);
            }
        }
        red[threadIdx.x] = t;
        __syncthreads();
        if (lane < 4) { // (all in the first wavefront)
            t = 0.0;
            for (int i = lane; i < NTF / 16; i += 4) t += red[16 * i + j];
            t += __shfl_xor(t, 16);
            t += __shfl_xor(t, 32);
            if (on && lane == 0) a.sums_all[2 * (int64_t)b * a.C + e] = (float)t;
            total += t;
        }
        __syncthreads();
    }
    if (lane == 0 && on) store_param(e % 2 ? a.dweight : a.dbias, e / 2, a.pdtype, (float)total);
}

template <typename T, int V, int ACT, bool RING> __global__ __launch_bounds__(NT) void grad_apply_kernel(const GArgs a)
{
    const int nchunk = (a.pieces + a.pieces_pb - 1) / a.pieces_pb;
    const int slab = blockIdx.x % a.slabs, chunk = (blockIdx.x / a.slabs) % nchunk, b = blockIdx.x / a.slabs / nchunk;
    const Place p = place(a, chunk);
    const int64_t first = (int64_t)slab * a.slab_rows, last = min(a.N, first + a.slab_rows);
    if (!p.on || first >= last) return;
    const int g = p.piece * V / a.Cg;
    const float *st = a.stats + 3 * ((int64_t)b * a.G + g);
    const float mean = st[0], r = st[1], inv_w = st[2];
    float A = 0.f, E = 0.f;
    for (int c = g * a.Cg; c < (g + 1) * a.Cg; c++) {
        const float gamma = param(a.weight, c, a.pdtype, 1.f);
        A = fmaf(gamma, a.sums_all[2 * ((int64_t)b * a.C + c)], A);
        E = fmaf(gamma, a.sums_all[2 * ((int64_t)b * a.C + c) + 1], E);
    }
    A *= inv_w, E *= inv_w;
    float ga[V], be[V];
#pragma unroll
    for (int i = 0; i < V; i++) ga[i] = param(a.weight, p.piece * V + i, a.pdtype, 1.f), be[i] = param(a.bias, p.piece * V + i, a.pdtype, 0.f);
    const T *x = static_cast<const T *>(a.x) + (int64_t)b * a.N * a.ldx + (int64_t)p.piece * V;
    const T *dy = static_cast<const T *>(a.dy) + (int64_t)b * a.N * a.lddy + (int64_t)p.piece * V;
    T *dx = static_cast<T *>(a.dx) + (int64_t)b * a.N * a.C + (int64_t)p.piece * V;
    const int64_t end = last_rows(a, first, last) + p.row;
    RingWalk ring;
    if (RING) ring.start(end, a.nlon);
    for (int64_t n = end; n >= first; n -= (int64_t)UN * a.rows_pb) {
        float v[UN][V], d[UN][V], w[UN];
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int64_t row = n + (int64_t)u * a.rows_pb;
            w[u] = 1.f;
            if (RING && row < last) w[u] = a.ring[ring.lat];
            if (RING) ring.step(a.rows_pb, a.nlon);
            load<T, V>(v[u], x + min(row, last - 1) * a.ldx), load<T, V>(d[u], dy + min(row, last - 1) * a.lddy);
        }
        if (RING) ring.back(2 * UN * a.rows_pb, a.nlon);
#pragma unroll
        for (int u = 0; u < UN; u++) {
            const int64_t row = n + (int64_t)u * a.rows_pb;
            if (row < last) {
                const float wa = w[u] * A, we = w[u] * E;
#pragma unroll
                for (int i = 0; i < V; i++) {
                    const float xh = (v[u][i] - mean) * r, dz = d[u][i] * slope<ACT>(fmaf(xh, ga[i], be[i]));
                    v[u][i] = r * (fmaf(ga[i], dz, -wa) - xh * we);
                }
                store<T, V>(dx + row * a.C, v[u]);
            }
        }
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------
bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int esize(int dtype) { return dtype == S2ATTN_F32 ? 4 : 2; }

int check(const s2attn_gnorm *n)
{
    if (!n) return s2attn_fail(S2ATTN_E_INVALID, "group norm: null arguments");
    if (n->batch < 1 || n->nlat < 1 || n->nlon < 1 || n->channels < 1) return s2attn_fail(S2ATTN_E_INVALID, "group norm: batch, grid extents and channels must be positive");
    if (n->groups < 1 || n->channels % n->groups != 0) return s2attn_fail(S2ATTN_E_INVALID, "group norm: %d groups do not divide %d channels", n->groups, n->channels);
    if (n->dtype != S2ATTN_F32 && n->dtype != S2ATTN_BF16 && n->dtype != S2ATTN_F16) return s2attn_fail(S2ATTN_E_INVALID, "group norm: unknown dtype code %d", n->dtype);
    if (n->param_dtype != S2ATTN_F32 && n->param_dtype != S2ATTN_BF16 && n->param_dtype != S2ATTN_F16)
        return s2attn_fail(S2ATTN_E_INVALID, "group norm: unknown dtype code %d of the parameters", n->param_dtype);
    if (n->activation < S2ATTN_ACT_NONE || n->activation > S2ATTN_ACT_GELU) return s2attn_fail(S2ATTN_E_INVALID, "group norm: unknown activation %d", n->activation);
    if (!(n->eps >= 0.f)) return s2attn_fail(S2ATTN_E_INVALID, "group norm: eps must not be negative");
    if ((n->ld_x && n->ld_x < n->channels) || (n->ld_dy && n->ld_dy < n->channels)) return s2attn_fail(S2ATTN_E_INVALID, "group norm: point stride smaller than the channels");
    if ((int64_t)n->nlat * n->nlon > 0x7fffffffL) return s2attn_fail(S2ATTN_E_UNSUPPORTED, "group norm: grids of more than 2^31 points");
    if (n->batch > (1 << 22) || (int64_t)n->batch * n->groups > (1 << 24)) return s2attn_fail(S2ATTN_E_UNSUPPORTED, "group norm: more than 2^24 statistics");
    return S2ATTN_OK;
}

// Slabs of rows per batch entry whose sums are kept apart: enough workgroups to fill the GPU, few enough to add up quickly.
int slabs_of(const s2attn_gnorm *n)
{
    const int64_t rows = (int64_t)n->nlat * n->nlon;
    return (int)std::max<int64_t>(1, std::min<int64_t>(1024 / std::min(n->batch, 1024), rows / 16));
}

// channels a thread takes at a time: up to 16 bytes, a divisor of a group's channels, as the addresses allow
int width_of(const s2attn_gnorm *n, std::initializer_list<const void *> ptrs)
{
    const int es = esize(n->dtype), cg = n->channels / n->groups;
    for (int v = 16 / es; v > 1; v /= 2) {
        if (v == 2) break; // (pairs gain nothing over single channels worth their kernels)
        bool ok = cg % v == 0 && (n->ld_x ? n->ld_x : n->channels) % v == 0 && (n->ld_dy ? n->ld_dy : n->channels) % v == 0;
        for (const void *p : ptrs) ok = ok && aligned(p, (size_t)v * es);
        if (ok) return v;
    }
    return 1;
}

GArgs args_of(const s2attn_gnorm *n, int V, int slabs)
{
    GArgs a = {};
    a.x = n->x, a.dy = n->dy, a.weight = n->weight, a.bias = n->bias;
    a.y = n->y, a.dx = n->dx, a.dweight = n->dweight, a.dbias = n->dbias;
    a.ring = n->ring_weights, a.stats = n->stats;
    a.N = (int64_t)n->nlat * n->nlon, a.nlon = n->nlon, a.C = n->channels, a.G = n->groups, a.Cg = n->channels / n->groups, a.B = n->batch;
    a.ldx = n->ld_x ? n->ld_x : n->channels, a.lddy = n->ld_dy ? n->ld_dy : n->channels;
    a.pdtype = n->param_dtype, a.eps = n->eps, a.act = n->activation;
    a.pieces = n->channels / V;
    a.pieces_pb = std::min(a.pieces, NT);
    a.rows_pb = NT / a.pieces_pb;
    a.slabs = slabs;
    a.slab_rows = (a.N + slabs - 1) / slabs;
    return a;
}
int chunks_of(const GArgs &a) { return (a.pieces + a.pieces_pb - 1) / a.pieces_pb; }

int launched(const char *what)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? S2ATTN_OK : s2attn_fail(S2ATTN_E_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

template <typename T, int V> int forward_v(const s2attn_gnorm *n, hipStream_t s)
{
    GArgs a = args_of(n, V, slabs_of(n));
    a.part = static_cast<Moments *>(n->workspace);
    const int64_t blocks = (int64_t)a.slabs * chunks_of(a) * a.B;
    if (blocks >= (1 << 24)) return s2attn_fail(S2ATTN_E_UNSUPPORTED, "group norm needs %lld workgroups, more than one grid holds", (long long)blocks);
    const unsigned nb = (unsigned)blocks;
    if (a.ring)
        stats_kernel<T, V, true><<<nb, NT, 0, s>>>(a);
    else
        stats_kernel<T, V, false><<<nb, NT, 0, s>>>(a);
    stats_finish_kernel<<<a.B * a.G, NT, 0, s>>>(a, a.pieces_pb * V);
    switch (a.act) {
    case S2ATTN_ACT_NONE: apply_kernel<T, V, S2ATTN_ACT_NONE><<<nb, NT, 0, s>>>(a); break;
    case S2ATTN_ACT_RELU: apply_kernel<T, V, S2ATTN_ACT_RELU><<<nb, NT, 0, s>>>(a); break;
    case S2ATTN_ACT_SILU: apply_kernel<T, V, S2ATTN_ACT_SILU><<<nb, NT, 0, s>>>(a); break;
    case S2ATTN_ACT_GELU: apply_kernel<T, V, S2ATTN_ACT_GELU><<<nb, NT, 0, s>>>(a); break;
    }
    return launched("group norm");
}

template <typename T, int V, int ACT> void backward_act(const GArgs &a, unsigned nb, hipStream_t s)
{
    grad_sums_kernel<T, V, ACT><<<nb, NT, (size_t)a.rows_pb * a.pieces_pb * V * 2 * sizeof(float), s>>>(a);
    grad_finish_kernel<<<(2 * a.C + 15) / 16, NTF, 0, s>>>(a);
    if (!a.dx) return;
    if (a.ring)
        grad_apply_kernel<T, V, ACT, true><<<nb, NT, 0, s>>>(a);
    else
        grad_apply_kernel<T, V, ACT, false><<<nb, NT, 0, s>>>(a);
}

template <typename T, int V> int backward_v(const s2attn_gnorm *n, hipStream_t s)
{
    GArgs a = args_of(n, V, slabs_of(n));
    a.sums_all = static_cast<float *>(n->workspace);
    a.sums = a.sums_all + 2 * (int64_t)a.B * a.C;
    const int64_t blocks = (int64_t)a.slabs * chunks_of(a) * a.B;
    if (blocks >= (1 << 24)) return s2attn_fail(S2ATTN_E_UNSUPPORTED, "group norm needs %lld workgroups, more than one grid holds", (long long)blocks);
    const unsigned nb = (unsigned)blocks;
    switch (a.act) {
    case S2ATTN_ACT_NONE: backward_act<T, V, S2ATTN_ACT_NONE>(a, nb, s); break;
    case S2ATTN_ACT_RELU: backward_act<T, V, S2ATTN_ACT_RELU>(a, nb, s); break;
    case S2ATTN_ACT_SILU: backward_act<T, V, S2ATTN_ACT_SILU>(a, nb, s); break;
    case S2ATTN_ACT_GELU: backward_act<T, V, S2ATTN_ACT_GELU>(a, nb, s); break;
    }
    return launched("group norm backward");
}

template <typename T> int forward_t(const s2attn_gnorm *n, hipStream_t s)
{
    switch (width_of(n, {n->x, n->y})) {
    case 8:
        if constexpr (sizeof(T) == 2) return forward_v<T, 8>(n, s);
    case 4: return forward_v<T, 4>(n, s);
    }
    return forward_v<T, 1>(n, s);
}
template <typename T> int backward_t(const s2attn_gnorm *n, hipStream_t s)
{
    switch (width_of(n, {n->x, n->dy, n->dx})) {
    case 8:
        if constexpr (sizeof(T) == 2) return backward_v<T, 8>(n, s);
    case 4: return backward_v<T, 4>(n, s);
    }
    return backward_v<T, 1>(n, s);
}

} // namespace s2norm

extern "C" int64_t s2attn_group_norm_workspace_bytes(const s2attn_gnorm *n, int backward)
{
    using namespace s2norm;
    const int rc = check(n);
    if (rc != S2ATTN_OK) return rc;
    const int64_t slabs = (int64_t)n->batch * slabs_of(n);
    if (backward) return 2 * (int64_t)sizeof(float) * n->channels * (n->batch + slabs);
    return (int64_t)sizeof(Moments) * slabs * n->groups * ((n->channels + NT - 1) / NT); // (a chunk of workgroups has at least NT channels)
}

extern "C" int s2attn_group_norm(const s2attn_gnorm *n, void *stream)
{
    using namespace s2norm;
    const int rc = check(n);
    if (rc != S2ATTN_OK) return rc;
    if (!n->x || !n->y || !n->stats || !n->workspace) return s2attn_fail(S2ATTN_E_INVALID, "null tensor pointer");
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return n->dtype == S2ATTN_F32 ? forward_t<float>(n, s) : n->dtype == S2ATTN_BF16 ? forward_t<bf16_t>(n, s) : forward_t<f16_t>(n, s);
}

extern "C" int s2attn_group_norm_backward(const s2attn_gnorm *n, void *stream)
{
    using namespace s2norm;
    const int rc = check(n);
    if (rc != S2ATTN_OK) return rc;
    if (!n->x || !n->dy || !n->stats || !n->workspace) return s2attn_fail(S2ATTN_E_INVALID, "null tensor pointer");
    if (!n->dx && !n->dweight && !n->dbias) return S2ATTN_OK;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return n->dtype == S2ATTN_F32 ? backward_t<float>(n, s) : n->dtype == S2ATTN_BF16 ? backward_t<bf16_t>(n, s) : backward_t<f16_t>(n, s);
}
