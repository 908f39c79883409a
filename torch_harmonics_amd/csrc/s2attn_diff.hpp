// Differential attention: the difference of two softmax maps over the same neighborhood with one learned weight per head.  Forward, dq and
// dk/dv.  Included by s2attn_kernels.hip inside namespace s2 after s2attn_s16.hpp.
//
// A head's query and key are two vectors of d channels, packed (q1 | q2, k1 | k2); with pi_j = w_j exp(qi . ki_j) / Zi
//   y    = sum_j (p1_j - lam p2_j) v_j
//   g_j  = <dy, v_j>,  Di = sum_j pi_j g_j = <dy, yi>,  yi = sum_j pi_j v_j,  y1 = y + lam y2
//   ds1  = p1 (g - D1),  ds2 = -lam p2 (g - D2)
//   dqi  = sum_j dsi_j ki_j,  dki_j = sum_queries dsi_j qi,  dv_j = sum_queries (p1_j - lam p2_j) dy,  dlam = - sum_points D2
// The forward keeps y2 and the two normalisers (log2 Zi) for the backward.  A point that sees nothing (no neighbor, or only latitudes of weight
// zero) has y = 0 and its normalisers are +inf, so that all its probabilities are zero in the backward.

// n / d for 0 <= n < 2^24, 0 < d < 2^24: m = floor(2^s / d) + 1, s = 24 + ceil(log2 d): n m / 2^s is less than 1 / d too large
struct QuadDiv {
    unsigned m;
    int s;
};
struct DArgs : Args {
    const void *lam; // [nh], of type lam_dtype
    void *dlam;      // [nh], of type lam_dtype, or null
    void *y2;        // forward, optional: the second map's output, packed [B, nlat_out, nlon_out, nh * cv]
    const void *y2saved;
    float2 *lse2;    // per point (virtual coordinates): log2 Z of the two maps; forward: optional
    float4 *dstats;  // per point: (lse1, lse2, D1, D2), written by the dq pass
    float *lam_part; // [B * nh][lam_n] summands of -dlam, written by the dq pass
    int lam_n;
    int lam_dtype;
    // the plan's bands of four latitudes (s2attn_plan.cpp, build_quads) in the pass's grouping; quads: the section
    const int *quads, *q_list, *q_bands;
    int q_groups;
    QuadDiv q_first, q_tiles, q_head;
    int lam_blocks;  // leading workgroups of the dk/dv launch that sum dlam, a head each
};

__device__ inline float load_as_f32(const void *p, int i, int dtype)
{
    if (dtype == S2ATTN_F32) return static_cast<const float *>(p)[i];
    if (dtype == S2ATTN_BF16) return to_f32(static_cast<const bf16_t *>(p)[i]);
    return to_f32(static_cast<const f16_t *>(p)[i]);
}
__device__ inline void store_from_f32(void *p, int i, int dtype, float x)
{
    if (dtype == S2ATTN_F32)
        static_cast<float *>(p)[i] = x;
    else if (dtype == S2ATTN_BF16)
        from_f32(static_cast<bf16_t *>(p)[i], x);
    else
        from_f32(static_cast<f16_t *>(p)[i], x);
}

// ---- one point at a time --------------------------------------------------------------------------------------------------
// A wavefront evaluates one grid point over its neighbors, four at a time: lane l = (j = l % 16, g = l / 16) holds channels j, j + 16, ... of
// neighbor g.  Any head widths up to 16 N, any strides and alignment: what the matrix-core kernels below do not take, and the columns
// of theirs whose sums are not finite (a tile multiplies rows that a column does not see by a probability of zero, and 0 x NaN is NaN).
// Bound by the latency of the loads.

// <x, y> over the channels of each of the two maps (d channels each, the second from channel d on)
template <typename T, int N> __device__ inline float2 diff_point_dots(const PointRow<T, N> &x, const PointRow<T, N> &y, int d, int j)
{
    float a = 0.f, s = 0.f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float t = x.x[i] * y.x[i];
        a += j + 16 * i < d ? t : 0.f;
        s += j + 16 * i < d ? 0.f : t;
    }
    return make_float2(point_lanes_sum(a), point_lanes_sum(s));
}

template <typename T, int N> __device__ inline void diff_point_forward(const DArgs &a, int b, int h, int bh, int ho, int wo, int lane)
{
    const int j = lane & 15, g = lane >> 4, d = a.dk_ / 2;
    const size_t pq = (size_t)query_point(a, b, ho, ho / a.qps) + (size_t)wo * a.qps;
    PointRow<T, N> q, k, v;
    q.load(static_cast<const T *>(a.q) + pq * a.ldq + h * a.dk_, a.dk_, j);
    float acc[2][N] = {}, m[2] = {NEG_BIG, NEG_BIG}, Z[2] = {0.f, 0.f};
    bool over = false; // both maps' sums are NaN by now
    for (int ri = a.goff[ho]; ri < a.goff[ho + 1] && !over; ri++) {
        const Run run = a.gruns[ri];
        const float w = a.quad_w[run.pad];
        const size_t row = (size_t)key_point(a, b, run.lat, run.pad);
        for (int t0 = 0; t0 < run.len && !over; t0 += 4) {
            const bool in = t0 + g < run.len;
            const size_t pk = row + (size_t)((run.ws + wo + t0 + (in ? g : 0)) % a.Wi) * a.kps;
            k.load(static_cast<const T *>(a.k) + pk * a.ldk + h * a.dk_, a.dk_, j);
            v.load(static_cast<const T *>(a.v) + pk * a.ldv + h * a.dv_, a.dv_, j);
            const float2 s2 = diff_point_dots(q, k, d, j);
            const float s[2] = {s2.x * LOG2E, s2.y * LOG2E};
            if (in) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float mn = fmaxf(m[i], s[i]), corr = fast_exp2(m[i] - mn), p = fast_exp2(s[i] - mn) * w;
                    m[i] = mn;
                    Z[i] = fmaf(Z[i], corr, p);
#pragma unroll
                    for (int n = 0; n < N; n++) acc[i][n] = fmaf(p, v.x[n], acc[i][n] * corr);
                }
            }
            over = __any(is_nan(Z[0]) || is_nan(Z[1])); // (y is their difference)
        }
    }
    float inv[2], lse[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float mx = h16_quarter_max(m[i]), f = fast_exp2(m[i] - mx);
        const float z = h16_quarter_sum(Z[i] * f);
        inv[i] = z == 0.f ? 0.f : f / z;
        lse[i] = z == 0.f ? INFINITY : mx + fast_log2(z);
    }
    const float lam = load_as_f32(a.lam, h, a.lam_dtype);
    T *y = static_cast<T *>(a.y) + pq * a.ldy + h * a.dv_;
    T *y2 = a.y2 ? static_cast<T *>(a.y2) + (pq * a.nh + h) * a.dv_ : nullptr;
#pragma unroll
    for (int n = 0; n < N; n++) {
        const float o1 = h16_quarter_sum(acc[0][n] * inv[0]), o2 = h16_quarter_sum(acc[1][n] * inv[1]);
        if (g == 0 && j + 16 * n < a.dv_) {
            from_f32(y[j + 16 * n], fmaf(-lam, o2, o1));
            if (y2) from_f32(y2[j + 16 * n], o2);
        }
    }
    if (a.lse2 && lane == 0) a.lse2[((size_t)bh * a.Ho + ho) * a.Wo + wo] = make_float2(lse[0], lse[1]);
}

// 16-bit storage: D1 and D2 come from the rounded y and y2, so they are only first values of the means of g.  The walk adds up how far the means
// are from them, off_i = sum pi (g - Di), and AKi = sum pi ki, and dq takes the product of the two off at the end.  On smooth fields, where
// the sums cancel, dq would be 1e-2 off without.  Returns D2.
template <typename T, int N> __device__ inline float diff_point_dq(const DArgs &a, int b, int h, int bh, int ho, int wo, int lane)
{
    constexpr bool EXACT_I = std::is_same<T, float>::value;
    const int j = lane & 15, g = lane >> 4, d = a.dk_ / 2;
    const size_t pq = (size_t)query_point(a, b, ho, ho / a.qps) + (size_t)wo * a.qps, si = ((size_t)bh * a.Ho + ho) * a.Wo + wo;
    const float lam = load_as_f32(a.lam, h, a.lam_dtype);
    PointRow<T, N> q, dy, k, v;
    q.load(static_cast<const T *>(a.q) + pq * a.ldq + h * a.dk_, a.dk_, j);
    dy.load(static_cast<const T *>(a.dy) + pq * a.ldg + h * a.dv_, a.dv_, j);
    v.load(static_cast<const T *>(a.y2saved) + (pq * a.nh + h) * a.dv_, a.dv_, j);
    float D[2];
    D[1] = dy.dot(v);
    v.load(static_cast<const T *>(a.ysaved) + pq * a.ldy + h * a.dv_, a.dv_, j);
    D[0] = fmaf(lam, D[1], dy.dot(v));
    const float2 l2 = a.lse2[si];
    const float lse[2] = {l2.x, l2.y};
    float acc[N] = {}, ak[EXACT_I ? 1 : N] = {}, off[2] = {0.f, 0.f};
    bool over = false;
    for (int ri = a.goff[ho]; ri < a.goff[ho + 1] && !over; ri++) {
        const Run run = a.gruns[ri];
        const float w = a.quad_w[run.pad];
        const size_t row = (size_t)key_point(a, b, run.lat, run.pad);
        for (int t0 = 0; t0 < run.len && !over; t0 += 4) {
            const bool in = t0 + g < run.len;
            const size_t pk = row + (size_t)((run.ws + wo + t0 + (in ? g : 0)) % a.Wi) * a.kps;
            k.load(static_cast<const T *>(a.k) + pk * a.ldk + h * a.dk_, a.dk_, j);
            v.load(static_cast<const T *>(a.v) + pk * a.ldv + h * a.dv_, a.dv_, j);
            const float2 s2 = diff_point_dots(q, k, d, j);
            const float gj = dy.dot(v);
            const float p[2] = {fast_exp2(fmaf(s2.x, LOG2E, -lse[0])) * w, fast_exp2(fmaf(s2.y, LOG2E, -lse[1])) * w};
            const float ds[2] = {p[0] * (gj - D[0]), p[1] * (gj - D[1])};
            if (in) {
                if (!EXACT_I) off[0] += ds[0], off[1] += ds[1];
#pragma unroll
                for (int n = 0; n < N; n++) {
                    const bool first = j + 16 * n < d;
                    acc[n] = fmaf(first ? ds[0] : ds[1], k.x[n], acc[n]);
                    if (!EXACT_I) ak[EXACT_I ? 0 : n] = fmaf(first ? p[0] : p[1], k.x[n], ak[EXACT_I ? 0 : n]);
                }
            }
            over = __any(in && is_nan(ds[0]) && is_nan(ds[1]));
        }
    }
    off[0] = h16_quarter_sum(off[0]), off[1] = h16_quarter_sum(off[1]);
    T *dq = static_cast<T *>(a.dq) + pq * a.lddq + h * a.dk_;
#pragma unroll
    for (int n = 0; n < N; n++) {
        const bool first = j + 16 * n < d;
        float x = acc[n];
        if (!EXACT_I) x = fmaf(-(first ? off[0] : off[1]), ak[EXACT_I ? 0 : n], x);
        x = h16_quarter_sum(x);
        if (g == 0 && j + 16 * n < a.dk_) from_f32(dq[j + 16 * n], first ? x : -lam * x);
    }
    if (lane == 0) a.dstats[si] = make_float4(lse[0], lse[1], D[0] + off[0], D[1] + off[1]);
    return D[1] + off[1];
}

template <typename T, int N> __device__ inline void diff_point_dkdv(const DArgs &a, int b, int h, int bh, int hi, int wi, int lane)
{
    const int j = lane & 15, g = lane >> 4, d = a.dk_ / 2;
    const size_t pk = (size_t)key_point(a, b, hi, hi / a.kps) + (size_t)wi * a.kps;
    const float lam = load_as_f32(a.lam, h, a.lam_dtype);
    PointRow<T, N> k, v, q, dy;
    k.load(static_cast<const T *>(a.k) + pk * a.ldk + h * a.dk_, a.dk_, j);
    v.load(static_cast<const T *>(a.v) + pk * a.ldv + h * a.dv_, a.dv_, j);
    const float w = a.quad_w[hi / a.kps];
    float dk[N] = {}, dv[N] = {};
    for (int ri = a.soff[hi]; ri < a.soff[hi + 1]; ri++) {
        const Run run = a.sruns[ri]; // the key is neighbor t of query column wi - ws - t
        const size_t row = (size_t)query_point(a, b, run.lat, run.pad), srow = ((size_t)bh * a.Ho + run.lat) * a.Wo;
        for (int t0 = 0; t0 < run.len; t0 += 4) {
            const bool in = t0 + g < run.len;
            int col = (wi - run.ws - t0 - (in ? g : 0)) % a.Wo;
            col += col < 0 ? a.Wo : 0;
            const size_t pq = row + (size_t)col * a.qps;
            const float4 st = a.dstats[srow + col];
            q.load(static_cast<const T *>(a.q) + pq * a.ldq + h * a.dk_, a.dk_, j);
            dy.load(static_cast<const T *>(a.dy) + pq * a.ldg + h * a.dv_, a.dv_, j);
            const float2 s2 = diff_point_dots(q, k, d, j);
            const float gj = dy.dot(v);
            const float p1 = fast_exp2(fmaf(s2.x, LOG2E, -st.x)) * w, p2 = lam * fast_exp2(fmaf(s2.y, LOG2E, -st.y)) * w;
            const float c = p1 - p2, ds1 = p1 * (gj - st.z), ds2 = -p2 * (gj - st.w);
            if (in) {
#pragma unroll
                for (int n = 0; n < N; n++) {
                    dv[n] = fmaf(c, dy.x[n], dv[n]);
                    dk[n] = fmaf(j + 16 * n < d ? ds1 : ds2, q.x[n], dk[n]);
                }
            }
        }
    }
    point_store(static_cast<T *>(a.dk) + pk * a.lddk + h * a.dk_, dk, 1.f, a.dk_, j, g);
    point_store(static_cast<T *>(a.dv) + pk * a.lddv + h * a.dv_, dv, 1.f, a.dv_, j, g);
}

// dlam of one head from the summands that the dq pass left, in a fixed order, by one workgroup.  The summands of a head are added up in 64 bits:
// there are up to millions of them, of both signs.  part: LDS, a number per wavefront.
__device__ inline void diff_sum_lam(const DArgs &a, int h, int tid, int nthreads, double *part)
{
    double s = 0.0;
    for (int b = 0; b < a.B; b++) {
        const float *p = a.lam_part + (size_t)(b * a.nh + h) * a.lam_n;
        int i = tid;
        for (; i + 7 * nthreads < a.lam_n; i += 8 * nthreads) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; u++) x[u] = p[i + u * nthreads];
#pragma unroll
            for (int u = 0; u < 8; u++) s += x[u];
        }
        for (; i < a.lam_n; i += nthreads) s += p[i];
    }
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((tid & 63) == 0) part[tid >> 6] = s;
    __syncthreads();
    if (tid == 0) {
        double t = 0.0;
        for (int i = 0; i < nthreads / 64; i++) t += part[i];
        store_from_f32(a.dlam, h, a.lam_dtype, (float)-t);
    }
}

// Workgroups of four points, as many as a launch of 2^31 threads has, each then the next four; the first `lam_blocks` workgroups of the dk/dv launch sum dlam, a head each.
constexpr int DPT = 4;
template <typename T, int N, Which PASS> __global__ __launch_bounds__(64 * DPT) void diff_points_kernel(const DArgs a, long npoints)
{
    const int lam_blocks = PASS == DKDV ? a.lam_blocks : 0;
    if ((int)blockIdx.x < lam_blocks) {
        __shared__ double part[DPT];
        diff_sum_lam(a, blockIdx.x, threadIdx.x, 64 * DPT, part);
        return;
    }
    const int lane = threadIdx.x & 63;
    const int W = PASS == DKDV ? a.Wi : a.Wo, BH = a.B * a.nh;
    const long stride = (long)(gridDim.x - lam_blocks) * DPT;
    for (long id = (long)(blockIdx.x - lam_blocks) * DPT + (threadIdx.x >> 6); id < npoints; id += stride) {
        const long r = id / BH;
        const int bh = (int)(id % BH), b = bh / a.nh, h = bh % a.nh, col = (int)(r % W);
        const int row = (PASS == DKDV ? a.sorder : a.gorder)[r / W];
        if (PASS == FWD) diff_point_forward<T, N>(a, b, h, bh, row, col, lane);
        if (PASS == DQ) {
            const float D2 = diff_point_dq<T, N>(a, b, h, bh, row, col, lane);
            if (lane == 0) a.lam_part[(size_t)bh * a.lam_n + (size_t)row * a.Wo + col] = D2;
        }
        if (PASS == DKDV) diff_point_dkdv<T, N>(a, b, h, bh, row, col, lane);
    }
}
