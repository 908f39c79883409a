// Differential attention with the accuracy of fp32 on bf16 matrix instructions, for fp32 storage and for 16-bit head widths that the kernels of
// s2attn_diff16.hpp do not take.  Included by s2attn_kernels.hip inside namespace s2 after s2attn_diff16.hpp.
//
// Tiles and layout as there, values as terms as in s2attn_s16.hpp: staged rows are split once per workgroup, probabilities and dS once per
// step, and a product is the six term products of at most second order.  A step's products are added to sums of 32 bits, those of low order first; the
// forward and the dk/dv pass keep one register per sum, not two, and so a wavefront more per SIMD (181x360, 4 x 64 channels, forward: 281 -> 249 us).
//
// Shape domain: ck and cv multiples of 4, 2 ck and cv at most D (16, 32, 64; fp32 also 128), at least 32 columns per virtual latitude, rows
// aligned to four 16-bit values, or to a float.

// The lane's own row of both maps: channels outside a map are zero.  (Heads of up to 16 channels: the packing of S16Own.  PACKED: maps of exactly 16
// channels in three terms, two terms in the 32 k slots of an instruction, rows [h m] of the map's own channels against [h h] and [m m], [l h] against
// [h l]: twelve products fewer a step; 128x256, 4 heads: forward 188 -> 172 us, dq 202 -> 186, dk/dv 259 -> 240.)
template <typename T, int D, bool SCALED, bool PAD> struct SplitMaps {
    typedef S16Own<T, D, SCALED> Own;
    static constexpr int NS = Own::NS, S = Own::S;
    static constexpr bool PACKED = D == 32 && !PAD && S == 3;
    Own own[2];
    static constexpr __device__ bool has(int i, int s) { return i == 0 ? 2 * s < (NS > 1 ? NS : 2) : PAD || D <= 32 || 2 * s >= NS; } // (see DiffOwn)
    __device__ inline void load(const T *p, int n, int qd)
    {
        const int d = n / 2;
        if constexpr (PACKED) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                S16Piece<T> r;
                r.template load<false>(p, 16 * i + 8 * (qd & 1), n);
                float x[8];
                r.widen(x);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] *= SCALED ? LOG2E : 1.f;
                s16_split8(own[i].t[0], x);
                if (qd < 2) own[i].t[0][2] = own[i].t[0][0];
            }
            return;
        }
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const int first = D == 16 ? 8 * (qd & 1) : 32 * s + 8 * qd;
            S16Piece<T> r;
            r.template load<PAD>(p, first, n);
            float x[8];
            r.widen(x);
            if (SCALED) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] *= LOG2E;
            }
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (!has(i, s)) continue;
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; e++) y[e] = (first + e < d) == (i == 0) ? x[e] : 0.f;
                s16_split8(own[i].t[s], y);
                if (D == 16 && S == 3 && qd < 2) own[i].t[0][2] = own[i].t[0][0];
                if (D == 16 && S == 1) {
                    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
                    if (qd >= 2) own[i].t[0][0] = own[i].t[0][1], own[i].t[0][2] = zero;
                    own[i].t[0][1] = own[i].t[0][2];
                }
            }
        }
    }
    __device__ inline void settle_()
    {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int s = 0; s < NS; s++)
                if (has(i, s)) settle(own[i].t[s]);
    }
    // sums += (rows of the 16-row block) x own, both maps
    __device__ inline void scores(S16Sum &s0, S16Sum &s1, const char *blk, int c, int qd) const
    {
        typedef H16<bf16_t> M;
        const char *row = blk + c * s16_pitch<D, S>();
        if constexpr (PACKED) {
            row += 16 * (qd & 1);
            const int hm = qd < 2 ? 0 : 2 * D, lh = qd < 2 ? 4 * D : 0;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                S16Sum &s = i ? s1 : s0;
                const uint4 x = *reinterpret_cast<const uint4 *>(row + 32 * i + hm), y = *reinterpret_cast<const uint4 *>(row + 32 * i + lh);
                s.lo = M::mfma(y, own[i].t[0][2], s.lo);
                s.hi = M::mfma(x, own[i].t[0][0], s.hi);
                s.lo = M::mfma(x, own[i].t[0][1], s.lo);
            }
        } else if constexpr (D == 16) {
            const uint4 hm = *reinterpret_cast<const uint4 *>(row + (S == 1 ? 16 * (qd & 1) : 16 * qd));
            if constexpr (S == 3) {
                const uint4 lh = *reinterpret_cast<const uint4 *>(row + (qd < 2 ? 64 + 16 * qd : 16 * qd - 32));
                s0.lo = M::mfma(lh, own[0].t[0][2], s0.lo);
                s1.lo = M::mfma(lh, own[1].t[0][2], s1.lo);
            } else if constexpr (S == 2 && SCALED) {
                s0.lo = M::mfma(hm, own[0].t[0][2], s0.lo);
                s1.lo = M::mfma(hm, own[1].t[0][2], s1.lo);
            }
            s0.hi = M::mfma(hm, own[0].t[0][0], s0.hi);
            s1.hi = M::mfma(hm, own[1].t[0][0], s1.hi);
            if (S > 1 || SCALED) {
                s0.lo = M::mfma(hm, own[0].t[0][1], s0.lo);
                s1.lo = M::mfma(hm, own[1].t[0][1], s1.lo);
            }
        } else {
#pragma unroll
            for (int s = 0; s < NS; s++) {
                uint4 x[3];
#pragma unroll
                for (int n = 0; n < S; n++) x[n] = *reinterpret_cast<const uint4 *>(row + 64 * s + 16 * qd + 2 * D * n);
                if (has(0, s)) s16_mma<S, Own::NT>(s0, x, own[0].t[s]);
                if (has(1, s)) s16_mma<S, Own::NT>(s1, x, own[1].t[s]);
            }
        }
    }
};

// As DiffSum; A: S16Sum, or f4v where registers are short (see s16_accumulate)
template <typename A, int D, int S, bool PAD> struct SplitMapSum {
    static constexpr int NCB = D / 16;
    A acc[NCB], both[1];
    __device__ inline void zero() { s16_zero(acc), s16_zero(both); }
    static __device__ inline void mma(S16Sum &s, const uint4 (&x)[3], const uint4 (&p)[3]) { s16_mma<S, 3>(s, x, p); }
    static __device__ inline void mma(f4v &s, const uint4 (&x)[3], const uint4 (&p)[3])
    {
        S16Sum t = {s, f4v{0.f, 0.f, 0.f, 0.f}};
        s16_mma<S, 3>(t, x, p);
        s = t.hi + t.lo;
    }
    // + rows^T (p0 | p1)
    __device__ inline void add(const char *blk0, const char *blk1, int c, int qd, const uint4 (&p0)[3], const uint4 (&p1)[3], int d)
    {
#pragma unroll
        for (int cb = 0; cb < NCB; cb++) {
            uint4 x[3], p[3];
            rows(x, blk0, blk1, cb, c, qd);
#pragma unroll
            for (int n = 0; n < 3; n++) p[n] = DiffSum<H16<bf16_t>, D, PAD>::of_map(cb, p0[n], p1[n], d);
            if (D == 16) {
                mma(acc[0], x, p0);
                mma(both[0], x, p1);
            } else {
                mma(acc[cb], x, p);
            }
        }
        if (PAD && D > 16) {
            uint4 x[3];
            rows(x, blk0, blk1, d / 16, c, qd);
            mma(both[0], x, p1);
        }
    }
    static __device__ inline void rows(uint4 (&x)[3], const char *blk0, const char *blk1, int cb, int c, int qd)
    {
#pragma unroll
        for (int n = 0; n < S; n++) x[n] = h16_read_transposed<s16_pitch<D, S>()>(blk0 + 2 * D * n, blk1 + 2 * D * n, cb, c, qd);
    }
    __device__ inline f4v value(int cb, int qd, int d) const { return (PAD || D == 16) && 16 * cb < d && 16 * cb + 4 * qd >= d ? s16_value(both[0]) : s16_value(acc[cb]); }
    static __device__ inline bool first(int cb, int qd, int d) { return PAD || D == 16 ? 16 * cb + 4 * qd < d : cb < NCB / 2; }
    __device__ inline float check() const
    {
        float s = PAD || D == 16 ? point_sum(s16_value(both[0])) : 0.f;
#pragma unroll
        for (int cb = 0; cb < NCB; cb++) s += point_sum(s16_value(acc[cb]));
        return s;
    }
};

// The rows of a step: a piece of eight channels per thread and iteration, split as it goes to LDS
template <typename T, int D, bool PAD> struct SplitStage {
    typedef QuadPieces<D / 8> P;
    static constexpr int S = S16Piece<T>::S, PITCH = s16_pitch<D, S>(), BYTES = 2 * HK * PITCH;
    S16Piece<T> r[P::N];
    float w; // gather: the quadrature weight

    // rows cs .. cs + n of W columns; columns lda, ldb elements apart; na, nb channels
    __device__ inline void fetch(const T *pa, const T *pb, int tid, int cs, int W, int n, unsigned lda, unsigned ldb, int na, int nb)
    {
#pragma unroll
        for (int it = 0; it < P::N; it++) {
            const int i = P::at(it, tid);
            const bool second = P::second(i);
            unsigned col = (unsigned)(cs + min(P::row(i), n - 1));
            col = min(col, col - (unsigned)W); // (wraps to a huge value when col < W; 32 <= W)
            r[it].template load<PAD>((second ? pb : pa) + col * (second ? ldb : lda), 8 * P::piece(i), second ? nb : na);
        }
    }
    // SCALED: the first tensor's times log2 e (fp32)
    template <bool SCALED = false> __device__ inline void commit(char *buf, int tid)
    {
#pragma unroll
        for (int it = 0; it < P::N; it++) {
            const int i = P::at(it, tid);
            if constexpr (SCALED) {
                const float f = P::second(i) ? 1.f : LOG2E;
                r[it].a *= f, r[it].b *= f;
            }
            uint4 t[3];
            s16_terms<T>(t, r[it]);
            if (P::on(i)) {
                char *o = buf + (P::second(i) ? HK * PITCH : 0) + P::row(i) * PITCH + 16 * P::piece(i);
#pragma unroll
                for (int k = 0; k < S; k++) *reinterpret_cast<uint4 *>(o + 2 * D * k) = t[k];
            }
        }
    }
};
template <typename T, int D> constexpr int dsplit_lds_bytes(bool stats) { return 2 * (SplitStage<T, D, false>::BYTES + (stats ? HK * 16 : 0)); }

// Start values of a step's scores: `start` where the point sees the position
__device__ inline void quad_start(S16Sum (&sc)[2], const QuadStep &cur, int c, int qd, float start)
{
    sc[0].lo = sc[1].lo = f4v{0.f, 0.f, 0.f, 0.f};
    sc[0].hi = sc[1].hi = f4v{start, start, start, start};
    if (!cur.inner()) {
        const int tb = cur.first(c) + 4 * qd;
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int v = 0; v < 4; v++) sc[kb].hi[v] = (unsigned)(tb + 16 * kb + v) < (unsigned)cur.l ? start : -INFINITY;
    }
}

// ---- forward -------------------------------------------------------------------------------------------------------------------
template <typename T, int D, bool PAD> __global__ __launch_bounds__(64 * NW, D <= 32 ? 4 : 1) void fwd_dsplit_kernel(const DArgs a)
{
    typedef SplitStage<T, D, PAD> Band_;
    constexpr int S = Band_::S, PITCH = Band_::PITCH, NCB = D / 16;
    extern __shared__ __attribute__((aligned(16))) char h16_lds[];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, qd = lane >> 4, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const QuadUnit u = quad_unit(a, blockIdx.x);
    const int bh = u.bh, b = u.b, h = u.h, w0 = u.w0;
    const int ho = min(QUAD * u.g + wv, a.Ho - 1); // (a latitude that is not there sees nothing and stores nothing)
    const int nk = PAD ? a.dk_ : D, nv = PAD ? a.dv_ : D;
    const T *kx = static_cast<const T *>(a.k) + (size_t)b * a.Hi * a.Wi * a.ldk + h * nk;
    const T *vx = static_cast<const T *>(a.v) + (size_t)b * a.Hi * a.Wi * a.ldv + h * nv;
    const bool mine = QUAD * u.g + wv < a.Ho && w0 + c < a.Wo;
    const size_t pt = (size_t)query_point(a, b, ho, a.qps == 1 ? ho : ho / a.qps) + (size_t)(w0 + (mine ? c : 0)) * a.qps;

    SplitMaps<T, D, true, PAD> own; // q log2 e: scores come out in the log2 domain
    own.load(static_cast<const T *>(a.q) + pt * a.ldq + h * nk, nk, qd);
    typedef SplitMapSum<f4v, D, S, PAD> Sums;
    f4v acc[2][NCB];
    s16_zero(acc[0]), s16_zero(acc[1]);
    float m[2] = {0.f, 0.f}, Z[2] = {0.f, 0.f};
    bool first = true; // this column has seen no neighbor of positive weight

    QuadWalk wk;
    Band_ bd;
    const unsigned lda = a.ldk * a.kps, ldb = a.ldv * a.kps; // elements between two columns of a virtual input latitude
    auto fetch = [&]() {
        const size_t row = quad_row(wk.lat, wk.aux, a.kps, a.Wi);
        bd.w = a.quad_w[wk.aux + wk.zero];
        bd.fetch(kx + row * a.ldk, vx + row * a.ldv, tid, wk.column(w0), a.Wi, wk.rows(), lda, ldb, nk, nv);
    };
    char *buf = h16_lds, *other = h16_lds + Band_::BYTES;
    wk.start(a, u, wv, lane);
    QuadStep cur = wk.step();
    float weight = 1.f;
    if (cur.some) {
        fetch();
        bd.commit(buf, tid);
        weight = bd.w;
    }
    __syncthreads();
    own.settle_();

    while (cur.some) {
        wk.follow();
        fetch();
        if (cur.seen()) {
            const char *k0 = buf, *k1 = buf + 16 * PITCH, *v0 = buf + HK * PITCH, *v1 = buf + (HK + 16) * PITCH;
            // The sums start at log2 w - m, so they end as the exponents of the probabilities.
            S16Sum s0[2], s1[2];
            const float lw = fast_log2(weight);
            quad_start(s0, cur, c, qd, lw - m[0]);
            quad_start(s1, cur, c, qd, lw - m[1]);
            own.scores(s0[0], s1[0], k0, c, qd);
            own.scores(s0[1], s1[1], k1, c, qd);
            f4v p[2][2] = {{s16_value(s0[0]), s16_value(s0[1])}, {s16_value(s1[0]), s16_value(s1[1])}};
            float mx[2];
#pragma unroll
            for (int i = 0; i < 2; i++)
                mx[i] = fmaxf(fmaxf(fmaxf(p[i][0][0], p[i][0][1]), fmaxf(p[i][0][2], p[i][0][3])), fmaxf(fmaxf(p[i][1][0], p[i][1][1]), fmaxf(p[i][1][2], p[i][1][3])));
            // The running maxima are only the reference points of the exponentials: see fwd_s16_kernel.
            if (__any(first || mx[0] > RESCALE_THR || mx[1] > RESCALE_THR)) {
                bool seen = false;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float cm = h16_quarter_max(mx[i]);
                    const float dm = (first && cm > -INFINITY) || cm > RESCALE_THR ? cm : 0.f;
                    const float corr = first ? 0.f : fast_exp2(-dm);
                    Z[i] *= corr;
#pragma unroll
                    for (int cb = 0; cb < NCB; cb++) acc[i][cb] *= corr;
                    p[i][0] -= dm, p[i][1] -= dm;
                    m[i] += dm;
                    seen |= cm > -INFINITY;
                }
                first = first && !seen;
            }
            uint4 ps[2][3];
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        p[i][kb][v] = fast_exp2(p[i][kb][v]); // masked: exp2(-inf) = 0
                        Z[i] += p[i][kb][v];                  // this lane's share; the four lanes of a column are added up at the end
                    }
                s16_split_blocks(ps[i], p[i]);
            }
#pragma unroll
            for (int cb = 0; cb < NCB; cb++) {
                uint4 x[3];
#pragma unroll
                for (int n = 0; n < S; n++) x[n] = h16_read_transposed<PITCH>(v0 + 2 * D * n, v1 + 2 * D * n, cb, c, qd);
                Sums::mma(acc[0][cb], x, ps[0]);
                Sums::mma(acc[1][cb], x, ps[1]);
            }
        }
        bd.commit(other, tid);
        weight = bd.w;
        __syncthreads();
        char *t = buf;
        buf = other, other = t;
        cur = wk.step();
    }

    const float z0 = h16_quarter_sum(Z[0]), z1 = h16_quarter_sum(Z[1]);
    float check = z0 + z1;
#pragma unroll
    for (int cb = 0; cb < NCB; cb++) check += point_sum(acc[0][cb] + acc[1][cb]);
    const unsigned redo = point_columns(mine && not_finite(check));
    if (mine) {
        if (a.lse2 && qd == 0)
            a.lse2[((size_t)bh * a.Ho + ho) * a.Wo + w0 + c] = make_float2(z0 == 0.f ? INFINITY : m[0] + fast_log2(z0), z1 == 0.f ? INFINITY : m[1] + fast_log2(z1));
        const float i0 = z0 == 0.f ? 0.f : 1.0f / z0, i1 = z1 == 0.f ? 0.f : 1.0f / z1, lam = load_as_f32(a.lam, h, a.lam_dtype);
        T *y = static_cast<T *>(a.y) + pt * a.ldy + h * nv + 4 * qd;
        T *y2 = static_cast<T *>(a.y2) + (pt * a.nh + h) * nv + 4 * qd;
#pragma unroll
        for (int cb = 0; cb < NCB; cb++)
            if (!PAD || 16 * cb + 4 * qd < nv) {
                const f4v o2 = acc[1][cb] * i1;
                s16_store4(y + 16 * cb, acc[0][cb] * i0 - lam * o2);
                if (a.y2) s16_store4(y2 + 16 * cb, o2);
            }
    }
    if (__builtin_expect(redo != 0, 0)) diff_redo<T, D, FWD>(wv, blockIdx.x, redo);
}

// ---- backward, dq pass -----------------------------------------------------------------------------------------------------------
template <typename T, int D, bool PAD> __global__ __launch_bounds__(64 * NW) void dq_dsplit_kernel(const DArgs a)
{
    typedef SplitStage<T, D, PAD> Band_;
    constexpr int S = Band_::S, PITCH = Band_::PITCH, NCB = D / 16;
    extern __shared__ __attribute__((aligned(16))) char h16_lds[];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, qd = lane >> 4, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const QuadUnit u = quad_unit(a, blockIdx.x);
    const int bh = u.bh, b = u.b, h = u.h, w0 = u.w0;
    const int ho = min(QUAD * u.g + wv, a.Ho - 1); // (a latitude that is not there sees nothing and stores nothing)
    const int nk = PAD ? a.dk_ : D, nv = PAD ? a.dv_ : D, d = nk / 2;
    const T *kx = static_cast<const T *>(a.k) + (size_t)b * a.Hi * a.Wi * a.ldk + h * nk;
    const T *vx = static_cast<const T *>(a.v) + (size_t)b * a.Hi * a.Wi * a.ldv + h * nv;
    const bool mine = QUAD * u.g + wv < a.Ho && w0 + c < a.Wo;
    const size_t pt = (size_t)query_point(a, b, ho, a.qps == 1 ? ho : ho / a.qps) + (size_t)(w0 + (mine ? c : 0)) * a.qps;
    const size_t sidx = ((size_t)bh * a.Ho + ho) * a.Wo + w0 + (mine ? c : 0);
    const float lam = load_as_f32(a.lam, h, a.lam_dtype);

    SplitMaps<T, D, true, PAD> qo;
    S16Own<T, D, false> go;
    qo.load(static_cast<const T *>(a.q) + pt * a.ldq + h * nk, nk, qd);
    const T *dyp = static_cast<const T *>(a.dy) + pt * a.ldg + h * nv;
    go.template load<PAD>(dyp, nv, qd);
    float D1 = 0.f, D2 = 0.f;
    {
        const T *yp = static_cast<const T *>(a.ysaved) + pt * a.ldy + h * nv, *y2p = static_cast<const T *>(a.y2saved) + (pt * a.nh + h) * nv;
#pragma unroll
        for (int s = 0; s < (D + 31) / 32; s++) {
            S16Piece<T> yr, y2r, gr;
            yr.template load<PAD || D == 16>(yp, 32 * s + 8 * qd, nv); // (16 channels: the upper two quarters have none)
            y2r.template load<PAD || D == 16>(y2p, 32 * s + 8 * qd, nv);
            gr.template load<PAD || D == 16>(dyp, 32 * s + 8 * qd, nv);
            float x[8], x2[8], g[8];
            yr.widen(x), y2r.widen(x2), gr.widen(g);
#pragma unroll
            for (int i = 0; i < 8; i++) D1 = fmaf(g[i], x[i], D1), D2 = fmaf(g[i], x2[i], D2);
        }
    }
    D2 = h16_quarter_sum(D2);
    D1 = fmaf(lam, D2, h16_quarter_sum(D1));
    float2 lse = a.lse2[sidx];

    constexpr bool EXACT_I = S == 3;
    SplitMapSum<S16Sum, D, S, PAD> acc;
    acc.zero();
    DiffSum<H16<bf16_t>, D, PAD || D == 16> ak; // (leading terms)
    ak.zero();
    float off[2] = {0.f, 0.f};

    QuadWalk wk;
    Band_ bd;
    const unsigned lda = a.ldk * a.kps, ldb = a.ldv * a.kps; // elements between two columns of a virtual input latitude
    auto fetch = [&]() {
        const size_t row = quad_row(wk.lat, wk.aux, a.kps, a.Wi);
        bd.w = a.quad_w[wk.aux + wk.zero];
        bd.fetch(kx + row * a.ldk, vx + row * a.ldv, tid, wk.column(w0), a.Wi, wk.rows(), lda, ldb, nk, nv);
    };
    char *buf = h16_lds, *other = h16_lds + Band_::BYTES;
    wk.start(a, u, wv, lane);
    QuadStep cur = wk.step();
    float weight = 1.f;
    if (cur.some) {
        fetch();
        bd.commit(buf, tid);
        weight = bd.w;
    }
    __syncthreads();
    qo.settle_();
    go.settle_();
    settle(lse.x), settle(lse.y);
    const float step21 = D1 - D2; // g - D2 = (g - D1) + (D1 - D2)

    while (cur.some) {
        wk.follow();
        fetch();
        if (cur.seen()) {
            const char *k0 = buf, *k1 = buf + 16 * PITCH, *v0 = buf + HK * PITCH, *v1 = buf + (HK + 16) * PITCH;
            // The sums start at log2 w - lse and at -D1, so they end as the exponents of p and as g - D1.
            S16Sum s0[2], s1[2], gc[2];
            const float lw = fast_log2(weight);
            quad_start(s0, cur, c, qd, lw - lse.x);
            quad_start(s1, cur, c, qd, lw - lse.y);
            gc[0].hi = gc[1].hi = f4v{-D1, -D1, -D1, -D1};
            gc[0].lo = gc[1].lo = f4v{0.f, 0.f, 0.f, 0.f};
            qo.scores(s0[0], s1[0], k0, c, qd);
            qo.scores(s0[1], s1[1], k1, c, qd);
            s16_scores(gc[0], v0, c, qd, go);
            s16_scores(gc[1], v1, c, qd, go);
            f4v p[2][2], ds[2][2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const float g = gc[kb].hi[v] + gc[kb].lo[v];
                    p[0][kb][v] = fast_exp2(s0[kb].hi[v] + s0[kb].lo[v]);
                    p[1][kb][v] = fast_exp2(s1[kb].hi[v] + s1[kb].lo[v]);
                    ds[0][kb][v] = p[0][kb][v] * g;
                    ds[1][kb][v] = p[1][kb][v] * (g + step21);
                    if (!EXACT_I) off[0] += ds[0][kb][v], off[1] += ds[1][kb][v];
                }
            if constexpr (!EXACT_I) {
                const uint4 pb0 = d16_pack<H16<bf16_t>>(p[0]), pb1 = d16_pack<H16<bf16_t>>(p[1]);
#pragma unroll
                for (int cb = 0; cb < NCB; cb++) ak.add(cb, h16_read_transposed<PITCH>(k0, k1, cb, c, qd), pb0, pb1, d);
                if (PAD) ak.add_both(h16_read_transposed<PITCH>(k0, k1, d / 16, c, qd), pb1);
            }
            uint4 d0[3], d1[3];
            s16_split_blocks(d0, ds[0]);
            s16_split_blocks(d1, ds[1]);
            acc.add(k0, k1, c, qd, d0, d1, d);
        }
        bd.commit(other, tid);
        weight = bd.w;
        __syncthreads();
        char *t = buf;
        buf = other, other = t;
        cur = wk.step();
    }

    // (stored after the walk, see dq_d16_kernel)
    const float o0 = EXACT_I ? 0.f : h16_quarter_sum(off[0]), o1 = EXACT_I ? 0.f : h16_quarter_sum(off[1]);
    float check = o0 + o1 + acc.check();
    if (!EXACT_I) {
#pragma unroll
        for (int cb = 0; cb < NCB; cb++) check += point_sum(ak.acc[cb]);
        check += point_sum(ak.both);
    }
    const unsigned redo = point_columns(mine && not_finite(check));
    float part = 0.f;
    if (mine) {
        const float s2 = not_finite(o1) ? D2 : D2 + o1;
        part = qd == 0 ? s2 : 0.f;
        if (qd == 0) a.dstats[sidx] = make_float4(lse.x, lse.y, D1 + o0, s2);
        T *dq = static_cast<T *>(a.dq) + pt * a.lddq + h * nk + 4 * qd;
#pragma unroll
        for (int cb = 0; cb < NCB; cb++)
            if (!PAD || 16 * cb + 4 * qd < nk) {
                const bool one = acc.first(cb, qd, d);
                f4v x = acc.value(cb, qd, d);
                if (!EXACT_I) x -= (one ? o0 : o1) * ak.value(cb, qd, d);
                s16_store4(dq + 16 * cb, x * (one ? 1.f : -lam));
            }
    }
    if (QUAD * u.g + wv < a.Ho) {
        part = point_lanes_sum(part);
        if (lane == 0) a.lam_part[(size_t)bh * a.lam_n + (size_t)ho * ((a.Wo + HQ - 1) / HQ) + w0 / HQ] = part;
    }
    if (__builtin_expect(redo != 0, 0)) diff_redo<T, D, DQ>(wv, blockIdx.x, redo);
}

// ---- backward, dk/dv pass: transposed gather (see dkdv_s16_kernel) ---------------------------------------------------------------------
template <typename T, int D, bool PAD> __global__ __launch_bounds__(64 * NW, D <= 32 ? 3 : 1) void dkdv_dsplit_kernel(const DArgs a)
{
    typedef SplitStage<T, D, PAD> Band_;
    constexpr int S = Band_::S, PITCH = Band_::PITCH, NCB = D / 16;
    extern __shared__ __attribute__((aligned(16))) char h16_lds[];
    if ((int)blockIdx.x < a.lam_blocks) {
        diff_sum_lam(a, blockIdx.x, threadIdx.x, 64 * NW, reinterpret_cast<double *>(h16_lds));
        return;
    }
    const int block = blockIdx.x - a.lam_blocks;

    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, qd = lane >> 4, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const QuadUnit u = quad_unit(a, block);
    const int bh = u.bh, b = u.b, h = u.h, w0 = u.w0;
    const int hi = min(QUAD * u.g + wv, a.Hi - 1);
    const int nk = PAD ? a.dk_ : D, nv = PAD ? a.dv_ : D, d = nk / 2;
    const T *qy = static_cast<const T *>(a.q) + (size_t)b * a.Ho * a.Wo * a.ldq + h * nk;
    const T *gy = static_cast<const T *>(a.dy) + (size_t)b * a.Ho * a.Wo * a.ldg + h * nv;
    const float4 *stats = a.dstats + (size_t)bh * a.Ho * a.Wo;
    const bool mine = QUAD * u.g + wv < a.Hi && w0 + c < a.Wi;
    const size_t pt = (size_t)key_point(a, b, hi, a.kps == 1 ? hi : hi / a.kps) + (size_t)(w0 + (mine ? c : 0)) * a.kps;
    float lam = load_as_f32(a.lam, h, a.lam_dtype);

    constexpr bool QSCALED = S == 3;
    SplitMaps<T, D, !QSCALED, PAD> ko;
    S16Own<T, D, false> vo;
    ko.load(static_cast<const T *>(a.k) + pt * a.ldk + h * nk, nk, qd);
    vo.template load<PAD>(static_cast<const T *>(a.v) + pt * a.ldv + h * nv, nv, qd);
    SplitMapSum<f4v, D, S, PAD> dkt;
    dkt.zero();
    f4v dvt[NCB];
    s16_zero(dvt);
    const float lw = fast_log2(a.quad_w[a.kps == 1 ? hi : hi / a.kps]);

    QuadWalk wk;
    Band_ bd;
    float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
    const unsigned lda = a.ldq * a.qps, ldb = a.ldg * a.qps; // elements between two columns of a virtual output latitude
    auto fetch = [&]() {
        const size_t row = quad_row(wk.lat, wk.aux, a.qps, a.Wo);
        const int cs = wk.column(w0), n = wk.rows();
        bd.fetch(qy + row * a.ldq, gy + row * a.ldg, tid, cs, a.Wo, n, lda, ldb, nk, nv);
        int col = cs + min(tid & (HK - 1), n - 1); // (the first threads' are used)
        if (col >= a.Wo) col -= a.Wo;
        st = stats[(size_t)wk.lat * a.Wo + col];
    };
    auto commit = [&](char *to) {
        bd.template commit<QSCALED>(to, tid);
        if (tid < HK) { // -lse of the two maps, -D1, D1 - D2
            float *t = reinterpret_cast<float *>(to + Band_::BYTES) + tid;
            t[0] = -st.x, t[HK] = -st.y, t[2 * HK] = -st.z, t[3 * HK] = st.z - st.w;
        }
    };
    char *buf = h16_lds, *other = h16_lds + Band_::BYTES + HK * 16;
    wk.start(a, u, wv, lane);
    QuadStep cur = wk.step();
    if (cur.some) {
        fetch();
        commit(buf);
    }
    __syncthreads();
    ko.settle_();
    vo.settle_();
    settle(lam);

    while (cur.some) {
        wk.follow();
        fetch();
        if (cur.seen()) {
            const char *q0 = buf, *q1 = buf + 16 * PITCH, *g0 = buf + HK * PITCH, *g1 = buf + (HK + 16) * PITCH;
            // The sums start at the staged statistics, so they end as the exponents of p and as g - D1.
            S16Sum s0[2], s1[2], gc[2];
            f4v step[2];
#pragma unroll
            for (int qb = 0; qb < 2; qb++) {
                const float *t = reinterpret_cast<const float *>(buf + Band_::BYTES) + 16 * qb + 4 * qd;
                s0[qb].hi = *reinterpret_cast<const f4v *>(t) + lw;
                s1[qb].hi = *reinterpret_cast<const f4v *>(t + HK) + lw;
                gc[qb].hi = *reinterpret_cast<const f4v *>(t + 2 * HK);
                step[qb] = *reinterpret_cast<const f4v *>(t + 3 * HK);
                s0[qb].lo = s1[qb].lo = gc[qb].lo = f4v{0.f, 0.f, 0.f, 0.f};
            }
            const int tb = cur.first(c) + 4 * qd;
            if (!cur.inner()) { // (rows outside the neighborhood: a probability of zero)
#pragma unroll
                for (int qb = 0; qb < 2; qb++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const bool in = (unsigned)(tb + 16 * qb + v) < (unsigned)cur.l;
                        s0[qb].hi[v] = in ? s0[qb].hi[v] : -INFINITY;
                        s1[qb].hi[v] = in ? s1[qb].hi[v] : -INFINITY;
                    }
            }
            ko.scores(s0[0], s1[0], q0, c, qd);
            ko.scores(s0[1], s1[1], q1, c, qd);
            s16_scores(gc[0], g0, c, qd, vo);
            s16_scores(gc[1], g1, c, qd, vo);
            f4v co[2], ds[2][2];
#pragma unroll
            for (int qb = 0; qb < 2; qb++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const float g = gc[qb].hi[v] + gc[qb].lo[v];
                    const float p0 = fast_exp2(s0[qb].hi[v] + s0[qb].lo[v]), p1 = fast_exp2(s1[qb].hi[v] + s1[qb].lo[v]);
                    co[qb][v] = fmaf(-lam, p1, p0);
                    ds[0][qb][v] = p0 * g;
                    ds[1][qb][v] = p1 * (g + step[qb][v]);
                }
            uint4 ps[3], d1[3];
            s16_split_blocks(ps, co);
            s16_accumulate<D, S>(dvt, g0, g1, c, qd, ps);
            s16_split_blocks(ps, ds[0]);
            s16_split_blocks(d1, ds[1]);
            dkt.add(q0, q1, c, qd, ps, d1, d);
        }
        commit(other);
        __syncthreads();
        char *t = buf;
        buf = other, other = t;
        cur = wk.step();
    }

    float check = dkt.check();
#pragma unroll
    for (int cb = 0; cb < NCB; cb++) check += point_sum(s16_value(dvt[cb]));
    const unsigned redo = point_columns(mine && not_finite(check));
    if (mine) {
        T *dk = static_cast<T *>(a.dk) + pt * a.lddk + h * nk + 4 * qd, *dv = static_cast<T *>(a.dv) + pt * a.lddv + h * nv + 4 * qd;
        constexpr float unscale = QSCALED ? 1.f / LOG2E : 1.f;
#pragma unroll
        for (int cb = 0; cb < NCB; cb++) {
            if (!PAD || 16 * cb + 4 * qd < nk) s16_store4(dk + 16 * cb, dkt.value(cb, qd, d) * (dkt.first(cb, qd, d) ? unscale : -lam * unscale));
            if (!PAD || 16 * cb + 4 * qd < nv) s16_store4(dv + 16 * cb, s16_value(dvt[cb]));
        }
    }
    if (__builtin_expect(redo != 0, 0)) diff_redo<T, D, DKDV>(wv, block, redo);
}
