// Differential attention on 16-bit matrix instructions, 16-bit storage.  Included by s2attn_kernels.hip inside namespace s2 after s2attn_diff.hpp.
//
// Tiles as in s2attn_quads.hpp: sixteen columns of a latitude per wavefront, steps of 32 band positions; lane l = (c = l % 16, qd = l / 16);
// scores are produced transposed, S^T[position][column].  Facts about the instruction as in s2attn_h16.hpp.
//
// The row of k (q) holds both maps' channels and is staged once; map i's scores take the 32-channel blocks it has channels in, with the other map's
// channels zero on the side that stays in registers.  <dy, v>, the masks, the staged rows and the transposed reads of v serve both maps.
// Sums of probabilities (forward) and of dS and of P (dq pass: the corrections of D, see diff_point_dq) are of the rounded values that
// the products take: pairwise products with one (d16_sum: products on the matrix cores hold ten more registers), or with the staged rows.
//
// Shape domain: ck a multiple of 8, cv a multiple of 8, 2 ck and cv at most D (a tile is D channels wide, 32, 64 or 128; zeros are staged past
// a head's channels and never stored; PAD = false: 2 ck = cv = D), at least 32 columns per virtual latitude, rows 16-byte aligned.

template <int D, bool PAD> struct DiffStage {
    typedef QuadPieces<D / 8> P;
    static constexpr int PITCH = 2 * D + 32;    // bytes (32 or 96 modulo 128: free of bank conflicts, see WgBand)
    static constexpr int BYTES = 2 * HK * PITCH; // one buffer
    uint4 r[P::N];
    float4 st; // dk/dv pass: the statistics of row tid
    float w;   // gather: the quadrature weight

    // rows cs .. cs + n of W columns; lda, ldb: bytes between two columns; na, nb channels.  (Rows past n stay an earlier step's.)
    __device__ inline void fetch(const char *pa, const char *pb, int tid, int cs, int W, int n, unsigned lda, unsigned ldb, int na, int nb)
    {
#pragma unroll
        for (int it = 0; it < P::N; it++) {
            const int i = P::at(it, tid);
            const bool second = P::second(i);
            unsigned col = (unsigned)(cs + P::row(i));
            col = min(col, col - (unsigned)W); // (wraps to a huge value when col < W; 32 <= W)
            if (P::row(i) < n) r[it] = h16_load_piece((second ? pb : pa) + col * (second ? ldb : lda) + 16 * P::piece(i), !PAD || 8 * P::piece(i) < (second ? nb : na));
        }
    }
    __device__ inline void commit(char *buf, int tid) const
    {
#pragma unroll
        for (int it = 0; it < P::N; it++) {
            const int i = P::at(it, tid);
            if (P::on(i)) *reinterpret_cast<uint4 *>(buf + (P::second(i) ? HK * PITCH : 0) + P::row(i) * PITCH + 16 * P::piece(i)) = r[it];
        }
    }
};
template <int D> constexpr int d16_lds_bytes(bool stats) { return 2 * (DiffStage<D, false>::BYTES + (stats ? HK * 16 : 0)); }

// The lane's own row of both maps (a query's q, or a key's k): op[i][s] = channels 32 s + 8 qd .. + 8 of its row that belong to map i, zeros elsewhere
template <typename M, int D, bool PAD> struct DiffOwn {
    static constexpr int NS = D / 32;
    uint4 op[2][NS];
    __device__ inline void load(const char *row, int qd, int d)
    {
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const int ch = 32 * s + 8 * qd;
            const uint4 x = h16_load_piece(row + 2 * ch, !PAD || ch < 2 * d), zero = make_uint4(0u, 0u, 0u, 0u);
            op[0][s] = ch < d ? x : zero;
            op[1][s] = ch < d ? zero : x;
        }
    }
    __device__ inline void settle_()
    {
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int s = 0; s < NS; s++)
                if (has(i, s)) settle(op[i][s]);
    }
    // Does block s hold channels of map i?  PAD: it may, for some d.  (Decided when compiled: a branch on d around matrix instructions saves a few
    // of them, but the compiler, which waits for their results where it reads them, does not count right over the edges of such
    // branches: reads after too few clocks, seen in its output and in results.)
    static constexpr __device__ bool has(int i, int s) { return i == 0 ? 2 * s < (NS > 1 ? NS : 2) : PAD || D == 32 || 2 * s >= NS; }
    // sc[i] += (16 staged rows) x own, both maps
    __device__ inline void scores(f4v &s0, f4v &s1, const char *blk, int c, int qd) const
    {
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const uint4 x = h16_read_row<DiffStage<D, PAD>::PITCH>(blk, s, c, qd);
            if (has(0, s)) s0 = M::mfma(x, op[0][s], s0);
            if (has(1, s)) s1 = M::mfma(x, op[1][s], s1);
        }
    }
};

// Sums over positions of row[channel] * coefficient for rows of two maps: 16-channel block cb takes the coefficients of its map (PAD: chosen by
// selects, not by branches, see DiffOwn::has).  The block that channel d lies in may hold channels of both: it is computed with either, the
// second map's in `both`.
template <typename M, int D, bool PAD> struct DiffSum {
    static constexpr int NCB = D / 16;
    f4v acc[NCB], both;
    __device__ inline void zero()
    {
#pragma unroll
        for (int cb = 0; cb < NCB; cb++) acc[cb] = f4v{0.f, 0.f, 0.f, 0.f};
        both = f4v{0.f, 0.f, 0.f, 0.f};
    }
    static __device__ inline uint4 of_map(int cb, uint4 p0, uint4 p1, int d)
    {
        if (NCB > 1 && cb >= NCB / 2) return p1;
        if (!PAD || cb == 0) return p0;
        const bool first = 16 * cb < d;
        return make_uint4(first ? p0.x : p1.x, first ? p0.y : p1.y, first ? p0.z : p1.z, first ? p0.w : p1.w);
    }
    __device__ inline void add(int cb, uint4 rows, uint4 p0, uint4 p1, int d) { acc[cb] = M::mfma(rows, of_map(cb, p0, p1, d), acc[cb]); }
    // PAD: rows of the 16-channel block d / 16
    __device__ inline void add_both(uint4 rows, uint4 p1) { both = M::mfma(rows, p1, both); }
    // of this lane's channels 16 cb + 4 qd .. + 4
    __device__ inline f4v value(int cb, int qd, int d) const { return PAD && 16 * cb < d && 16 * cb + 4 * qd >= d ? both : acc[cb]; }
    static __device__ inline bool first(int cb, int qd, int d) { return PAD ? 16 * cb + 4 * qd < d : cb < NCB / 2; }
};

template <typename M> __device__ inline uint4 d16_pack(const f4v (&x)[2])
{
    return make_uint4(M::pack2(x[0][0], x[0][1]), M::pack2(x[0][2], x[0][3]), M::pack2(x[1][0], x[1][1]), M::pack2(x[1][2], x[1][3]));
}
// s + the sum of eight values as they were rounded
template <typename T> __device__ inline float d16_sum(float s, uint4 p)
{
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const unsigned w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (std::is_same<T, bf16_t>::value)
            s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w[i]), b2{(__bf16)1.f, (__bf16)1.f}, s, false);
        else
            s = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w[i]), h2{(_Float16)1.f, (_Float16)1.f}, s, false);
    }
    return s;
}

// The kernel's arguments again and the lanes counted anew, as point_args() has it
__device__ inline DArgs diff_point_args()
{
    typedef const int __attribute__((address_space(4))) * words;
    words p = (words)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    DArgs a;
    static_assert(sizeof(DArgs) % 4 == 0, "read as 32-bit words");
#pragma unroll
    for (unsigned i = 0; i < sizeof(DArgs) / 4; i++) reinterpret_cast<int *>(&a)[i] = p[i];
    return a;
}
// The columns `redo` of a wavefront whose sums are not finite, stored already
template <typename T, int D, Which PASS> __device__ __forceinline__ void diff_redo(int wv, int block, unsigned redo)
{
    __threadfence(); // what is written here comes after it
    const DArgs a = diff_point_args();
    const QuadUnit u = quad_unit(a, block);
    const int lane = point_lane(), row = QUAD * u.g + wv;
    for (; redo; redo &= redo - 1) {
        const int col = u.w0 + __builtin_ctz(redo);
        if (PASS == FWD) diff_point_forward<T, D / 16>(a, u.b, u.h, u.bh, row, col, lane);
        if (PASS == DQ) diff_point_dq<T, D / 16>(a, u.b, u.h, u.bh, row, col, lane);
        if (PASS == DKDV) diff_point_dkdv<T, D / 16>(a, u.b, u.h, u.bh, row, col, lane);
    }
}

// Registers decide how many wavefronts a SIMD holds; where the compiler comes close to one more by itself, the launch bounds ask for it.  361x720, 64
// channels: dk/dv pass 143 registers, three wavefronts 379 us / 128, four 326; dq 356 / 330 (four); forward 110, four 287 / 96, five 267.  (Asked for more
// than fits, the loop spills: the forward with fourteen registers too few took 441.)

// ---- forward -------------------------------------------------------------------------------------------------------------------
template <typename T, int D, bool PAD> __global__ __launch_bounds__(64 * NW, D == 32 ? 6 : D == 128 ? 3 : PAD ? 4 : 5) void fwd_d16_kernel(const DArgs a)
{
    typedef DiffStage<D, PAD> Tile;
    typedef H16<T> M;
    constexpr int PITCH = Tile::PITCH, NCB = D / 16;
    extern __shared__ __attribute__((aligned(16))) char h16_lds[];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, qd = lane >> 4, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const QuadUnit u = quad_unit(a, blockIdx.x);
    const int bh = u.bh, b = u.b, h = u.h, w0 = u.w0;
    const int ho = min(QUAD * u.g + wv, a.Ho - 1); // (a latitude that is not there sees nothing and stores nothing)
    const int nk = PAD ? a.dk_ : D, nv = PAD ? a.dv_ : D, d = nk / 2;
    const char *kx = static_cast<const char *>(a.k) + ((size_t)b * a.Hi * a.Wi * a.ldk + (size_t)h * nk) * 2;
    const char *vx = static_cast<const char *>(a.v) + ((size_t)b * a.Hi * a.Wi * a.ldv + (size_t)h * nv) * 2;
    const bool mine = QUAD * u.g + wv < a.Ho && w0 + c < a.Wo;
    const size_t pt = (size_t)query_point(a, b, ho, a.qps == 1 ? ho : ho / a.qps) + (size_t)(w0 + (mine ? c : 0)) * a.qps;

    DiffOwn<M, D, PAD> own;
    own.load(static_cast<const char *>(a.q) + (pt * a.ldq + (size_t)h * nk) * 2, qd, d);
    f4v acc[2][NCB]; // Y^T of each map: register v of block cb is channel 16 cb + 4 qd + v of column c; sums of probabilities
#pragma unroll
    for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int cb = 0; cb < NCB; cb++) acc[i][cb] = f4v{0.f, 0.f, 0.f, 0.f};
    }
    float m[2] = {NEG_BIG, NEG_BIG}, Z[2] = {0.f, 0.f};

    QuadWalk wk;
    Tile bd = {}; // the next step's rows, on their way
    const unsigned lda = 2u * a.ldk * a.kps, ldb = 2u * a.ldv * a.kps; // bytes between two columns of a virtual input latitude
    auto fetch = [&]() {
        const size_t row = quad_row(wk.lat, wk.aux, a.kps, a.Wi);
        bd.w = a.quad_w[wk.aux + wk.zero];
        bd.fetch(kx + 2 * row * a.ldk, vx + 2 * row * a.ldv, tid, wk.column(w0), a.Wi, wk.rows(), lda, ldb, nk, nv);
    };
    char *buf = h16_lds, *other = h16_lds + Tile::BYTES;
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
            const float lw = fast_log2(weight);
            const char *kblk[2] = {buf, buf + 16 * PITCH}, *vblk[2] = {buf + HK * PITCH, buf + (HK + 16) * PITCH};
            f4v sc[2][2]; // [map][block]
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                sc[0][kb] = sc[1][kb] = f4v{0.f, 0.f, 0.f, 0.f};
                own.scores(sc[0][kb], sc[1][kb], kblk[kb], c, qd);
            }
            const int tb = cur.first(c) + 4 * qd; // neighbor index of element (kb, v): tb + 16 kb + v
            if (!cur.inner()) {
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int v = 0; v < 4; v++) {
                        const bool in = (unsigned)(tb + 16 * kb + v) < (unsigned)cur.l;
                        sc[0][kb][v] = in ? sc[0][kb][v] : -INFINITY;
                        sc[1][kb][v] = in ? sc[1][kb][v] : -INFINITY;
                    }
            }
            float mx[2];
#pragma unroll
            for (int i = 0; i < 2; i++)
                mx[i] = fmaxf(fmaxf(fmaxf(sc[i][0][0], sc[i][0][1]), fmaxf(sc[i][0][2], sc[i][0][3])), fmaxf(fmaxf(sc[i][1][0], sc[i][1][1]), fmaxf(sc[i][1][2], sc[i][1][3])));
            // The running maxima are only the reference points of the exponentials: see fwd_h16_kernel.
            if (__any(fmaf(mx[0], LOG2E, lw) > m[0] + RESCALE_THR || fmaf(mx[1], LOG2E, lw) > m[1] + RESCALE_THR)) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float cm = fmaf(h16_quarter_max(mx[i]), LOG2E, lw);
                    const float mn = (cm > m[i] + RESCALE_THR) ? cm : m[i]; // m starts finite, so mn is finite
                    const float corr = fast_exp2(m[i] - mn);
                    Z[i] *= corr;
#pragma unroll
                    for (int cb = 0; cb < NCB; cb++) acc[i][cb] *= corr;
                    m[i] = mn;
                }
            }
            uint4 p[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float sh = lw - m[i];
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int v = 0; v < 4; v++) sc[i][kb][v] = fast_exp2(fmaf(sc[i][kb][v], LOG2E, sh)); // masked: exp2(-inf) = 0
                p[i] = d16_pack<M>(sc[i]);
                Z[i] = d16_sum<T>(Z[i], p[i]); // this lane's share
            }
#pragma unroll
            for (int cb = 0; cb < NCB; cb++) {
                const uint4 vt = h16_read_transposed<PITCH>(vblk[0], vblk[1], cb, c, qd);
                acc[0][cb] = M::mfma(vt, p[0], acc[0][cb]);
                acc[1][cb] = M::mfma(vt, p[1], acc[1][cb]);
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
        char *y = static_cast<char *>(a.y) + (pt * a.ldy + (size_t)h * nv + 4 * qd) * 2;
        char *y2 = static_cast<char *>(a.y2) + ((pt * a.nh + h) * nv + 4 * qd) * 2;
#pragma unroll
        for (int cb = 0; cb < NCB; cb++)
            if (!PAD || 16 * cb + 4 * qd < nv) {
                const f4v o2 = acc[1][cb] * i1, o = acc[0][cb] * i0 - lam * o2;
                *reinterpret_cast<uint2 *>(y + 32 * cb) = make_uint2(M::pack2(o[0], o[1]), M::pack2(o[2], o[3]));
                if (a.y2) *reinterpret_cast<uint2 *>(y2 + 32 * cb) = make_uint2(M::pack2(o2[0], o2[1]), M::pack2(o2[2], o2[3]));
            }
    }
    if (__builtin_expect(redo != 0, 0)) diff_redo<T, D, FWD>(wv, blockIdx.x, redo);
}

// ---- backward, dq pass -----------------------------------------------------------------------------------------------------------
// Per step and map S^T = K Q^T; G^T = V dY^T once; dQ^T += K^T dS^T, and AK^T += K^T P^T and sum dS for the corrections of D.
template <typename T, int D, bool PAD> __global__ __launch_bounds__(64 * NW, D == 64 && !PAD ? 4 : 1) void dq_d16_kernel(const DArgs a)
{
    typedef DiffStage<D, PAD> Tile;
    typedef H16<T> M;
    constexpr int PITCH = Tile::PITCH, NS = D / 32, NCB = D / 16;
    extern __shared__ __attribute__((aligned(16))) char h16_lds[];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, qd = lane >> 4, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const QuadUnit u = quad_unit(a, blockIdx.x);
    const int bh = u.bh, b = u.b, h = u.h, w0 = u.w0;
    const int ho = min(QUAD * u.g + wv, a.Ho - 1); // (a latitude that is not there sees nothing and stores nothing)
    const int nk = PAD ? a.dk_ : D, nv = PAD ? a.dv_ : D, d = nk / 2;
    const char *kx = static_cast<const char *>(a.k) + ((size_t)b * a.Hi * a.Wi * a.ldk + (size_t)h * nk) * 2;
    const char *vx = static_cast<const char *>(a.v) + ((size_t)b * a.Hi * a.Wi * a.ldv + (size_t)h * nv) * 2;
    const bool mine = QUAD * u.g + wv < a.Ho && w0 + c < a.Wo;
    const size_t pt = (size_t)query_point(a, b, ho, a.qps == 1 ? ho : ho / a.qps) + (size_t)(w0 + (mine ? c : 0)) * a.qps;
    const size_t sidx = ((size_t)bh * a.Ho + ho) * a.Wo + w0 + (mine ? c : 0);
    const float lam = load_as_f32(a.lam, h, a.lam_dtype);

    DiffOwn<M, D, PAD> own;
    own.load(static_cast<const char *>(a.q) + (pt * a.ldq + (size_t)h * nk) * 2, qd, d);
    uint4 gop[NS];
    float D1 = 0.f, D2 = 0.f;
#pragma unroll
    for (int s = 0; s < NS; s++) {
        const bool ok = !PAD || 32 * s + 8 * qd < nv;
        const size_t off = 16 * qd + 64 * s;
        gop[s] = h16_load_piece(static_cast<const char *>(a.dy) + (pt * a.ldg + (size_t)h * nv) * 2 + off, ok);
        const uint4 yv = h16_load_piece(static_cast<const char *>(a.ysaved) + (pt * a.ldy + (size_t)h * nv) * 2 + off, ok);
        const uint4 y2 = h16_load_piece(static_cast<const char *>(a.y2saved) + (pt * a.nh + h) * nv * 2 + off, ok);
        const unsigned gu[4] = {gop[s].x, gop[s].y, gop[s].z, gop[s].w}, yu[4] = {yv.x, yv.y, yv.z, yv.w}, y2u[4] = {y2.x, y2.y, y2.z, y2.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 g_ = M::unpack2(gu[i]), y_ = M::unpack2(yu[i]), y2_ = M::unpack2(y2u[i]);
            D1 = fmaf(g_.x, y_.x, D1), D1 = fmaf(g_.y, y_.y, D1);
            D2 = fmaf(g_.x, y2_.x, D2), D2 = fmaf(g_.y, y2_.y, D2);
        }
    }
    D2 = h16_quarter_sum(D2);
    D1 = fmaf(lam, D2, h16_quarter_sum(D1));
    float2 lse = a.lse2[sidx];

    DiffSum<M, D, PAD> acc, ak;
    acc.zero(), ak.zero();
    float off[2] = {0.f, 0.f};

    QuadWalk wk;
    Tile bd = {}; // the next step's rows, on their way
    const unsigned lda = 2u * a.ldk * a.kps, ldb = 2u * a.ldv * a.kps; // bytes between two columns of a virtual input latitude
    auto fetch = [&]() {
        const size_t row = quad_row(wk.lat, wk.aux, a.kps, a.Wi);
        bd.w = a.quad_w[wk.aux + wk.zero];
        bd.fetch(kx + 2 * row * a.ldk, vx + 2 * row * a.ldv, tid, wk.column(w0), a.Wi, wk.rows(), lda, ldb, nk, nv);
    };
    char *buf = h16_lds, *other = h16_lds + Tile::BYTES;
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
    settle(gop);
    settle(lse.x), settle(lse.y);
    const float step21 = D1 - D2; // g - D2 = (g - D1) + (D1 - D2)

    while (cur.some) {
        wk.follow();
        fetch();
        if (cur.seen()) {
            const float lw = fast_log2(weight), l0 = lw - lse.x, l1 = lw - lse.y;
            const char *kblk[2] = {buf, buf + 16 * PITCH}, *vblk[2] = {buf + HK * PITCH, buf + (HK + 16) * PITCH};
            // g starts at -D1, so the matrix cores hand back g - D1.  (The scores could start at log2 w - lse with log2 e in q's operand: rounding
            // that to 16 bits again moves a score of s by s 2^-9, and so every p alike: half of the error of the gradients, and no faster.)
            f4v sc[2][2], gc[2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                sc[0][kb] = sc[1][kb] = f4v{0.f, 0.f, 0.f, 0.f};
                gc[kb] = f4v{-D1, -D1, -D1, -D1};
                own.scores(sc[0][kb], sc[1][kb], kblk[kb], c, qd);
#pragma unroll
                for (int s = 0; s < NS; s++) gc[kb] = M::mfma(h16_read_row<PITCH>(vblk[kb], s, c, qd), gop[s], gc[kb]);
            }
            const int tb = cur.first(c) + 4 * qd;
            const bool inner = cur.inner(); // every element of the step is a neighbor: no band mask
            f4v ds[2][2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const bool in = inner || (unsigned)(tb + 16 * kb + v) < (unsigned)cur.l;
                    sc[0][kb][v] = in ? fast_exp2(fmaf(sc[0][kb][v], LOG2E, l0)) : 0.f;
                    sc[1][kb][v] = in ? fast_exp2(fmaf(sc[1][kb][v], LOG2E, l1)) : 0.f;
                    ds[0][kb][v] = sc[0][kb][v] * gc[kb][v];
                    ds[1][kb][v] = sc[1][kb][v] * (gc[kb][v] + step21);
                }
            const uint4 p0 = d16_pack<M>(sc[0]), p1 = d16_pack<M>(sc[1]), d0 = d16_pack<M>(ds[0]), d1 = d16_pack<M>(ds[1]);
            off[0] = d16_sum<T>(off[0], d0), off[1] = d16_sum<T>(off[1], d1); // this lane's share
#pragma unroll
            for (int cb = 0; cb < NCB; cb++) {
                const uint4 kt = h16_read_transposed<PITCH>(kblk[0], kblk[1], cb, c, qd);
                acc.add(cb, kt, d0, d1, d);
                ak.add(cb, kt, p0, p1, d);
            }
            if (PAD) {
                const uint4 kt = h16_read_transposed<PITCH>(kblk[0], kblk[1], d / 16, c, qd);
                acc.add_both(kt, d1);
                ak.add_both(kt, p1);
            }
        }
        bd.commit(other, tid);
        weight = bd.w;
        __syncthreads();
        char *t = buf;
        buf = other, other = t;
        cur = wk.step();
    }

    // (stored after the walk: a global store ahead of the loop would turn the loop's scalar loads of runs and weights,
    // which the compiler only uses while nothing in the kernel can have written memory, into vector loads with waits)
    const float o0 = h16_quarter_sum(off[0]), o1 = h16_quarter_sum(off[1]);
    float check = o0 + o1;
#pragma unroll
    for (int cb = 0; cb < NCB; cb++) check += point_sum(acc.acc[cb] + ak.acc[cb]);
    if (PAD) check += point_sum(acc.both + ak.both);
    const unsigned redo = point_columns(mine && not_finite(check));
    float part = 0.f;
    if (mine) {
        // (a column that is evaluated again may hold a value here that it does not see)
        const float s2 = not_finite(o1) ? D2 : D2 + o1;
        part = qd == 0 ? s2 : 0.f;
        if (qd == 0) a.dstats[sidx] = make_float4(lse.x, lse.y, D1 + o0, s2);
        char *dq = static_cast<char *>(a.dq) + (pt * a.lddq + (size_t)h * nk + 4 * qd) * 2;
#pragma unroll
        for (int cb = 0; cb < NCB; cb++)
            if (!PAD || 16 * cb + 4 * qd < nk) {
                const bool first = acc.first(cb, qd, d);
                f4v x = acc.value(cb, qd, d) - (first ? o0 : o1) * ak.value(cb, qd, d);
                x *= first ? 1.f : -lam;
                *reinterpret_cast<uint2 *>(dq + 32 * cb) = make_uint2(M::pack2(x[0], x[1]), M::pack2(x[2], x[3]));
            }
    }
    if (QUAD * u.g + wv < a.Ho) {
        part = point_lanes_sum(part);
        if (lane == 0) a.lam_part[(size_t)bh * a.lam_n + (size_t)ho * ((a.Wo + HQ - 1) / HQ) + w0 / HQ] = part;
    }
    if (__builtin_expect(redo != 0, 0)) diff_redo<T, D, DQ>(wv, blockIdx.x, redo);
}

// ---- backward, dk/dv pass: transposed gather (see dkdv_h16_kernel) -------------------------------------------------------------------
// Per step and map S = Q K^T; G = dY V^T once; dV^T += dY^T (P1 - lam P2) once; dK^T += Q^T dS.
// The statistics of the staged queries lie behind the buffers, log2 w - lse of the two maps, -D1 and D1 - D2, each for 32 rows, so a lane reads
// those of its four queries at once.  (The key's log2 w is added to the first two in 32 bits.)
template <typename T, int D, bool PAD> __global__ __launch_bounds__(64 * NW, PAD || D == 128 ? 1 : D == 64 ? 4 : 5) void dkdv_d16_kernel(const DArgs a)
{
    typedef DiffStage<D, PAD> Tile;
    typedef H16<T> M;
    constexpr int PITCH = Tile::PITCH, NS = D / 32, NCB = D / 16;
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
    const char *qy = static_cast<const char *>(a.q) + ((size_t)b * a.Ho * a.Wo * a.ldq + (size_t)h * nk) * 2;
    const char *gy = static_cast<const char *>(a.dy) + ((size_t)b * a.Ho * a.Wo * a.ldg + (size_t)h * nv) * 2;
    const float4 *stats = a.dstats + (size_t)bh * a.Ho * a.Wo;
    const bool mine = QUAD * u.g + wv < a.Hi && w0 + c < a.Wi;
    const size_t pt = (size_t)key_point(a, b, hi, a.kps == 1 ? hi : hi / a.kps) + (size_t)(w0 + (mine ? c : 0)) * a.kps;
    float lam = load_as_f32(a.lam, h, a.lam_dtype);

    DiffOwn<M, D, PAD> own;
    own.load(static_cast<const char *>(a.k) + (pt * a.ldk + (size_t)h * nk) * 2, qd, d);
    uint4 vop[NS];
#pragma unroll
    for (int s = 0; s < NS; s++) vop[s] = h16_load_piece(static_cast<const char *>(a.v) + (pt * a.ldv + (size_t)h * nv) * 2 + 16 * qd + 64 * s, !PAD || 32 * s + 8 * qd < nv);
    DiffSum<M, D, PAD> dkt;
    dkt.zero();
    f4v dvt[NCB];
#pragma unroll
    for (int cb = 0; cb < NCB; cb++) dvt[cb] = f4v{0.f, 0.f, 0.f, 0.f};
    const float lw = fast_log2(a.quad_w[a.kps == 1 ? hi : hi / a.kps]);

    QuadWalk wk;
    Tile bd = {}; // the next step's rows, on their way
    const unsigned lda = 2u * a.ldq * a.qps, ldb = 2u * a.ldg * a.qps; // bytes between two columns of a virtual output latitude
    auto fetch = [&]() {
        const size_t row = quad_row(wk.lat, wk.aux, a.qps, a.Wo);
        const int cs = wk.column(w0), n = wk.rows();
        bd.fetch(qy + 2 * row * a.ldq, gy + 2 * row * a.ldg, tid, cs, a.Wo, n, lda, ldb, nk, nv);
        int col = cs + min(tid & (HK - 1), n - 1); // (the first threads' are used)
        if (col >= a.Wo) col -= a.Wo;
        bd.st = stats[(size_t)wk.lat * a.Wo + col];
    };
    auto commit = [&](char *to) {
        bd.commit(to, tid);
        if (tid < HK) {
            float *t = reinterpret_cast<float *>(to + Tile::BYTES) + tid;
            t[0] = -bd.st.x, t[HK] = -bd.st.y, t[2 * HK] = -bd.st.z, t[3 * HK] = bd.st.z - bd.st.w;
        }
    };
    char *buf = h16_lds, *other = h16_lds + Tile::BYTES + HK * 16;
    wk.start(a, u, wv, lane);
    QuadStep cur = wk.step();
    if (cur.some) {
        fetch();
        commit(buf);
    }
    __syncthreads();
    own.settle_();
    settle(vop);
    settle(lam);

    while (cur.some) {
        wk.follow();
        fetch();
        if (cur.seen()) {
            const char *qblk[2] = {buf, buf + 16 * PITCH}, *gblk[2] = {buf + HK * PITCH, buf + (HK + 16) * PITCH};
            const float *stat = reinterpret_cast<const float *>(buf + Tile::BYTES) + 4 * qd;
            f4v sc[2][2], gc[2], l0[2], l1[2], step21[2];
#pragma unroll
            for (int qb = 0; qb < 2; qb++) {
                sc[0][qb] = sc[1][qb] = f4v{0.f, 0.f, 0.f, 0.f};
                l0[qb] = *reinterpret_cast<const f4v *>(stat + 16 * qb) + lw;
                l1[qb] = *reinterpret_cast<const f4v *>(stat + 16 * qb + HK) + lw;
                gc[qb] = *reinterpret_cast<const f4v *>(stat + 16 * qb + 2 * HK);
                step21[qb] = *reinterpret_cast<const f4v *>(stat + 16 * qb + 3 * HK);
                own.scores(sc[0][qb], sc[1][qb], qblk[qb], c, qd);
#pragma unroll
                for (int s = 0; s < NS; s++) gc[qb] = M::mfma(h16_read_row<PITCH>(gblk[qb], s, c, qd), vop[s], gc[qb]);
            }
            const int tb = cur.first(c) + 4 * qd; // r - c of element (qb, v): tb + 16 qb + v
            const bool inner = cur.inner(); // every element of the step is a (query, key) pair of the band
            f4v ds[2][2], co[2];
#pragma unroll
            for (int qb = 0; qb < 2; qb++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    const bool in = inner || (unsigned)(tb + 16 * qb + v) < (unsigned)cur.l;
                    const float p0 = in ? fast_exp2(fmaf(sc[0][qb][v], LOG2E, l0[qb][v])) : 0.f, p1 = in ? fast_exp2(fmaf(sc[1][qb][v], LOG2E, l1[qb][v])) : 0.f;
                    co[qb][v] = fmaf(-lam, p1, p0);
                    ds[0][qb][v] = p0 * gc[qb][v];
                    ds[1][qb][v] = p1 * (gc[qb][v] + step21[qb][v]);
                }
            const uint4 cop = d16_pack<M>(co), d0 = d16_pack<M>(ds[0]), d1 = d16_pack<M>(ds[1]);
#pragma unroll
            for (int cb = 0; cb < NCB; cb++) {
                dvt[cb] = M::mfma(h16_read_transposed<PITCH>(gblk[0], gblk[1], cb, c, qd), cop, dvt[cb]);
                dkt.add(cb, h16_read_transposed<PITCH>(qblk[0], qblk[1], cb, c, qd), d0, d1, d);
            }
            if (PAD) dkt.add_both(h16_read_transposed<PITCH>(qblk[0], qblk[1], d / 16, c, qd), d1);
        }
        commit(other);
        __syncthreads();
        char *t = buf;
        buf = other, other = t;
        cur = wk.step();
    }

    float check = 0.f;
#pragma unroll
    for (int cb = 0; cb < NCB; cb++) check += point_sum(dkt.acc[cb] + dvt[cb]);
    if (PAD) check += point_sum(dkt.both);
    const unsigned redo = point_columns(mine && not_finite(check));
    if (mine) {
        char *dk = static_cast<char *>(a.dk) + (pt * a.lddk + (size_t)h * nk + 4 * qd) * 2, *dv = static_cast<char *>(a.dv) + (pt * a.lddv + (size_t)h * nv + 4 * qd) * 2;
#pragma unroll
        for (int cb = 0; cb < NCB; cb++) {
            if (!PAD || 16 * cb + 4 * qd < nk) {
                const f4v x = dkt.value(cb, qd, d) * (dkt.first(cb, qd, d) ? 1.f : -lam);
                *reinterpret_cast<uint2 *>(dk + 32 * cb) = make_uint2(M::pack2(x[0], x[1]), M::pack2(x[2], x[3]));
            }
            if (!PAD || 16 * cb + 4 * qd < nv) *reinterpret_cast<uint2 *>(dv + 32 * cb) = make_uint2(M::pack2(dvt[cb][0], dvt[cb][1]), M::pack2(dvt[cb][2], dvt[cb][3]));
        }
    }
    if (__builtin_expect(redo != 0, 0)) diff_redo<T, D, DKDV>(wv, block, redo);
}
