// The walk of the differential matrix-core kernels.  Included by s2attn_kernels.hip inside namespace s2 after s2attn_diff.hpp.
//
// A workgroup owns sixteen columns of four adjacent latitudes, a latitude per wavefront, and walks the bands of the other grid that any of them
// sees (build_quads in s2attn_plan.cpp) in steps of 32 band positions: all four wavefronts stage the step's rows of two tensors, and those
// whose latitude sees any of them work on them.  Position t of a band is column ws + w0 + t of its latitude; point c of the tile sees
// t in [c + d, c + d + l), or t in [0, W) where its latitude sees the whole ring.
//
// Rows staged for 64 points, disk of radius R rings, arcs of a columns: (2 R + 4) (15 + a); with a latitude's 64 columns in the four wavefronts
// (2 R + 1) (63 + a), in a ring of 128 (80) rows with two barriers a run.  Forward, dq and dk/dv took, us, that way / this way: 361x720 bf16 4 x 64
// channels, R = 2: 269 / 267, 341 / 330, 369 / 326; 180x360 from 90x180 bf16 2 x 128 channels: 92 / 56, 98 / 68, 142 / 120; 128x256 fp32 4 x 32 channels
// R = 4: 250 / 205, 252 / 220, 303 / 279; 91x180 bf16 forward alone, which is as long as its longest walk: 24 / 26.
// Whole rings as such, in W positions: the last one 26.5 -> 24.5; 91x181 fp32 3 x 40 channels 77 -> 68, 75 -> 73, 106 -> 95.
//
// Two buffers, one barrier a step.  Bound by issue: vector instructions keep the SIMDs busy half the time, matrix instructions a tenth (16-bit) to a
// quarter, at 3 to 5 wavefronts per SIMD, as registers allow.

constexpr int QUAD = 4;           // latitudes of a workgroup (= NW)
constexpr int QUAD_RING = 0xffff; // (see build_quads)
static_assert(QUAD == NW, "a latitude per wavefront");

struct QuadUnit {
    int bh, b, h, g, w0; // (batch, head), group of latitudes, first column
    int first, last;     // its bands
};
// (divisors are known to the host: a division by a variable takes 35 instructions of the scalar unit, this one three)
__device__ inline int quad_div(const QuadDiv &d, int n) { return (int)((unsigned long)(unsigned)n * d.m >> d.s); }
__device__ inline QuadUnit quad_unit(const DArgs &a, int block)
{
    QuadUnit u;
    const int BH = a.B * a.nh, nt = (a.Wi + HQ - 1) / HQ;
    int id;
    if ((BH & 7) == 0) { // as xcd_split
        const int r = block >> 3, x = quad_div(a.q_first, r);
        u.bh = (block & 7) + 8 * x, id = r - x * a.q_groups * nt;
    } else {
        id = quad_div(a.q_first, block), u.bh = block - id * BH;
    }
    const int n = quad_div(a.q_tiles, id);
    u.w0 = HQ * (id - n * nt);
    u.b = quad_div(a.q_head, u.bh), u.h = u.bh - u.b * a.nh;
    const int4 group = *reinterpret_cast<const int4 *>(a.q_list + 4 * (size_t)n);
    u.g = group.x, u.first = group.y, u.last = group.z;
    return u;
}

// A step of the walk as its products need it
struct QuadStep {
    bool some;
    int pos;  // first position of its band
    int d, l; // what the wavefront's latitude sees of the band
    bool ring;
    // does any point of the wavefront see any of the positions; do all see all
    __device__ inline bool seen() const { return l > 0 && pos + HK > d && pos < d + l + (ring ? 0 : HQ - 1); }
    __device__ inline bool inner() const { return pos - d >= (ring ? 0 : HQ - 1) && pos - d + HK <= l; }
    // point c sees position r of the step iff 0 <= first(c) + r < l
    __device__ inline int first(int c) const { return pos - d - (ring ? 0 : c); }
};

// Where the walk's loads are: the step to fetch, and the band after its own, read while that is worked on.  All that a step loads, it loads in every
// step and in one order with vector loads, so that each is waited for by itself: under a condition, or mixed with scalar loads, which return out of
// order, the compiler waits for all.
struct QuadWalk {
    const int *bands;
    int wv, word, zero; // word: lane % 8; zero: 0, in a vector register
    int W;
    int band, end, pos;
    int lat, aux, ws, len, dl;
    int ahead; // int `word` of the band after

    __device__ inline void read() { ahead = bands[8 * (size_t)min(band + 1, end) + word]; } // (one band follows the last)
    __device__ inline void take()
    {
        lat = __builtin_amdgcn_readlane(ahead, 0), aux = __builtin_amdgcn_readlane(ahead, 1), ws = __builtin_amdgcn_readlane(ahead, 2), len = __builtin_amdgcn_readlane(ahead, 3);
        dl = __builtin_amdgcn_readlane(ahead, 4 + wv);
    }
    __device__ inline void start(const DArgs &a, const QuadUnit &u, int wv_, int lane)
    {
        bands = a.q_bands, wv = wv_, word = lane & 7, zero = 0, W = a.Wi, end = u.last, pos = 0;
        asm("" : "+v"(zero));
        band = u.first - 1;
        read();
        take();
        band++;
        read();
    }
    __device__ inline bool more() const { return band < end; }
    // to the next step; after the last one the walk stays at it, with more() false
    __device__ inline void follow()
    {
        const bool turn = pos + HK >= len + HQ - 1;
        if (turn) band = min(band + 1, end);
        if (turn && more()) {
            take();
            pos = 0;
        } else if (!turn) {
            pos += HK;
        }
        read();
    }
    __device__ inline QuadStep step() const
    {
        const bool ring = dl == QUAD_RING;
        return QuadStep{more(), pos, ring ? 0 : dl >> 16, ring ? W : dl & 0xffff, ring};
    }
    // first column of the step, in [0, W)
    __device__ inline int column(int w0) const
    {
        int c = ws + w0 + pos;
        while (c >= W) c -= W;
        return c;
    }
    __device__ inline int rows() const { return more() ? min(HK, len + HQ - 1 - pos) : 1; }
};

// Point index of column 0 of a latitude inside a batch entry (ratio: of its grid)
__device__ inline unsigned quad_row(int vlat, int rlat, int ratio, int W) { return (unsigned)rlat * ratio * W + (vlat - rlat * ratio); }

// A step's 32 rows of two tensors on their way to LDS: piece p of row r of tensor t by thread 32 CPR t + CPR r + p (modulo the workgroup)
template <int CPR> struct QuadPieces {
    static constexpr int N = (2 * HK * CPR + 64 * NW - 1) / (64 * NW); // per thread
    static __device__ inline int at(int it, int tid) { return tid + 64 * NW * it; }
    static __device__ inline bool second(int i) { return i >= HK * CPR; }
    static __device__ inline bool on(int i) { return 2 * HK * CPR % (64 * NW) == 0 || i < 2 * HK * CPR; }
    static __device__ inline int row(int i) { return i % (HK * CPR) / CPR; }
    static __device__ inline int piece(int i) { return i % CPR; }
};
