// esr_wgrad8.hip — a convolution's weight gradient from an input kept in 8-bit blocks (esr_act8.h):
//   gw[co][ci][ky][kx] = Σ_{b, Y, X} x[b, s·Y + ky − p, s·X + kx − p, ci] · dy[b, Y, X, co]   (x zero outside the image)
// One matrix product per tap, M = ci, N = co, K = output pixels, on v_mfma_f32_32x32x16_f16.  A code is an integer of 7
// bits times a power of two, so x is ONE exact f16 number (at a scale of the workgroup's largest exponent; a block more
// than 2^27 below it counts as zero, a subnormal f16's sums round like those of 2^-14), and only dy is split, into hi +
// lo f16 at a power-of-two scale of the largest |dy| so far (|dy − hi − lo| <= 2^-22 |dy| + 2^-36 of that largest): two
// products where fp32 x takes three, and a quarter of its bytes.  The scales leave room for a growth of 2^4 (dy) and 2^2
// (x); a tile beyond that raises a flag, and the workgroup finds its maxima, rescales the float32 accumulators by the
// exact power of two and stages the tile again.
//
// A workgroup owns 64 ci × 64 co and ALL the taps of a tap group (3×3: nine; 4×4 stride 2: sixteen; 4×4 stride 1: two
// rows; 8×8: one row), a wave one 32×32 tile for each of up to nine taps: dy is expanded once per K step for all of
// them, and the halo tile of x as well.  K step = RY rows × 16 columns of one image, so that a row of 16 pixels is one
// MFMA's K and a tap is an LDS address offset.  Both operands lie pixel-major in LDS and are read transposed
// (ds_read_b64_tr_b16), 32-byte chunks XOR-swizzled by pixel so that the four pixels of a read cover the banks once; at
// stride 2 the even and the odd columns of x lie apart, which makes a tap's pixels neighbours again.  Two LDS tiles: one
// is multiplied while the next is expanded into the other and the one after that is on its way into registers, one
// barrier per step.  Two workgroups of four waves share a CU (4×4 stride 2: one of eight, half of whose waves multiply
// first and expand second), so that one's expansion runs under the other's MFMAs.  The pixels are split over the grid,
// the partial sums added in a fixed order by a second launch into torch's weight layout.
//
// 3×3, 64 -> 128 channels, 16×152×152 pixels: 108 to 120 us back to back and 14 us of reduction, 0.9 to 1.0 PFLOP/s of f16
// products (two for each of the definition's) where a large f16 matrix product reaches 1.2 on this card; 4×4 stride 2,
// 64 -> 64, 16×304×304: 103 to 113 and 12 us, 0.86 to 0.94.  The matrix pipes are busy 57 and 53 % of the cycles, at a
// clock of 2.06 and 2.12 GHz; what the rest goes to (LDS reads, expansion, the first tile and the partial sums, which have
// no MFMA beside them) has not been taken apart.
#include "esr_act8.h"
#include "esr_amd.h"
#include "esr_knobs.h"
#include "esr_wgrad8_map.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int NT = 256;

struct WgP {
    const int8_t *codes;
    const uint8_t *exps;
    const float *dy;
    int B, Hs, Ws, cin, cp, nb, MH, MW, cout, k, s, p, nci, nco, groups;
    int Hr, Wr;                            // rows and columns of x that an output reads (non-finite ones behind them count not)
    int tY, tX, tiles, per_split, splits;  // K steps: rows and columns of tiles per image, all, per split
    float *partial;                        // [splits][k·k][nci·64][nco·64]
};

__device__ __forceinline__ f16x8 tr_pair(const unsigned char *lds, int at, int step) {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(lds + at));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(lds + at + step));
    return __builtin_bit_cast(f16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// two codes (bytes of w ^ 0x80808080, picked by sel) times s as f16: the byte in the mantissa of 1024 is 1024 + 128 +
// code, and one fused multiply-add leaves the exact code·s (s a power of two <= 2^5; off = −1152·s)
__device__ __forceinline__ f16x2 code_pair(uint32_t w, uint32_t sel, f16x2 s, f16x2 off) {
    return __builtin_elementwise_fma(__builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, sel)), s, off);
}

// S: the LDS tile's stride between the pixels of a tap; a group of one tap stages exactly its pixels (any stride).
// TG: tap groups of a workgroup, four waves each.
template <int KR, int KC, int S, int TG>
struct Shape {
    static constexpr bool ONE = KR == 1 && KC == 1;
    static constexpr int RY = 4, NT = 256 * TG;
    static constexpr int ROWS = (RY - 1) * S + KR * TG, COLS = 15 * S + KC;
    static constexpr int HALF = ((COLS + S - 1) / S + 3) / 4 * 4, PITCH = HALF * S;  // pixels of a row in LDS
    static constexpr int KPX = RY * 16, XB = ROWS * PITCH * 128, BUF = XB + KPX * 256;
    static constexpr int NX = (ROWS * COLS * 4 + NT - 1) / NT, NG = KPX * 16 / NT;
};

// G4: four gradients at once (cout a multiple of 4), or one by one.
template <int KR, int KC, int S, int TG, bool G4>
__global__ __launch_bounds__(256 * TG, 2) void wgrad8_kernel(WgP p) {
    using H = Shape<KR, KC, S, TG>;
    constexpr int RY = H::RY;
    __shared__ __attribute__((aligned(16))) unsigned char lds[2 * H::BUF];
    __shared__ unsigned s_red[4 * TG][2];
    __shared__ int s_flag[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hl = lane >> 5;
    const wgrad8::Place place = wgrad8::place((int)blockIdx.x, p.splits, p.nci * p.nco * p.groups);
    const int split = place.split;
    int w = place.item;
    const int cob = w % p.nco;
    w /= p.nco;
    const int cib = w % p.nci, grp = w / p.nci;
    const int ci0 = cib * 64, co0 = cob * 64;
    const int oy = (H::ONE ? grp / p.k : grp * KR * TG) - p.p, ox = (H::ONE ? grp % p.k : 0) - p.p;
    const int t0 = split * p.per_split, t1 = min(p.tiles, t0 + p.per_split);

    // this thread's places: x pixel (row, column) and its 16 channels, their bytes in the LDS tile
    int xr[H::NX], xd[H::NX];
#pragma unroll
    for (int j = 0; j < H::NX; ++j) {
        const int idx = tid + j * H::NT, px = idx >> 2, ry = px / H::COLS, cx = px % H::COLS;
        const int pos = cx % S * H::HALF + cx / S;
        xr[j] = ry < H::ROWS && ci0 + 16 * (idx & 3) < p.cin ? ry << 16 | cx : -1;
        xd[j] = ry < H::ROWS ? (ry * H::PITCH + pos) * 128 + (((idx & 3) ^ (2 * ((pos >> 1) & 1))) << 5) : -1;
    }
    // Every load is issued, from the tensor's first element where its place is outside, and its value dropped when it is
    // expanded: no branch for which the loads in flight would have to be waited for.
    uint4 rx[H::NX];
    int re[H::NX], ok = 0;
    f32x4 rg[H::NG];
    auto load = [&](int t) {
        const int img = t / (p.tY * p.tX), r = t - img * p.tY * p.tX, ty = r / p.tX;
        const int Y0 = ty * RY, X0 = (r - ty * p.tX) * 16;
        const int st = H::ONE ? p.s : 1, ys = Y0 * (H::ONE ? p.s : S) + oy, xs = X0 * (H::ONE ? p.s : S) + ox;
        const long long pix0 = (long long)img * p.Hs * p.Ws;
        const int8_t *codes = p.codes + pix0 * p.cp;
        const uint8_t *exps = p.exps + pix0 * p.nb;
        const float *dy = p.dy + (long long)img * p.MH * p.MW * p.cout;
        ok = 0;
#pragma unroll
        for (int j = 0; j < H::NX; ++j) {
            const int sy = ys + (xr[j] >> 16) * st, sx = xs + (xr[j] & 0xffff) * st, ci = ci0 + 16 * (tid & 3);
            const bool in = xr[j] >= 0 && (unsigned)sy < (unsigned)p.Hr && (unsigned)sx < (unsigned)p.Wr;
            // (no branch; unsigned, for the places outside are computed too)
            const unsigned m = -(unsigned)in, pix = ((unsigned)sy * p.Ws + sx) & m, c = (unsigned)ci & m;
            ok |= (int)in << j;
            re[j] = exps[pix * (unsigned)p.nb + c / act8::BLK];
            rx[j] = *reinterpret_cast<const uint4 *>(codes + (pix * (unsigned)p.cp + c));
        }
#pragma unroll
        for (int j = 0; j < H::NG; ++j) {
            const int idx = tid + j * H::NT, q = idx >> 4, co = co0 + 4 * (idx & 15), Y = Y0 + (q >> 4), X = X0 + (q & 15);
            const bool in = Y < p.MH && X < p.MW && co < p.cout;
            const float *src = dy + (((unsigned)(Y * p.MW + X) * (unsigned)p.cout + co) & -(unsigned)in);
            ok |= (int)in << (16 + j);
            if constexpr (G4) {
                rg[j] = *reinterpret_cast<const f32x4 *>(src);
            } else {
                const int n = in ? p.cout - co : 1;
#pragma unroll
                for (int i = 0; i < 4; ++i) rg[j][i] = src[i < n ? i : 0];
            }
        }
    };
    auto drop = [&]() {  // the values that are outside
#pragma unroll
        for (int j = 0; j < H::NX; ++j) {
            const unsigned m = -(unsigned)(ok >> j & 1);
            re[j] &= m;
            rx[j] = make_uint4(rx[j].x & m, rx[j].y & m, rx[j].z & m, rx[j].w & m);
        }
#pragma unroll
        for (int j = 0; j < H::NG; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                rg[j][i] = (ok >> (16 + j) & 1) && (G4 || co0 + 4 * (tid & 15) + i < p.cout) ? rg[j][i] : 0.f;
    };

    f32x16 acc[KR * KC];
#pragma unroll
    for (int t = 0; t < KR * KC; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;
    int ex = 0, eg = -110;  // x is staged at 2^(135 − ex), dy at 2^(11 − eg)

    // The loaded tile's largest exponent byte and |dy| (finite ones) over the workgroup; the scales raised to them.
    auto rescale = [&]() {
        unsigned me = 0, mg = 0;
        drop();
#pragma unroll
        for (int j = 0; j < H::NX; ++j) me = max(me, re[j] == 255 ? 0u : (unsigned)re[j]);
#pragma unroll
        for (int j = 0; j < H::NG; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned b = act8::abs_bits(rg[j][i]);
                mg = max(mg, b >= 0x7f800000u ? 0u : b);
            }
        me = act8::block_max<64>(me);
        mg = act8::block_max<64>(mg);
        if (lane == 0) {
            s_red[wave][0] = me;
            s_red[wave][1] = mg;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4 * TG; ++i) {
            me = max(me, s_red[i][0]);
            mg = max(mg, s_red[i][1]);
        }
        const int ex2 = max(ex, (int)me), eg2 = max(eg, (int)(mg >> 23) - 126), down = ex2 - ex + eg2 - eg;
#pragma unroll
        for (int q = 0; q < KR * KC; ++q)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[q][r] = ldexpf(acc[q][r], -down);
        ex = __builtin_amdgcn_readfirstlane(ex2);
        eg = __builtin_amdgcn_readfirstlane(eg2);
    };
    // The loaded tile into an LDS tile; whether one of this thread's values is beyond the scales.
    auto expand = [&](unsigned char *buf) {
        int me = 0;
        drop();
#pragma unroll
        for (int j = 0; j < H::NX; ++j) {
            if (xd[j] < 0) break;
            me = max(me, re[j] == 255 ? 0 : re[j]);
            const _Float16 sc = re[j] == 255 ? (_Float16)__builtin_nanf("") : (_Float16)ldexpf(1.f, min(re[j] - ex, 2) + 3);
            const f16x2 s = {sc, sc}, off = s * (_Float16)-1152.f;
            const uint32_t q[4] = {rx[j].x, rx[j].y, rx[j].z, rx[j].w};
            f16x2 o[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = q[i] ^ 0x80808080u;
                o[2 * i] = code_pair(u, 0x04010400u, s, off);
                o[2 * i + 1] = code_pair(u, 0x04030402u, s, off);
            }
            *reinterpret_cast<uint4 *>(buf + xd[j]) = *reinterpret_cast<const uint4 *>(&o[0]);
            *reinterpret_cast<uint4 *>(buf + xd[j] + 16) = *reinterpret_cast<const uint4 *>(&o[4]);
        }
        unsigned mg = 0;
        const float sg = ldexpf(1.f, 11 - eg);
#pragma unroll
        for (int j = 0; j < H::NG; ++j) {
            const int idx = tid + j * H::NT, q = idx >> 4, c = 4 * (idx & 15);
            f16x4 h, l;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                mg = max(mg, act8::abs_bits(rg[j][i]));
                const float v = rg[j][i] * sg;
                h[i] = (_Float16)v;
                l[i] = (_Float16)(v - (float)h[i]);
            }
            const int d = H::XB + q * 256 + (((c >> 4) ^ (2 * (q & 3))) << 5) + (c & 15) * 2;
            *reinterpret_cast<f16x4 *>(buf + d) = h;
            *reinterpret_cast<f16x4 *>(buf + (((d - H::XB) ^ 128) + H::XB)) = l;
        }
        return me > ex + 2 || (int)(mg >> 23) - 126 > eg + 4;
    };

    // transposed-read lane roles: pixel rq of four, channels 16·(group of 16 lanes) + 4·(lane & 3) of a 32-channel tile
    const int wm = (wave >> 1) & 1, wn = wave & 1, tg = TG > 1 ? wave >> 2 : 0, i16 = lane & 15, rq = i16 >> 2;
    const int cb = 16 * ((lane >> 4) & 1) + 4 * (i16 & 3);
    int ax[KC];
#pragma unroll
    for (int b = 0; b < KC; ++b) {
        const int pos = (b % S) * H::HALF + 8 * hl + rq + b / S, c = 32 * wm + cb;
        ax[b] = (tg * KR * H::PITCH + pos) * 128 + (((c >> 4) ^ (2 * ((pos >> 1) & 1))) << 5) + (c & 15) * 2;
    }
    const int cg = 32 * wn + cb, ag = (8 * hl + rq) * 256 + (((cg >> 4) ^ (2 * rq)) << 5) + (cg & 15) * 2;
    auto multiply = [&](const unsigned char *buf) {
#pragma unroll
        for (int kq = 0; kq < RY; ++kq) {
            const f16x8 gh = tr_pair(buf + H::XB, ag + kq * 4096, 1024), gl = tr_pair(buf + H::XB, (ag ^ 128) + kq * 4096, 1024);
#pragma unroll
            for (int a = 0; a < KR; ++a)
#pragma unroll
                for (int b = 0; b < KC; ++b) {
                    const f16x8 x = tr_pair(buf, ax[b] + (kq * S + a) * H::PITCH * 128, 512);
                    acc[a * KC + b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, gl, acc[a * KC + b], 0, 0, 0);
                    acc[a * KC + b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, gh, acc[a * KC + b], 0, 0, 0);
                }
        }
    };

    if (tid < 2) s_flag[tid] = -1;
    load(t0);
    rescale();
    expand(lds);
    if (t0 + 1 < t1) load(t0 + 1);
    // (an int of unknown origin, once: where every value that meets in the loop's re[j] is a widened byte, the compiler
    // carries bytes, widens them behind each load and so waits for the load where it is issued)
#pragma unroll
    for (int j = 0; j < H::NX; ++j) asm("" : "+v"(re[j]));
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        unsigned char *now = lds + ((t - t0) & 1) * H::BUF, *next = lds + ((t - t0 + 1) & 1) * H::BUF;
        const bool more = t + 1 < t1;
        auto stage = [&]() {
            if (!more) return;
            const bool beyond = expand(next);
            if (__any(beyond) && lane == 0) s_flag[(t + 1) & 1] = t + 1;
            if (t + 2 < t1) load(t + 2);
        };
        if (TG == 1 || tg == 0) {
            stage();
            multiply(now);
        } else {
            multiply(now);
            stage();
        }
        __syncthreads();
        if (more && s_flag[(t + 1) & 1] == t + 1) {  // (the same for all: written before the barrier)
            load(t + 1);
            rescale();
            expand(next);
            if (t + 2 < t1) load(t + 2);
            __syncthreads();
        }
    }
    const int cip = p.nci * 64, cop = p.nco * 64, back = ex - 135 + eg - 11;
    const int tap0 = (grp * TG + tg) * KR * KC;
    float *dst = p.partial + (((long long)split * p.k * p.k + tap0) * cip + ci0 + 32 * wm) * cop + co0 + 32 * wn + (lane & 31);
#pragma unroll
    for (int t = 0; t < KR * KC; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            dst[((long long)t * cip + (r & 3) + 8 * (r >> 2) + 4 * hl) * cop] = ldexpf(acc[t][r], back);
}

// gw[co][ci][t] = Σ over the splits: 64 consecutive co (four to a thread: 256 bytes together) × 16 slices of the splits,
// a slice in order, then the slices.  (256 splits of 9×64×128 sums, 75 MB: 13 us; 32 co × 32 slices took 15.)
__global__ __launch_bounds__(NT) void wgrad8_reduce(const float *partial, int splits, int T, int cin, int cout, int cip,
                                                    int cop, float *gw) {
    __shared__ f32x4 sl[16][16];
    const int q = threadIdx.x >> 4, o = threadIdx.x & 15, nco = (cout + 63) / 64;
    const int co = blockIdx.x % nco * 64, row = blockIdx.x / nco, ci = row % cin, t = row / cin;
    const long long step = (long long)T * cip * cop;
    const float *src = partial + ((long long)t * cip + ci) * cop + co + 4 * o;  // (cop is a multiple of 64)
    const int s0 = splits * q / 16, s1 = splits * (q + 1) / 16;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int s = s0; s < s1; ++s) v += *reinterpret_cast<const f32x4 *>(src + s * step);
    sl[q][o] = v;
    __syncthreads();
    if (threadIdx.x < 64 && co + (int)threadIdx.x < cout) {
        const float *col = reinterpret_cast<const float *>(sl) + threadIdx.x;
        float s = col[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) s += col[64 * r];
        gw[((long long)(co + threadIdx.x) * cin + ci) * T + t] = s;
    }
}

// The same for many weights (and so few splits): a workgroup adds 32 co × cb ci × all taps (at most 64 of the latter two)
// and writes them by rows of one co, which lie together in gw (one by one, at a stride of cin·T, each would cost a
// sector).
__global__ __launch_bounds__(NT) void wgrad8_reduce_rows(const float *partial, int splits, int T, int cin, int cout, int cip,
                                                         int cop, int cb, float *gw) {
    __shared__ float tile[32][65];
    const int nco = (cout + 31) / 32, co0 = blockIdx.x % nco * 32, ci0 = blockIdx.x / nco * cb, n = min(cb, cin - ci0) * T;
    const long long step = (long long)T * cip * cop;
    for (int i = threadIdx.x; i < n * 8; i += NT) {
        const int o = 4 * (i & 7), r = i >> 3, ci = ci0 + r / T, t = r % T;
        const float *src = partial + ((long long)t * cip + ci) * cop + co0 + o;
        f32x4 v = *reinterpret_cast<const f32x4 *>(src);
#pragma unroll 4
        for (int s = 1; s < splits; ++s) v += *reinterpret_cast<const f32x4 *>(src + s * step);
#pragma unroll
        for (int k = 0; k < 4; ++k) tile[o + k][r] = v[k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * n; i += NT) {
        const int o = i / n, r = i - o * n;
        if (co0 + o < cout) gw[((long long)(co0 + o) * cin + ci0) * T + r] = tile[o][r];
    }
}

// input channels of a workgroup of wgrad8_reduce_rows
constexpr int reduced(int T) { return T < 64 ? 64 / T : 1; }

struct Geo {
    int kind;  // 0: 3×3, 1: 4×4 stride 2, 2: 4×4 stride 1, 3: 8×8, 4: tap by tap
    WgP p;
};
bool geometry(int64_t B, int32_t Hs, int32_t Ws, int32_t cin, int32_t MH, int32_t MW, int32_t cout, int32_t k,
              int32_t s, int32_t pad, Geo &g) {
    if (B <= 0 || Hs <= 0 || Ws <= 0 || cin <= 0 || MH <= 0 || MW <= 0 || cout <= 0 || k <= 0 || s <= 0 || pad < 0)
        return false;
    if (k > 8 || Hs > 65535 || Ws > 65535 || pad > 8192 || s > 8192 || cin > 65536 || cout > 65536) return false;
    if (Hs + 2 * pad < k || Ws + 2 * pad < k) return false;
    if (MH != (Hs + 2 * pad - k) / s + 1 || MW != (Ws + 2 * pad - k) / s + 1) return false;
    // (offsets within an image are 32-bit)
    if ((int64_t)MH * MW > 0x7fffffffLL / cout / 4 || (int64_t)Hs * Ws > 0x7fffffffLL / act8::pitch(cin)) return false;
    if (B > 0x7fffffff) return false;
    g.kind = k == 3 && s == 1 ? 0 : k == 4 && s == 2 ? 1 : k == 4 && s == 1 ? 2 : k == 8 && s == 1 ? 3 : 4;
    WgP &p = g.p;
    p = WgP{};
    p.B = (int)B; p.Hs = Hs; p.Ws = Ws; p.cin = cin; p.cp = act8::pitch(cin); p.nb = (cin + 31) / 32;
    p.MH = MH; p.MW = MW; p.cout = cout; p.k = k; p.s = s; p.p = pad;
    auto read = [&](int size, int out) {
        const int n = (out - 1) * s + k - pad;
        return n < 0 ? 0 : n < size ? n : size;
    };
    p.Hr = read(Hs, MH);
    p.Wr = read(Ws, MW);
    p.nci = (cin + 63) / 64;
    p.nco = (cout + 63) / 64;
    p.groups = g.kind <= 1 ? 1 : g.kind == 2 ? 2 : g.kind == 3 ? 8 : k * k;
    p.tY = (MH + 3) / 4;
    p.tX = (MW + 15) / 16;
    const long long tiles = B * p.tY * p.tX, work = (long long)p.nci * p.nco * p.groups;
    if (tiles > 0x7fffffffLL || work > (1 << 24)) return false;
    p.tiles = (int)tiles;
    // Splits: a K step takes about 1 + 0.19·taps us with a workgroup on each CU and 1.45 of that with two (3×3, measured:
    // 2.7 and 3.9 us), and a split's partial sums are written and read again at some 5 TB/s.  The cheapest of the numbers
    // that fill the CUs once or twice, or a half, a quarter ... of them.
    const long long places = g.kind == 1 ? 256 : 512;
    const double step = 1.0 + 0.19 * k * k / p.groups, mb = 4e-6 * k * k * 4096.0 * p.nci * p.nco;
    double best = 0;
    for (long long n = work >= places ? 1 : places / work; n; n /= 2) {
        const long long per = (tiles + n - 1) / n, used = (tiles + per - 1) / per;
        const double cost = per * step * (work * used > 256 ? 1.45 : 1.0) + 0.4 * mb * used;
        if (best == 0 || cost < best) {
            best = cost;
            p.per_split = (int)per;
        }
    }
    p.splits = (p.tiles + p.per_split - 1) / p.per_split;
    // (below 2^32 threads of a grid, the reduction's by rows among them)
    const int cb = reduced(k * k);
    return p.splits * work * (g.kind == 1 ? 2 * NT : NT) < 1LL << 32 &&
           (long long)((cout + 31) / 32) * ((cin + cb - 1) / cb) * NT < 1LL << 32;
}

template <bool G4>
void run(const Geo &g, hipStream_t st) {
    const WgP &p = g.p;
    const dim3 grid((unsigned)(p.splits * p.nci * p.nco * p.groups)), block(NT);
    switch (g.kind) {
        case 0: hipLaunchKernelGGL((wgrad8_kernel<3, 3, 1, 1, G4>), grid, block, 0, st, p); break;
        case 1: hipLaunchKernelGGL((wgrad8_kernel<2, 4, 2, 2, G4>), grid, dim3(2 * NT), 0, st, p); break;
        case 2: hipLaunchKernelGGL((wgrad8_kernel<2, 4, 1, 1, G4>), grid, block, 0, st, p); break;
        case 3: hipLaunchKernelGGL((wgrad8_kernel<1, 8, 1, 1, G4>), grid, block, 0, st, p); break;
        default: hipLaunchKernelGGL((wgrad8_kernel<1, 1, 1, 1, G4>), grid, block, 0, st, p);
    }
}

}  // namespace

extern "C" int64_t esr_dconv_wgrad_act8_workspace_bytes(int64_t B, int32_t Hs, int32_t Ws, int32_t cin, int32_t MH,
                                                        int32_t MW, int32_t cout, int32_t k, int32_t s, int32_t pad) {
    Geo g;
    if (!geometry(B, Hs, Ws, cin, MH, MW, cout, k, s, pad, g)) return ESR_EINVAL;
    return 4LL * g.p.splits * k * k * g.p.nci * 64 * g.p.nco * 64;
}

extern "C" int esr_dconv_wgrad_act8(const int8_t *codes, const uint8_t *exps, int64_t B, int32_t Hs, int32_t Ws,
                                    int32_t cin, const float *dy, int32_t MH, int32_t MW, int32_t cout, int32_t k,
                                    int32_t s, int32_t pad, float *gw, void *ws, esr_stream_t stream) {
    Geo g;
    if (!codes || !exps || !dy || !gw || !ws || (uintptr_t)codes % 16 || (uintptr_t)ws % 16 ||
        !geometry(B, Hs, Ws, cin, MH, MW, cout, k, s, pad, g))
        return ESR_EINVAL;
    const hipStream_t st = (hipStream_t)stream;
    WgP &p = g.p;
    p.codes = codes; p.exps = exps; p.dy = dy; p.partial = (float *)ws;
    if (cout % 4 == 0 && (uintptr_t)dy % 16 == 0) run<true>(g, st);
    else run<false>(g, st);
    const int T = k * k, nco = (cout + 31) / 32, cb = reduced(T);
    const long long rows = (long long)nco * ((cin + cb - 1) / cb);
    if (rows >= 256)  // enough workgroups without cutting the splits (64->512 8x8 of 8 images: 75 -> 43 us in all)
        hipLaunchKernelGGL(wgrad8_reduce_rows, dim3((unsigned)rows), dim3(NT), 0, st, p.partial, p.splits, T, cin, cout,
                           p.nci * 64, p.nco * 64, cb, gw);
    else
        hipLaunchKernelGGL(wgrad8_reduce, dim3((unsigned)p.nco * cin * T), dim3(NT), 0, st, p.partial, p.splits, T, cin, cout,
                           p.nci * 64, p.nco * 64, gw);
    return hipGetLastError() == hipSuccess ? ESR_OK : ESR_ELAUNCH;
}
