// Gated linear recurrence along one axis, f32 / f64:
//
//   h_s = a_s h_{s-1} + b_s        b = x, or (1 - a) x in the coupled form;   h_{-1} = h0 or 0
//
// and its gradient.  A step is the affine map h -> a h + b; maps compose associatively,
// (A2, B2) o (A1, B1) = (A2 A1, A2 B1 + B2), so the axis is cut into chunks whose maps are formed in
// parallel, and only the carry between chunks is sequential.  The backward pass is the same recurrence
// run the other way, g_s = dy_s + a_{s+1} g_{s+1}, with an epilogue (dx = g, da = g h_{s-1}), so one
// kernel body serves both: `s` below is always the PROCESSING index; the host folds the direction into
// signed strides.
//
// Every element is read once and written once.  The lanes (sequences) are cut into groups, the axis into rounds; a
// cluster of CTAs owns a group and takes one round after the other, each CTA a consecutive part of it, each warp a part of
// that.  Within a round the parts' maps travel through (distributed) shared memory, the carry between rounds stays in
// registers: no CTA waits for memory that another one writes, and no workspace is needed.  The folds have one order,
// so results are deterministic.  Copies run ahead in a ring of shared-memory stages; a thread (or a warp) copies what it
// will read itself, so the ring needs no barrier.
//
// A product of gates that leaves the type's range inside one round (at most 8192 steps of neighbouring lanes, 65536 along a contiguous
// axis) makes the carry's share inf or NaN where step-by-step evaluation might not; gates in [-1, 1] cannot.  Where such a
// product underflows, a finite carry's share is zero and an infinite one's NaN.
#include <algorithm>
#include <vector>

#include "rtb_internal.h"
#include "rtb_ckpt8.cuh"
#include "rtb_cluster.cuh"

namespace rtb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxLaneDims = 6;


__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return fma(a, b, c); }
__device__ __forceinline__ float nan_of(float) { return __int_as_float(0x7fffffff); }
__device__ __forceinline__ double nan_of(double) { return __longlong_as_double(0x7fffffffffffffffll); }

// The dims other than the axis, merged as far as every operand allows, outermost first.  A lane is one
// sequence; its element s sits at base + s * step in each operand.
struct LaneDims {
    int nd;
    uint64_t n[kMaxLaneDims];
    int64_t so[kMaxLaneDims], sg[kMaxLaneDims], sb[kMaxLaneDims], sx[kMaxLaneDims], sd[kMaxLaneDims];
};

template <typename T> struct ScanArgs {
    LaneDims dims;
    uint64_t lanes, steps;
    int64_t to, tg, tb, tx, td;  // signed steps along the axis in processing order (elements)
    int64_t o0, d0;          // flat position of processing index 0 in the dense outputs, and in dg
    const T *g;              // gate, at processing index 0
    const T *b;              // forward: x; backward: the upstream
    const T *x;              // backward, coupled: x
    const T *h0;             // dense over the lanes, or null
    const T *h;              // backward: dense states (flat)
    const int8_t *codes;     // or their 8-bit checkpoint
    const T *mags;
    T *out;                  // forward: h; backward: dx (may be null)
    T *dg;                   // backward: gradient of the gate, dense (may be null)
    T *dh0;                  // backward (may be null)
    int seg_shift;           // log2 of the neighbouring lanes whose share of dg is summed before it is written
    unsigned cluster;        // CTAs that share a group of lanes
    struct Strides {
        int64_t g, b, x, o, d;
    } bytes, round_bytes;    // to, tg ... in bytes, and those of a whole round
};

struct LaneAt {
    int64_t o, g, b, x, d;
};

__device__ __forceinline__ LaneAt locate(const LaneDims &d, uint64_t lane, int seg_shift) {
    LaneAt at{0, 0, 0, 0, 0};
    // 32-bit division wherever the index allows: the 64-bit one costs about a hundred instructions
#pragma unroll
    for (int k = kMaxLaneDims - 1; k >= 0; --k) {
        if (k >= d.nd) continue;
        uint64_t q, r;
        if (k == 0) {
            q = 0, r = lane;
        } else if (((lane | d.n[k]) >> 32) == 0) {
            q = (uint32_t)lane / (uint32_t)d.n[k];
            r = (uint32_t)lane - (uint32_t)q * (uint32_t)d.n[k];
        } else {
            q = lane / d.n[k], r = lane - q * d.n[k];
        }
        at.o += (int64_t)r * d.so[k];
        at.g += (int64_t)r * d.sg[k];
        at.b += (int64_t)r * d.sb[k];
        at.x += (int64_t)r * d.sx[k];
        at.d += (int64_t)(k == d.nd - 1 ? r >> seg_shift : r) * d.sd[k];
        lane = q;
    }
    return at;
}

enum Mode { kForward = 0, kBackDense = 1, kBackCodes = 2 };

// V neighbouring codes, as bytes of one word
template <int V> __device__ __forceinline__ uint32_t codes_at(const int8_t *p) {
    if constexpr (V == 4) return *reinterpret_cast<const uint32_t *>(p);
    else if constexpr (V == 2) return *reinterpret_cast<const uint16_t *>(p);
    else return (uint8_t)*p;
}

// ---- lanes contiguous in memory ----------------------------------------------------------------------------
// A thread holds V lanes and R steps; LX threads side by side make a group of LX V lanes, the 32 / LX such rows of a warp, the warps
// of a CTA and the CTAs of a cluster take consecutive parts of a round.
// GVEC: the gate's lanes are contiguous too; otherwise the V lanes of a thread share one gate value (V = 1: any stride).
// HBM-bound where lanes are many: 8 x 8192 x 1024 f32 forward 142 us (12 bytes an element, 5.7 TB/s), backward 233 us (20 bytes, 5.8 TB/s).
// Otherwise bound by the exchange of a round, 2 to 4 us: 1 x 65536 x 1024 forward 150 us, backward 246 us; 16 x 256 x 512, two
// rounds, 8 us.
template <typename T, int V, int R, int MODE, bool COUPLED, bool GVEC> struct LanesRing {
    static constexpr bool kBack = MODE != kForward;
    static constexpr int kGateRows = kBack && COUPLED ? R + 1 : R;   // the coupled epilogue wants the gate of the step itself too
    static constexpr int kVecBytes = sizeof(T) * V;
    // whole vectors go through the ring; a shared gate, codes and magnitudes are narrow and wait in registers instead
    static constexpr int kGate = 0;
    static constexpr int kB = kGate + (GVEC ? kThreads * kGateRows * kVecBytes : 0);
    static constexpr int kH = kB + kThreads * R * kVecBytes;
    static constexpr int kX = kH + (MODE == kBackDense ? kThreads * R * kVecBytes : 0);
    static constexpr int kStageBytes = kX + (kBack && COUPLED ? kThreads * R * kVecBytes : 0);
};

template <typename T, int V, int LX, int R, int STAGES, int MODE, bool COUPLED, bool GVEC>
__global__ void __launch_bounds__(kThreads, 2) scan_lanes_kernel(const __grid_constant__ ScanArgs<T> p) {
    using Ring = LanesRing<T, V, R, MODE, COUPLED, GVEC>;
    using P = Pack<T, V>;
    constexpr int VA = GVEC ? V : 1;   // a shared gate makes one product of gates for the thread's V lanes
    using PA = Pack<T, VA>;
    constexpr int W = LX * V, WA = LX * VA, kRows = 32 / LX;
    constexpr bool kBack = Ring::kBack;
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ alignas(16) T warp_a[2][kWarps][WA], warp_h[2][kWarps][W];
    const int lane = threadIdx.x % LX, row = threadIdx.x % 32 / LX, warp = threadIdx.x >> 5;
    const unsigned nc = p.cluster, rank = nc > 1 ? cluster_rank() : 0;
    T *const cta_maps = (T *)(ring + STAGES * Ring::kStageBytes);   // [2][nc][map WA, state W], in clusters only
    __shared__ unsigned long long arrived[2];                       // by buffer: the maps of all CTAs are here
    const uint64_t group = blockIdx.x / nc;
    const uint64_t first_lane = group * W + (uint64_t)lane * V;
    const bool active = first_lane < p.lanes;
    const LaneAt at = locate(p.dims, active ? first_lane : 0, p.seg_shift);
    const int steps = (int)p.steps, round = (int)nc * kWarps * kRows * R;
    const int my0 = (int)((rank * kWarps + warp) * kRows + row) * R;
    const int rounds = (steps + round - 1) / round;
    const bool need_h = kBack && p.dg;
    grid_dep_wait();

    // Addresses advance by byte strides out of the constant bank.  Backward: row k of the gate's ring is the step in front of row
    // k's own; a kept state is the one behind it.
    auto ptr = [&](const T *base, int64_t lane_at, int64_t t, int off) { return (const char *)(base + lane_at) + (my0 + off) * t; };
    const char *in_g = ptr(p.g, at.g, p.bytes.g, kBack ? -1 : 0), *in_b = ptr(p.b, at.b, p.bytes.b, 0);
    const char *in_h = MODE == kBackDense ? ptr(p.h, p.o0 + at.o, p.bytes.o, 1) : nullptr, *in_x = kBack && COUPLED ? ptr(p.x, at.x, p.bytes.x, 0) : nullptr;
    int64_t in_c = MODE == kBackCodes ? p.o0 + at.o + (my0 + 1) * p.to : 0;   // flat position of a code
    char *to_o = (char *)(p.out + p.o0 + at.o) + my0 * p.bytes.o;
    char *to_d = kBack ? (char *)(p.dg + p.d0 + at.d) + my0 * p.bytes.d : nullptr;
    const char *at_g = in_g;
    // steps left from the thread's first of the round on: of the round that is copied, fetched, worked on
    int left_in = active ? steps - my0 : 0, left_f = left_in, left = left_in;

    auto slot = [&](int stage, int part, int k) { return ring + stage * Ring::kStageBytes + part + (k * kThreads + (int)threadIdx.x) * Ring::kVecBytes; };
    auto issue = [&](int stage, bool start) {
        if (left_in > 0) {
            if constexpr (GVEC) {
                const char *q = in_g;
#pragma unroll
                for (int k = 0; k < Ring::kGateRows; ++k, q += p.bytes.g)
                    if (k - (kBack ? 1 : 0) < left_in && !(kBack && k == 0 && start && my0 == 0)) copy_async<Ring::kVecBytes>(slot(stage, Ring::kGate, k), q);
            }
            const char *q = in_b;
#pragma unroll
            for (int r = 0; r < R; ++r, q += p.bytes.b)
                if (r < left_in) copy_async<Ring::kVecBytes>(slot(stage, Ring::kB, r), q);
            if constexpr (MODE == kBackDense) {
                if (need_h) {
                    q = in_h;
#pragma unroll
                    for (int r = 0; r < R; ++r, q += p.bytes.o)
                        if (r + 1 < left_in) copy_async<Ring::kVecBytes>(slot(stage, Ring::kH, r), q);
                }
            }
            if constexpr (kBack && COUPLED) {
                if (need_h) {
                    q = in_x;
#pragma unroll
                    for (int r = 0; r < R; ++r, q += p.bytes.x)
                        if (r < left_in) copy_async<Ring::kVecBytes>(slot(stage, Ring::kX, r), q);
                }
            }
        }
        copy_commit();
        in_b += p.round_bytes.b, left_in -= round;
        if constexpr (GVEC) in_g += p.round_bytes.g;
        if constexpr (MODE == kBackDense) in_h += p.round_bytes.o;
        if constexpr (kBack && COUPLED) in_x += p.round_bytes.x;
    };
    // the narrow operands of a round, loaded while the one before it is worked on
    T gate_now[GVEC ? 1 : Ring::kGateRows] = {}, gate_next[GVEC ? 1 : Ring::kGateRows];
    uint32_t code_now[MODE == kBackCodes ? R : 1] = {}, code_next[MODE == kBackCodes ? R : 1];
    T mag_now[MODE == kBackCodes ? R : 1] = {}, mag_next[MODE == kBackCodes ? R : 1];
    auto fetch = [&](bool start) {
        if constexpr (!GVEC) {
            const char *q = at_g;
#pragma unroll
            for (int k = 0; k < Ring::kGateRows; ++k, q += p.bytes.g) {
                gate_next[k] = (T)1;
                if (k - (kBack ? 1 : 0) < left_f && !(kBack && k == 0 && start && my0 == 0)) gate_next[k] = *(const T *)q;
            }
            at_g += p.round_bytes.g;
        }
        if constexpr (MODE == kBackCodes) {
            int64_t flat = in_c;
#pragma unroll
            for (int r = 0; r < R; ++r, flat += p.to) {
                code_next[r] = 0, mag_next[r] = (T)0;
                if (need_h && r + 1 < left_f) {
                    code_next[r] = codes_at<V>(p.codes + flat);
                    mag_next[r] = p.mags[flat >> kCkpt8Shift];   // V divides the block: one magnitude
                }
            }
            in_c += p.round_bytes.o / (int)sizeof(T);
        }
        left_f -= round;
    };
    auto gate_of = [&](int stage, int k) {
        if constexpr (GVEC) return ld<T, VA>((const T *)slot(stage, Ring::kGate, k));
        else return PA{{gate_now[k]}};
    };
    auto of = [](const PA &v, int j) { return v.e[GVEC ? j : 0]; };

    P carry;   // the state in front of the round
#pragma unroll
    for (int j = 0; j < V; ++j) carry.e[j] = !kBack && p.h0 && active ? p.h0[first_lane + j] : (T)0;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i, i == 0);
    fetch(true);
    if (nc > 1) {
        if (threadIdx.x == 0) mbar_init(&arrived[0]), mbar_init(&arrived[1]);
        cluster_barrier();   // every CTA runs, its barriers are set, before any is written to
    }
    bool lost = false;

    int stage = 0;
    for (int i = 0; i < rounds; ++i) {
        issue(stage == 0 ? STAGES - 1 : stage - 1, false);
        if constexpr (!GVEC) {
#pragma unroll
            for (int k = 0; k < Ring::kGateRows; ++k) gate_now[k] = gate_next[k];
        }
        if constexpr (MODE == kBackCodes) {
#pragma unroll
            for (int r = 0; r < R; ++r) code_now[r] = code_next[r], mag_now[r] = mag_next[r];
        }
        if constexpr (!GVEC || MODE == kBackCodes) fetch(false);
        copy_wait<STAGES - 1>();
        const bool at_start = kBack && i == 0 && my0 == 0;   // in front of the first step there is no gate
        PA a[R];
        P b[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (r < left) {
                a[r] = gate_of(stage, r);
                if (r == 0 && at_start) {
#pragma unroll
                    for (int j = 0; j < VA; ++j) a[r].e[j] = (T)0;
                }
                b[r] = ld<T, V>((const T *)slot(stage, Ring::kB, r));
                if constexpr (!kBack && COUPLED) {
#pragma unroll
                    for (int j = 0; j < V; ++j) b[r].e[j] = ((T)1 - of(a[r], j)) * b[r].e[j];
                }
            } else {
#pragma unroll
                for (int j = 0; j < VA; ++j) a[r].e[j] = (T)1;
#pragma unroll
                for (int j = 0; j < V; ++j) b[r].e[j] = (T)0;
            }
        }
        // the thread's map over its R steps
        PA A = a[0];
        P H = b[0];
#pragma unroll
        for (int r = 1; r < R; ++r) {
#pragma unroll
            for (int j = 0; j < VA; ++j) A.e[j] = a[r].e[j] * A.e[j];
#pragma unroll
            for (int j = 0; j < V; ++j) H.e[j] = fma_(of(a[r], j), H.e[j], b[r].e[j]);
        }
        // the rows in front of the thread's own in its warp
        PA ex_a;
        P ex_h;
        if constexpr (kRows > 1) {
#pragma unroll
            for (int d = 1; d < kRows; d <<= 1) {
                PA pa;
                P ph;
#pragma unroll
                for (int j = 0; j < VA; ++j) pa.e[j] = __shfl_up_sync(0xffffffffu, A.e[j], d * LX);
#pragma unroll
                for (int j = 0; j < V; ++j) ph.e[j] = __shfl_up_sync(0xffffffffu, H.e[j], d * LX);
                if (row >= d) {
#pragma unroll
                    for (int j = 0; j < V; ++j) H.e[j] = fma_(of(A, j), ph.e[j], H.e[j]);
#pragma unroll
                    for (int j = 0; j < VA; ++j) A.e[j] = A.e[j] * pa.e[j];
                }
            }
#pragma unroll
            for (int j = 0; j < VA; ++j) {
                ex_a.e[j] = __shfl_up_sync(0xffffffffu, A.e[j], LX);
                if (row == 0) ex_a.e[j] = (T)1;
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                ex_h.e[j] = __shfl_up_sync(0xffffffffu, H.e[j], LX);
                if (row == 0) ex_h.e[j] = (T)0;
            }
        }
        const int buf = i & 1;   // a warp is never a whole round ahead of another: two buffers suffice
        if (row == kRows - 1) {
            st<T, VA>(&warp_a[buf][warp][lane * VA], A);
            st<T, V>(&warp_h[buf][warp][lane * V], H);
        }
        __syncthreads();
        P c = carry;
        if (nc > 1) {
            if (warp == 0 && row == 0) {
                A = ld<T, VA>(&warp_a[buf][0][lane * VA]), H = ld<T, V>(&warp_h[buf][0][lane * V]);
#pragma unroll
                for (int w = 1; w < kWarps; ++w) {
                    const PA wa = ld<T, VA>(&warp_a[buf][w][lane * VA]);
                    const P wh = ld<T, V>(&warp_h[buf][w][lane * V]);
#pragma unroll
                    for (int j = 0; j < VA; ++j) A.e[j] = wa.e[j] * A.e[j];
#pragma unroll
                    for (int j = 0; j < V; ++j) H.e[j] = fma_(of(wa, j), H.e[j], wh.e[j]);
                }
                if (lane == 0) mbar_expect(&arrived[buf], nc * (WA + W) * sizeof(T));
                const unsigned to = smem_addr(cta_maps + (buf * nc + rank) * (WA + W)), bar = smem_addr(&arrived[buf]);
                for (unsigned q = 0; q < nc; ++q) {
                    send(in_cta(to + lane * VA * sizeof(T), q), A, in_cta(bar, q));
                    send(in_cta(to + (WA + lane * V) * sizeof(T), q), H, in_cta(bar, q));
                }
            }
            // a CTA sends the maps of round i + 2 only after it has those of round i + 1 from all, who then have read round i's
            if (!lost && !mbar_wait(&arrived[buf], (unsigned)(i >> 1) & 1u)) lost = true;
            if (lost) {
#pragma unroll
                for (int j = 0; j < V; ++j) carry.e[j] = nan_of(T());
            }
            for (unsigned q = 0; q < nc; ++q) {
                if (q == rank) c = carry;
                const T *from = cta_maps + (buf * nc + q) * (WA + W);
                const PA qa = ld<T, VA>(from + lane * VA);
                const P qh = ld<T, V>(from + WA + lane * V);
#pragma unroll
                for (int j = 0; j < V; ++j) carry.e[j] = fma_(of(qa, j), carry.e[j], qh.e[j]);
            }
        }
        P mine = c;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) mine = c;
            if (nc > 1 && w >= warp) break;   // a single CTA folds all of them: that is the next round's carry
            const PA wa = ld<T, VA>(&warp_a[buf][w][lane * VA]);
            const P wh = ld<T, V>(&warp_h[buf][w][lane * V]);
#pragma unroll
            for (int j = 0; j < V; ++j) c.e[j] = fma_(of(wa, j), c.e[j], wh.e[j]);
        }
        if (nc == 1) carry = c;
        else mine = c;
        c = mine;
        if constexpr (kRows > 1) {
#pragma unroll
            for (int j = 0; j < V; ++j) c.e[j] = fma_(of(ex_a, j), c.e[j], ex_h.e[j]);
        }
        // the states (or the gradients that reach them) take b's place
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int j = 0; j < V; ++j) b[r].e[j] = c.e[j] = fma_(of(a[r], j), c.e[j], b[r].e[j]);
            if (r >= left) continue;
            T *const o = (T *)(to_o + r * p.bytes.o);
            if constexpr (!kBack) {
                st<T, V>(o, c);
            } else {
                if (p.out) {
                    P d = c;
                    if constexpr (COUPLED) {
                        const PA now = gate_of(stage, r + 1);
#pragma unroll
                        for (int j = 0; j < V; ++j) d.e[j] = ((T)1 - of(now, j)) * c.e[j];
                    }
                    st<T, V>(o, d);
                }
                if (r + 1 == left && p.dh0) {
#pragma unroll
                    for (int j = 0; j < V; ++j) p.dh0[first_lane + j] = p.g[at.g + j * (GVEC ? 1 : 0) + (int64_t)(steps - 1) * p.tg] * c.e[j];
                }
            }
        }
        if constexpr (kBack) {
            if (need_h) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    P d;
                    if constexpr (MODE == kBackDense) d = ld<T, V>((const T *)slot(stage, Ring::kH, r));
                    else Ckpt8Scale<T>(mag_now[r]).template restore<V>(code_now[r], d.e);
                    if (r + 1 == left) {   // the last step: the state in front of the first one
#pragma unroll
                        for (int j = 0; j < V; ++j) d.e[j] = p.h0 ? p.h0[first_lane + j] : (T)0;
                    }
                    if constexpr (COUPLED) {
                        const P x = ld<T, V>((const T *)slot(stage, Ring::kX, r));
#pragma unroll
                        for (int j = 0; j < V; ++j) d.e[j] = d.e[j] - x.e[j];
                    }
                    // behind the axis, and in idle threads, the ring holds nothing: what is there must not count
#pragma unroll
                    for (int j = 0; j < V; ++j) b[r].e[j] = r < left ? b[r].e[j] * d.e[j] : (T)0;
                }
                if (p.seg_shift == 0) {
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        if (r < left) st<T, V>((T *)(to_d + r * p.bytes.d), b[r]);
                } else {
                    // a segment is a power of two of lanes, at least V, and whole within a row of the group
                    T sum[R];
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        sum[r] = b[r].e[0];
#pragma unroll
                        for (int j = 1; j < V; ++j) sum[r] += b[r].e[j];
                    }
#pragma unroll
                    for (int m = 1; m < LX; m <<= 1)
                        if (m < (1 << p.seg_shift) / V) {
#pragma unroll
                            for (int r = 0; r < R; ++r) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], m);
                        }
                    if (((lane * V) & ((1 << p.seg_shift) - 1)) == 0) {
#pragma unroll
                        for (int r = 0; r < R; ++r)
                            if (r < left) *(T *)(to_d + r * p.bytes.d) = sum[r];
                    }
                }
            }
            to_d += p.round_bytes.d;
        }
        to_o += p.round_bytes.o, left -= round;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    grid_dep_launch();               // late: CTAs of the next kernel that wait beside a long loop slow it down
    if (nc > 1) cluster_barrier();   // no CTA leaves while another may still write to it
}

// ---- lanes contiguous, and so many of them that a thread for each V fills the device; or only a few steps ------------
// A thread walks its V lanes from end to end, kAhead steps loaded before they are needed: nothing is exchanged.  The gate of a step
// serves the next one of the backward pass too, so it is read once.  HBM-bound, and more steps ahead open more DRAM pages at
// once than they hide latency: 1000 x 64 x 1024 f32 forward 134 us with 2 (5.9 TB/s), 164 with 3, 193 with 4; backward 206 us with 1
// (6.4 TB/s), 231 with 2, 261 with 4.
template <typename T, int V, int MODE, bool COUPLED, bool GVEC>
__global__ void __launch_bounds__(kThreads) scan_walk_kernel(const __grid_constant__ ScanArgs<T> p) {
    constexpr bool kBack = MODE != kForward;
    constexpr int kAhead = kBack ? 1 : V > 1 ? 2 : 3, VA = GVEC ? V : 1;
    using P = Pack<T, V>;
    using PA = Pack<T, VA>;
    grid_dep_sync();
    const uint64_t first_lane = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) * V;
    const bool active = first_lane < p.lanes;
    const LaneAt at = locate(p.dims, active ? first_lane : 0, p.seg_shift);
    const int steps = (int)p.steps;
    const bool need_h = kBack && p.dg;
    const bool writes_sum = ((threadIdx.x * V) & ((1 << p.seg_shift) - 1)) == 0;
    const T *in_g = p.g + at.g, *in_b = p.b + at.b, *in_h = kBack && MODE == kBackDense ? p.h + p.o0 + at.o + p.to : nullptr;
    const T *in_x = kBack && COUPLED ? p.x + at.x : nullptr;
    int64_t in_c = p.o0 + at.o + p.to;
    T *to_o = p.out + p.o0 + at.o, *to_d = p.dg + p.d0 + at.d;
    PA gate[kAhead], before;
    P b[kAhead], hp[kBack ? kAhead : 1], x[kBack && COUPLED ? kAhead : 1];
    auto load = [&](int k, int s) {   // step s, into place k
        if (!active || s >= steps) return;
        if constexpr (GVEC) gate[k] = ld<T, VA>(in_g);
        else gate[k].e[0] = *in_g;
        b[k] = ld<T, V>(in_b);
        in_g += p.tg, in_b += p.tb;
        if constexpr (kBack) {
            if (need_h) {
                if (s + 1 < steps) {
                    if constexpr (MODE == kBackDense) hp[k] = ld<T, V>(in_h);
                    else Ckpt8Scale<T>(p.mags[in_c >> kCkpt8Shift]).template restore<V>(codes_at<V>(p.codes + in_c), hp[k].e);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j) hp[k].e[j] = p.h0 ? p.h0[first_lane + j] : (T)0;
                }
                if constexpr (MODE == kBackDense) in_h += p.to;
                else in_c += p.to;
                if constexpr (COUPLED) x[k] = ld<T, V>(in_x), in_x += p.tx;
            }
        }
    };
    auto of = [](const PA &v, int j) { return v.e[GVEC ? j : 0]; };
    P c;
#pragma unroll
    for (int j = 0; j < V; ++j) c.e[j] = !kBack && p.h0 && active ? p.h0[first_lane + j] : (T)0;
#pragma unroll
    for (int j = 0; j < VA; ++j) before.e[j] = (T)0;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) load(k, k);
    for (int s0 = 0; s0 < steps; s0 += kAhead) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int s = s0 + k;
            if (s >= steps) break;   // the same in all threads
            const PA a = gate[k];
            const P in = b[k];
            P d;
            if constexpr (kBack) {
                if (need_h) {
                    d = hp[k];
                    if constexpr (COUPLED) {
#pragma unroll
                        for (int j = 0; j < V; ++j) d.e[j] = d.e[j] - x[k].e[j];
                    }
                }
            }
            load(k, s + kAhead);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (kBack) c.e[j] = fma_(of(before, j), c.e[j], in.e[j]);
                else c.e[j] = fma_(of(a, j), c.e[j], COUPLED ? ((T)1 - of(a, j)) * in.e[j] : in.e[j]);
            }
            if constexpr (!kBack) {
                if (active) st<T, V>(to_o, c);
            } else {
                before = a;
                if (active && p.out) {
                    P o = c;
                    if constexpr (COUPLED) {
#pragma unroll
                        for (int j = 0; j < V; ++j) o.e[j] = ((T)1 - of(a, j)) * c.e[j];
                    }
                    st<T, V>(to_o, o);
                }
                if (need_h) {
#pragma unroll
                    for (int j = 0; j < V; ++j) d.e[j] = active ? c.e[j] * d.e[j] : (T)0;
                    if (p.seg_shift == 0) {
                        if (active) st<T, V>(to_d, d);
                    } else {
                        T sum = d.e[0];
#pragma unroll
                        for (int j = 1; j < V; ++j) sum += d.e[j];
                        for (int m = 1; m < (1 << p.seg_shift) / V; m <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
                        if (active && writes_sum) *to_d = sum;
                    }
                    to_d += p.td;
                }
                if (active && p.dh0 && s + 1 == steps) {
#pragma unroll
                    for (int j = 0; j < V; ++j) p.dh0[first_lane + j] = of(a, j) * c.e[j];
                }
            }
            to_o += p.to;
        }
    }
}

// ---- the axis itself contiguous ---------------------------------------------------------------------------
// A warp takes K runs of 32 V consecutive steps of one lane; within a run a thread holds V steps, and the threads' maps
// are scanned across the warp by shuffles.  TEAM warps share a lane: one walks it alone (many lanes, no barrier at all), or a
// CTA's eight, and the CTAs of a cluster, take consecutive parts of each round.
// VEC: all operands have unit stride (either sign) along the axis and 16-byte aligned runs.
// HBM-bound: 2048 lanes of 8192 steps f32 forward 33 us (6.1 TB/s).
template <typename T> __device__ __forceinline__ T shfl_up(T v, int d) { return __shfl_up_sync(0xffffffffu, v, d); }
template <typename T> __device__ __forceinline__ T shfl_down1(T v) { return __shfl_down_sync(0xffffffffu, v, 1); }
template <typename T> __device__ __forceinline__ T shfl_at(T v, int l) { return __shfl_sync(0xffffffffu, v, l); }

template <typename T, int V, int K, int MODE, bool COUPLED> struct AxisRing {
    static constexpr int kRun = 32 * V;                      // steps
    static constexpr int kTile = K * kRun;                   // steps of a warp in a round
    static constexpr int kPart = kTile * (int)sizeof(T);     // bytes
    static constexpr int kGate = 0, kB = kPart, kH = 2 * kPart, kX = kH + (MODE == kBackDense ? kPart : 0);
    static constexpr int kHalo = kX + (MODE != kForward && COUPLED ? kPart : 0);   // the gate before, the state behind
    static constexpr int kWarpBytes = kHalo + (MODE != kForward ? 16 : 0);
    static constexpr int kStageBytes = kWarps * kWarpBytes;
};

template <typename T, int V, int K, int STAGES, int TEAM, int MODE, bool COUPLED, bool VEC>
__global__ void __launch_bounds__(kThreads, 2) scan_axis_kernel(const __grid_constant__ ScanArgs<T> p) {
    using Ring = AxisRing<T, V, K, MODE, COUPLED>;
    using P = Pack<T, V>;
    constexpr bool kBack = MODE != kForward;
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ T warp_a[2][kWarps], warp_h[2][kWarps];
    __shared__ alignas(16) Pack<T, 2> cta_maps[2][kWideCluster];
    __shared__ unsigned long long arrived[2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned nc = TEAM > 1 ? p.cluster : 1, rank = nc > 1 ? cluster_rank() : 0;
    const uint64_t seq = TEAM > 1 ? blockIdx.x / nc : (uint64_t)blockIdx.x * kWarps + warp;
    if (TEAM == 1 && seq >= p.lanes) return;
    const LaneAt at = locate(p.dims, seq, 0);
    const int64_t steps = (int64_t)p.steps;
    const int64_t round = (int64_t)nc * TEAM * Ring::kTile, my0 = TEAM > 1 ? (int64_t)(rank * kWarps + warp) * Ring::kTile : 0;
    const int64_t rounds = (steps + round - 1) / round;
    const bool need_h = kBack && p.dg;
    grid_dep_wait();

    auto part = [&](int64_t i, int at_byte) { return (T *)(ring + (i % STAGES) * Ring::kStageBytes + warp * Ring::kWarpBytes + at_byte); };
    // steps [s0, s0 + kTile) of an operand with signed step t into a part of the ring: whole 16-byte vectors as they lie in
    // memory, or element by element in processing order
    auto fill = [&](T *to, const T *from, int64_t s0, int64_t t) {
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int64_t s = s0 + (k * 32 + lane) * V;
                if (s < steps) copy_async<16>(to + (k * 32 + lane) * V, t > 0 ? from + s : from - s - (V - 1));
            }
        } else {
#pragma unroll
            for (int e = 0; e < K * V; ++e) {
                const int64_t s = s0 + e * 32 + lane;
                if (s < steps) copy_async<sizeof(T)>(to + e * 32 + lane, from + s * t);
            }
        }
    };
    // V steps of run k, in processing order
    auto take = [&](const T *from, int k, int64_t t, int64_t s, T pad) {
        P v = ld<T, V>(from + (k * 32 + lane) * V);
        if (VEC && t < 0) {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                const T w = v.e[j];
                v.e[j] = v.e[V - 1 - j], v.e[V - 1 - j] = w;
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (s + j >= steps) v.e[j] = pad;
        return v;
    };
    auto put = [&](T *to, int64_t s, int64_t t, const P &v) {
        if constexpr (VEC) {
            if (s >= steps) return;
            P w = v;
            if (t < 0) {
#pragma unroll
                for (int j = 0; j < V; ++j) w.e[j] = v.e[V - 1 - j];
            }
            st<T, V>(t > 0 ? to + s : to - s - (V - 1), w);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (s + j < steps) to[(s + j) * t] = v.e[j];
        }
    };
    auto code_of = [&](int64_t s) {
        const int64_t flat = p.o0 + at.o + s * p.to;
        return Ckpt8Scale<T>(p.mags[flat >> kCkpt8Shift]).restore(p.codes[flat]);
    };
    // V kept states from step s on, out of their codes
    auto codes_run = [&](int64_t s) {
        P v;
#pragma unroll
        for (int j = 0; j < V; ++j) v.e[j] = (T)0;
        if constexpr (VEC) {
            if (s < steps) {
                const int64_t flat = p.o0 + at.o + (p.to > 0 ? s : -s - (V - 1));   // V aligned codes: one magnitude
                const uint32_t c = codes_at<V>(p.codes + flat);
                P w;
                Ckpt8Scale<T>(p.mags[flat >> kCkpt8Shift]).template restore<V>(c, w.e);
#pragma unroll
                for (int j = 0; j < V; ++j) v.e[j] = w.e[p.to > 0 ? j : V - 1 - j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (s + j < steps) v.e[j] = code_of(s + j);
        }
        return v;
    };
    auto issue = [&](int64_t i) {
        const int64_t s0 = i * round + my0;
        if (s0 < steps) {
            fill(part(i, Ring::kGate), p.g + at.g, s0, p.tg);
            fill(part(i, Ring::kB), p.b + at.b, s0, p.tb);
            if constexpr (kBack) {
                if (lane == 0 && s0 > 0) copy_async<sizeof(T)>(part(i, Ring::kHalo), p.g + at.g + (s0 - 1) * p.tg);
                if (need_h) {
                    if constexpr (MODE == kBackDense) {
                        fill(part(i, Ring::kH), p.h + p.o0 + at.o, s0, p.to);
                        if (lane == 0 && s0 + Ring::kTile < steps)
                            copy_async<sizeof(T)>(part(i, Ring::kHalo) + 1, p.h + p.o0 + at.o + (s0 + Ring::kTile) * p.to);
                    }
                    if constexpr (COUPLED) fill(part(i, Ring::kX), p.x + at.x, s0, p.tx);
                }
            }
        }
        copy_commit();
    };

    T carry = !kBack && p.h0 ? p.h0[seq] : (T)0;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i);
    if (nc > 1) {
        if (threadIdx.x == 0) mbar_init(&arrived[0]), mbar_init(&arrived[1]);
        cluster_barrier();   // every CTA runs, its barriers are set, before any is written to
    }
    bool lost = false;

    for (int64_t i = 0; i < rounds; ++i) {
        __syncwarp();                // the stage that is filled next has been read by all lanes
        issue(i + STAGES - 1);
        copy_wait<STAGES - 1>();
        __syncwarp();                // a lane reads what others copied
        const int64_t s0 = i * round + my0;
        P a[K], b[K], g[kBack ? K : 1], hp[kBack ? K : 1];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t s = s0 + (k * 32 + lane) * V;
            a[k] = take(part(i, Ring::kGate), k, p.tg, s, (T)1);
            b[k] = take(part(i, Ring::kB), k, p.tb, s, (T)0);
            if constexpr (!kBack && COUPLED) {
#pragma unroll
                for (int j = 0; j < V; ++j) b[k].e[j] = ((T)1 - a[k].e[j]) * b[k].e[j];
            }
        }
        if constexpr (kBack) {
            // the gates move one step back, the states one ahead
            T edge = s0 > 0 ? *part(i, Ring::kHalo) : (T)0;
            T behind = (T)0;
            if (need_h && s0 + Ring::kTile < steps) {
                if constexpr (MODE == kBackDense) behind = part(i, Ring::kHalo)[1];
                else behind = code_of(s0 + Ring::kTile);
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int64_t s = s0 + (k * 32 + lane) * V;
                g[k] = a[k];
                T before = shfl_up(g[k].e[V - 1], 1);
                if (lane == 0) before = edge;
                edge = shfl_at(g[k].e[V - 1], 31);
#pragma unroll
                for (int j = V - 1; j > 0; --j) a[k].e[j] = s + j < steps ? g[k].e[j - 1] : (T)1;
                a[k].e[0] = s < steps ? before : (T)1;
                if (need_h) {
                    if constexpr (MODE == kBackDense) hp[k] = take(part(i, Ring::kH), k, p.to, s, (T)0);
                    else hp[k] = codes_run(s);
                }
            }
            if (need_h) {
#pragma unroll
                for (int k = K - 1; k >= 0; --k) {
                    T after = shfl_down1(hp[k].e[0]);
                    if (lane == 31) after = behind;
                    behind = shfl_at(hp[k].e[0], 0);
#pragma unroll
                    for (int j = 0; j + 1 < V; ++j) hp[k].e[j] = hp[k].e[j + 1];
                    hp[k].e[V - 1] = after;
                }
                if (p.h0) {
#pragma unroll
                    for (int k = 0; k < K; ++k)
#pragma unroll
                        for (int j = 0; j < V; ++j)
                            if (s0 + (k * 32 + lane) * V + j + 1 == steps) hp[k].e[j] = p.h0[seq];
                }
            }
        }
        // maps: of the steps in front of the thread's own in its warp, and of the warp's whole part
        T ex_a[K], ex_h[K], A = (T)1, H = (T)0;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            T la = a[k].e[0], lh = b[k].e[0];
#pragma unroll
            for (int j = 1; j < V; ++j) {
                la = a[k].e[j] * la;
                lh = fma_(a[k].e[j], lh, b[k].e[j]);
            }
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const T pa = shfl_up(la, d), ph = shfl_up(lh, d);
                if (lane >= d) {
                    lh = fma_(la, ph, lh);
                    la = la * pa;
                }
            }
            T ea = shfl_up(la, 1), eh = shfl_up(lh, 1);
            if (lane == 0) ea = (T)1, eh = (T)0;
            ex_a[k] = ea * A;
            ex_h[k] = fma_(ea, H, eh);
            const T ta = shfl_at(la, 31), th = shfl_at(lh, 31);
            H = fma_(ta, H, th);
            A = ta * A;
        }
        T c = carry;
        if constexpr (TEAM > 1) {
            const int buf = (int)(i & 1);
            if (lane == 0) warp_a[buf][warp] = A, warp_h[buf][warp] = H;
            __syncthreads();
            if (nc > 1) {
                if (warp == 0 && lane < (int)nc) {
                    T ca = warp_a[buf][0], ch = warp_h[buf][0];
#pragma unroll
                    for (int w = 1; w < kWarps; ++w) {
                        ca = warp_a[buf][w] * ca;
                        ch = fma_(warp_a[buf][w], ch, warp_h[buf][w]);
                    }
                    if (lane == 0) mbar_expect(&arrived[buf], nc * 2 * sizeof(T));
                    send(in_cta(smem_addr(&cta_maps[buf][rank]), lane), Pack<T, 2>{{ca, ch}}, in_cta(smem_addr(&arrived[buf]), lane));
                }
                // a CTA sends the maps of round i + 2 only after it has those of round i + 1 from all, who then have read round i's
                if (!lost && !mbar_wait(&arrived[buf], (unsigned)(i >> 1) & 1u)) lost = true;
                if (lost) carry = nan_of(T());
                for (unsigned q = 0; q < nc; ++q) {
                    if (q == rank) c = carry;
                    carry = fma_(cta_maps[buf][q].e[0], carry, cta_maps[buf][q].e[1]);
                }
            }
            T mine = c;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                if (w == warp) mine = c;
                c = fma_(warp_a[buf][w], c, warp_h[buf][w]);
            }
            if (nc == 1) carry = c;
            c = mine;
        } else {
            carry = fma_(A, carry, H);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t s = s0 + (k * 32 + lane) * V;
            T v = fma_(ex_a[k], c, ex_h[k]);
            P h;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v = fma_(a[k].e[j], v, b[k].e[j]);
                h.e[j] = v;
            }
            if constexpr (!kBack) {
                put(p.out + p.o0 + at.o, s, p.to, h);
            } else {
                if (p.out) {
                    P d = h;
                    if constexpr (COUPLED) {
#pragma unroll
                        for (int j = 0; j < V; ++j) d.e[j] = ((T)1 - g[k].e[j]) * h.e[j];
                    }
                    put(p.out + p.o0 + at.o, s, p.to, d);
                }
                if (need_h) {
                    P d = hp[k];
                    if constexpr (COUPLED) {
                        const P x = take(part(i, Ring::kX), k, p.tx, s, (T)0);
#pragma unroll
                        for (int j = 0; j < V; ++j) d.e[j] = d.e[j] - x.e[j];
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) d.e[j] = h.e[j] * d.e[j];
                    put(p.dg + p.d0 + at.d, s, p.td, d);
                }
                if (p.dh0) {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (s + j + 1 == steps) p.dh0[seq] = g[k].e[j] * h.e[j];
                }
            }
        }
    }
    grid_dep_launch();               // late, as above
    if (nc > 1) cluster_barrier();   // no CTA leaves while another may still write to it
}

// ---- one step in place: state = a state + b over any view ------------------------------------------------
// 16 bytes an element in f32; a launch's latency at the sizes of a decoding step (64 x 2048: 3.7 us).
template <typename T, int V, bool COUPLED, bool GVEC>
__global__ void __launch_bounds__(kThreads) step_kernel(LaneDims dims, uint64_t lanes, T *state, const T *g, const T *x) {
    grid_dep_sync();
    const uint64_t i = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) * V;
    if (i >= lanes) return;
    const LaneAt at = locate(dims, i, 0);
    Pack<T, V> h = ld<T, V>(state + at.o), a, b = ld<T, V>(x + at.b);
    if constexpr (GVEC) {
        a = ld<T, V>(g + at.g);
    } else {
        const T one = g[at.g];
#pragma unroll
        for (int j = 0; j < V; ++j) a.e[j] = one;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) h.e[j] = fma_(a.e[j], h.e[j], COUPLED ? ((T)1 - a.e[j]) * b.e[j] : b.e[j]);
    st<T, V>(state + at.o, h);
}

// dst[i] = sum of the k neighbours src[i k ..): what is left of a gate's gradient after the segments
template <typename T> __global__ void __launch_bounds__(kThreads) neighbour_sum_kernel(const T *src, uint64_t n, unsigned k, T *dst) {
    grid_dep_sync();
    const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= n) return;
    T sum = src[i * k];
    for (unsigned j = 1; j < k; ++j) sum += src[i * k + j];
    dst[i] = sum;
}

// ---- host ------------------------------------------------------------------------------------------------
// Merges the dims of `shape` other than `axis` (axis >= rank: all of them) as far as the strides (null: unused) of out, gate,
// b, x and dg allow.  -> false when more than kMaxLaneDims remain.
bool lane_dims(size_t rank, const size_t *shape, size_t axis, const ptrdiff_t *const in[5], LaneDims *out) {
    int64_t *const to[5] = {out->so, out->sg, out->sb, out->sx, out->sd};
    int nd = 0;
    for (size_t k = 0; k < rank; ++k) {
        if (k == axis || shape[k] == 1) continue;
        bool merge = nd > 0;
        for (int q = 0; q < 5 && merge; ++q)
            if (in[q] && to[q][nd - 1] != (int64_t)in[q][k] * (int64_t)shape[k]) merge = false;
        if (!merge) {
            if (nd == kMaxLaneDims) return false;
            out->n[nd++] = 1;
        }
        out->n[nd - 1] *= shape[k];
        for (int q = 0; q < 5; ++q) to[q][nd - 1] = in[q] ? (int64_t)in[q][k] : 0;
    }
    if (!nd) {
        out->n[nd++] = 1;
        for (int q = 0; q < 5; ++q) to[q][0] = 0;
    }
    out->nd = nd;
    return true;
}

template <typename T> bool aligned16(const T *p) { return ((uintptr_t)p & 15u) == 0; }

// every stride except the innermost lane's is a multiple of V elements
template <int V> bool strides_whole(const LaneDims &d, const int64_t *s, int64_t step) {
    if (step % V) return false;
    for (int k = 0; k + 1 < d.nd; ++k)
        if (s[k] % V) return false;
    return true;
}

// A grid that starts beside its predecessor's last CTAs (programmatic dependent launch) saves up to 3 us, but takes whatever SMs are free and
// keeps them: more than a few rounds long, it loses more.  Backward, early / not: f32 (1, 65536, 256) with 4 heads, 11 rounds,
// 126 / 78 us; f64 (1, 32768, 128) with 2 heads, 6 rounds, 74 / 48 us; f32 (16, 256, 512), 2 rounds, 14.6 / 16.7 us.  Warps that
// walk a lane alone wait for nobody: early up to some 30 us, (4, 512, 8192) along the contiguous axis 35 / 38 us.
constexpr uint64_t kEarlyRounds = 4, kEarlyElements = 1u << 24;

// How many CTAs share a group: as many as run at once, as long as each has a part of its own.  `smem` says what a size needs.
// f32, up to 8 in powers of two / any number up to 16: forward (1, 65536, 64) 56 / 34 us, (1, 32768, 768) 79 / 69 us,
// (1, 16384, 512) 39 / 33 us, backward 81 / 47, 126 / 105 and 65 / 48 us; one lane of 1000000 55 / 31 and 102 / 55 us;
// (1, 65536, 1024), 8 either way.
template <typename T, void (*kernel)(ScanArgs<T>), typename F> int cluster_for(Ctx *ctx, uint64_t groups, uint64_t steps, uint64_t part, F smem, unsigned *out) {
    unsigned n = 1;
    while (n < kWideCluster && steps > (uint64_t)n * part) {
        unsigned fit = 0;
        if (int rc = clusters_at_once<ScanArgs<T>, kernel>(ctx, kThreads, n + 1, smem(n + 1), &fit)) return rc;
        if (groups > fit) break;
        ++n;
    }
    *out = n;
    return RTB_OK;
}

template <typename T, int V, int LX, int R, int STAGES, int MODE, bool COUPLED, bool GVEC> int run_width(Ctx *ctx, ScanArgs<T> &p) {
    constexpr uint64_t W = LX * V;
    const uint64_t groups = (p.lanes + W - 1) / W, part = (uint64_t)kWarps * (32 / LX) * R;
    constexpr auto kernel = scan_lanes_kernel<T, V, LX, R, STAGES, MODE, COUPLED, GVEC>;
    auto smem = [](unsigned cluster) {
        return (size_t)STAGES * LanesRing<T, V, R, MODE, COUPLED, GVEC>::kStageBytes + (cluster > 1 ? (size_t)cluster * 2 * (W + (GVEC ? W : LX)) * sizeof(T) : 0);
    };
    if (int rc = cluster_for<T, kernel>(ctx, groups, p.steps, part, smem, &p.cluster)) return rc;
    const int64_t es = sizeof(T), n = (int64_t)(p.cluster * part) * es;
    p.bytes = {p.tg * es, p.tb * es, p.tx * es, p.to * es, p.td * es};
    p.round_bytes = {p.tg * n, p.tb * n, p.tx * n, p.to * n, p.td * n};
    return launch_cluster<ScanArgs<T>, kernel>(ctx, "scan_lanes_kernel", groups * p.cluster, kThreads, p.cluster, smem(p.cluster),
                                               p.steps <= kEarlyRounds * p.cluster * part, p);
}

// Threads side by side in a group.  With vectors, 8 give rows of 128 bytes, a full line, and the most steps a round can have with
// them; 4 double the steps again where groups of 8 in the widest clusters would leave SMs without work or get too few CTAs each.
// 4 / 8, f32: (1, 65536, D) forward D = 64 35 / 57 us, 256 71 / 90, 512 97 / 108, 640 119 / 113; backward 512 153 / 171, 576 197 / 171;
// (8, 8192, 1024) forward 171 / 142.  Where neighbours' sums are formed, 4 add fewer of them in the kernel: backward 256, 4 heads 78 / 90,
// 384, 6 heads 95 / 94, 512, 32 heads 134 / 123.
// By elements (V = 1), 32 give the full line, and 8 serve few lanes: (8, 8192, 1023) 186 us with 32, 212 with 8; (1, 40000, D) forward
// D = 75 55 us with 32, 25 with 8; 301 74 and 54; backward 601 167 and 182.
template <typename T, int V> int side_by_side(const Ctx *ctx, const ScanArgs<T> &p, bool back) {
    constexpr int wide = V == 1 ? 32 : 8;
    const uint64_t groups = (p.lanes + wide * V - 1) / (wide * V), sms = (uint64_t)ctx->sm_count;
    if (V == 1) return groups * kMaxCluster < sms ? 8 : 32;
    const bool sums = back && p.dims.sg[p.dims.nd - 1] == 0;   // whether or not they are wanted: dx has the same bits
    return groups * (sums ? 12 : 9) <= sms ? 4 : 8;
}

// A thread for each V lanes where rounds would leave most rows of a CTA idle (few steps), or where there are threads enough to
// fill the device: f32, rounds / walk: (244, 61, 2048) with 16 heads, forward 150 / 54 us, backward 211 / 70 us; (100, 20, 1024)
// 24 / 9 us; (300, 200, 1024) forward 150 / 164 us, backward 392 / 227 us; (150, 200, 1024) forward 79 / 142 us.
template <typename T, int V> bool walks(const Ctx *ctx, const ScanArgs<T> &p, bool back) {
    const uint64_t threads = p.lanes / V / (uint64_t)ctx->sm_count;   // on each SM
    return p.steps <= 16 || (threads >= 64 && p.steps <= 64) || (threads >= 512 && (back || p.steps <= 128));
}

// Steps of a thread, with two stages of the ring.  More steps make fewer rounds, each of which costs the same exchange, and take
// more registers and shared memory (beyond 104 KB one CTA fits an SM, not two).  us at 65536 x 1024 and, behind the slash,
// 8 x 8192 x 1024, f32, per channel or with one gate for 64 or 128 channels:
//   forward, per channel     4: 173 / 141   6: 150 / 151   8: 156 / 147        shared   4: 210 / 148   6: 172 / 126   8: 146 / 114
//   backward, dense          4: 239 / 263   6: 246 / 236   8: 265 / 251        shared   4: 187 / 156   6: 170 / 155   8: 201 / 187
//   backward from codes      4: 246 / 207   6: 299 / 282                       shared   4: 191 / 160   6: 175 / 150   8: 192 / 175
//   backward, coupled        3: 308 / 262   4: 325 / 305   6: 307 / 283        shared   3: 244 / 203   4: 225 / 195   6: 247 / 230
// By elements, at 8 x 8192 x 1023: forward 8: 186, 12: 192, 16: 191 (shared 16: 171, 8: 218); backward 8: 344, 12: 359, 16: 482.
template <typename T, int V, int MODE, bool COUPLED, bool GVEC> int run_lanes(Ctx *ctx, ScanArgs<T> &p) {
    constexpr bool back = MODE != kForward;
    if (walks<T, V>(ctx, p, back)) {
        const uint64_t grid = (p.lanes + (uint64_t)kThreads * V - 1) / ((uint64_t)kThreads * V);
        if (grid > kMaxGrid) return fail(RTB_ERR_TOO_LARGE, "gated scan: %zu sequences are beyond one launch", (size_t)p.lanes);
        launch_dep(ctx, (unsigned)grid, kThreads, scan_walk_kernel<T, V, MODE, COUPLED, GVEC>, p);
        return check_launch(ctx, "scan_walk_kernel");
    }
    if constexpr (V == 1) {
        constexpr int R = sizeof(T) == 4 ? (back || GVEC ? 8 : 16) : (back ? 4 : GVEC ? 6 : 8);
        if (side_by_side<T, 1>(ctx, p, back) == 8) return run_width<T, 1, 8, R, 2, MODE, COUPLED, GVEC>(ctx, p);
        return run_width<T, 1, 32, R, 2, MODE, COUPLED, GVEC>(ctx, p);
    } else {
        constexpr int R = GVEC ? (back ? (COUPLED ? 3 : MODE == kBackDense ? 6 : 4) : 6) : (back ? (COUPLED ? 4 : 6) : 8);
        if (side_by_side<T, V>(ctx, p, back) == 4) return run_width<T, V, 4, R, 2, MODE, COUPLED, GVEC>(ctx, p);
        if constexpr (!back && GVEC)   // many lanes: no clusters, the exchange is cheap
            if (p.lanes >= (uint64_t)ctx->sm_count * 8 * V) return run_width<T, V, 8, 4, 2, MODE, COUPLED, GVEC>(ctx, p);
        return run_width<T, V, 8, R, 2, MODE, COUPLED, GVEC>(ctx, p);
    }
}

// The V lanes of a thread are neighbours in every operand (or share the gate), at 16-byte aligned places.
template <typename T, int MODE> bool lanes_vector(const ScanArgs<T> &p) {
    constexpr int V = 16 / sizeof(T);
    const LaneDims &d = p.dims;
    const int in = d.nd - 1;
    const bool gvec = d.sg[in] == 1;
    bool vec = d.n[in] % V == 0 && d.so[in] == 1 && d.sb[in] == 1 && strides_whole<V>(d, d.so, p.to) && strides_whole<V>(d, d.sb, p.tb) &&
               aligned16(p.b) && p.o0 % V == 0 && (gvec || d.sg[in] == 0);
    if (gvec) vec = vec && strides_whole<V>(d, d.sg, p.tg) && aligned16(p.g);
    if (p.x) vec = vec && d.sx[in] == 1 && strides_whole<V>(d, d.sx, p.tx) && aligned16(p.x);
    for (const T *q : {(const T *)p.out, (const T *)p.dg, p.h}) vec = vec && aligned16(q);
    if (MODE == kBackCodes) vec = vec && aligned16((const T *)p.codes);
    return vec;
}

template <typename T, int MODE, bool COUPLED> int pick_lanes(Ctx *ctx, ScanArgs<T> &p, bool vec) {
    constexpr int V = 16 / sizeof(T);
    if (vec && p.dims.sg[p.dims.nd - 1] == 1) return run_lanes<T, V, MODE, COUPLED, true>(ctx, p);
    if (vec) return run_lanes<T, V, MODE, COUPLED, false>(ctx, p);
    return p.dims.sg[p.dims.nd - 1] ? run_lanes<T, 1, MODE, COUPLED, true>(ctx, p) : run_lanes<T, 1, MODE, COUPLED, false>(ctx, p);
}

template <typename T, int MODE, bool COUPLED, bool VEC> int run_axis(Ctx *ctx, ScanArgs<T> &p) {
    constexpr int V = 16 / sizeof(T), K = MODE == kForward ? 4 : 2, S = 3;
    using Ring = AxisRing<T, V, K, MODE, COUPLED>;
    constexpr size_t smem = (size_t)S * Ring::kStageBytes;
    p.cluster = 1;
    // A warp for each lane wherever that gives every SM eight, or one part is all there is; else a CTA or a cluster.
    if (p.lanes >= (uint64_t)ctx->sm_count * kWarps || p.steps <= Ring::kTile)
        return launch_cluster<ScanArgs<T>, scan_axis_kernel<T, V, K, S, 1, MODE, COUPLED, VEC>>(ctx, "scan_axis_kernel", (p.lanes + kWarps - 1) / kWarps, kThreads, 1, smem, p.lanes * p.steps <= kEarlyElements, p);
    constexpr auto team = scan_axis_kernel<T, V, K, S, kWarps, MODE, COUPLED, VEC>;
    constexpr uint64_t part = (uint64_t)kWarps * Ring::kTile;
    if (int rc = cluster_for<T, team>(ctx, p.lanes, p.steps, part, [](unsigned) { return smem; }, &p.cluster)) return rc;
    return launch_cluster<ScanArgs<T>, team>(ctx, "scan_axis_kernel", p.lanes * p.cluster, kThreads, p.cluster, smem, p.steps <= kEarlyRounds * p.cluster * part, p);
}

template <typename T, int MODE, bool COUPLED> int pick_axis(Ctx *ctx, ScanArgs<T> &p) {
    constexpr int V = 16 / sizeof(T);
    auto unit = [](int64_t s) { return s == 1 || s == -1; };
    auto rows = [&](const int64_t *s) {
        for (int k = 0; k < p.dims.nd; ++k)
            if (s[k] % V) return false;
        return true;
    };
    // a reversed operand's pointer stands on its last element
    auto whole = [&](const T *q, int64_t s) { return aligned16(s > 0 ? q : q - (V - 1)); };
    bool vec = p.steps % V == 0 && unit(p.tg) && unit(p.tb) && unit(p.to) && rows(p.dims.sg) && rows(p.dims.sb) && rows(p.dims.so) &&
               whole(p.g, p.tg) && whole(p.b, p.tb);
    if (p.x) vec = vec && unit(p.tx) && rows(p.dims.sx) && whole(p.x, p.tx);
    for (const T *q : {(const T *)p.out, (const T *)p.dg, p.h, (const T *)p.codes}) vec = vec && aligned16(q);
    return vec ? run_axis<T, MODE, COUPLED, true>(ctx, p) : run_axis<T, MODE, COUPLED, false>(ctx, p);
}

template <typename T, int MODE> int pick(Ctx *ctx, ScanArgs<T> &p, bool along_axis, bool coupled, bool vec) {
    if (along_axis) return coupled ? pick_axis<T, MODE, true>(ctx, p) : pick_axis<T, MODE, false>(ctx, p);
    return coupled ? pick_lanes<T, MODE, true>(ctx, p, vec) : pick_lanes<T, MODE, false>(ctx, p, vec);
}

// A temporary block of the context allocator, given back when the scope ends (stream order keeps it alive).
struct Temp {
    rtb_ctx *c;
    void *p = nullptr;
    explicit Temp(rtb_ctx *ctx) : c(ctx) {}
    ~Temp() {
        if (p) rtb_free(c, p);
    }
};

struct View {
    const void *p;
    const ptrdiff_t *strides;
    size_t offset;
};

// An operand is read in place when its lanes (or, along the axis, its steps) are neighbours in memory; a broadcast
// one as well.  Any other view (a transposed one, a negative step) is first copied row-major: one more
// pass, where reading it in place would fetch a 32-byte sector per element.
int in_place_or_copy(rtb_ctx *c, int dtype, size_t rank, const size_t *shape, size_t inner_dim, bool must_copy, size_t total,
                     const ptrdiff_t *dense, View *v, Temp *tmp) {
    const ptrdiff_t s = inner_dim < rank ? v->strides[inner_dim] : 1;
    if (!must_copy && (s == 0 || s == 1)) return RTB_OK;
    int rc = rtb_alloc(c, total * dtype_size(dtype), &tmp->p);
    if (rc) return rc;
    rc = rtb_copy_view(c, dtype, v->p, rank, shape, v->strides, v->offset, tmp->p);
    if (rc) return rc;
    v->p = tmp->p, v->strides = dense, v->offset = 0;
    return RTB_OK;
}

int check_scan(rtb_ctx *c, int dtype, int flags, size_t rank, const size_t *shape, size_t axis) {
    if (!c) return fail(RTB_ERR_INVALID, "null ctx");
    if (dtype != RTB_F32 && dtype != RTB_F64) return fail(RTB_ERR_DTYPE, "the gated scan is defined for f32 and f64 only");
    if (flags & ~(RTB_SCAN_REVERSE | RTB_SCAN_COUPLED)) return fail(RTB_ERR_INVALID, "unknown scan flags %d", flags);
    if (rank > RTB_MAX_RANK) return fail(RTB_ERR_DIM, "rank %zu exceeds %d", rank, RTB_MAX_RANK);
    if (rank && !shape) return fail(RTB_ERR_INVALID, "null shape");
    if (axis >= rank) return fail(RTB_ERR_DIM, "axis %zu out of range for rank %zu", axis, rank);
    // steps are counted in 32 bits inside the kernels, a round (at most 2^16 steps) beyond the last one included
    if (shape[axis] > 0x7fff0000u) return fail(RTB_ERR_TOO_LARGE, "gated scan: %zu steps, 2^31 - 2^16 is the limit", shape[axis]);
    return RTB_OK;
}

struct ScanCall {
    bool back;
    View gate, b, x;
    const void *h0, *h, *codes, *mags;
    void *out, *dg, *dh0;
};

// The gate's gradient when the gate is broadcast.  Where the innermost lanes share their gate, neighbours in segments of a power
// of two are summed before anything is written; what is left to sum goes through a tensor of `shape` (the lanes in segments)
// and rtb_reduce_to_shape.
struct SharedGate {
    std::vector<size_t> shape;
    std::vector<ptrdiff_t> strides, gate_strides;
    int seg_shift = 0;
    bool rest = false;   // dims remain to be summed
};

SharedGate shared_gate(size_t rank, const size_t *shape, const ptrdiff_t *stride_g, size_t axis, uint64_t inner, unsigned widest) {
    SharedGate s;
    s.shape.assign(shape, shape + rank);
    s.gate_strides.assign(stride_g, stride_g + rank);
    // the trailing dims that were merged into the innermost lane dim
    size_t k0 = rank;
    uint64_t n = 1;
    while (n < inner && k0 > axis + 1) n *= shape[--k0];
    if (n == inner && widest > 1) {
        while ((2u << s.seg_shift) <= widest && inner % (2u << s.seg_shift) == 0) ++s.seg_shift;
        s.shape.resize(k0);
        s.gate_strides.resize(k0);
        s.shape.push_back((size_t)(inner >> s.seg_shift));
        s.gate_strides.push_back(0);
    }
    for (size_t k = 0; k < s.shape.size(); ++k) s.rest = s.rest || (s.gate_strides[k] == 0 && s.shape[k] != 1);
    s.strides.resize(s.shape.size());
    rtb_meta_contiguous_strides(s.shape.size(), s.shape.data(), s.strides.data());
    // as strides of the original dims: the merged ones walk lanes, locate() shifts them into segments
    if (s.shape.size() != rank || s.seg_shift) {
        s.strides.resize(k0);
        s.strides.resize(rank);
        ptrdiff_t step = 1;
        for (size_t k = rank; k-- > k0;) s.strides[k] = step, step *= (ptrdiff_t)shape[k];
    }
    return s;
}

template <typename T> int run_scan(rtb_ctx *c, Ctx *ctx, int dtype, int flags, ScanCall call, size_t rank, const size_t *shape, size_t axis,
                                   size_t total) {
    ptrdiff_t dense[RTB_MAX_RANK];
    rtb_meta_contiguous_strides(rank, shape, dense);
    const bool coupled = flags & RTB_SCAN_COUPLED, need_x = call.back && coupled && call.dg;
    bool shared = false;
    if (call.dg)
        for (size_t k = 0; k < rank; ++k) shared = shared || (call.gate.strides[k] == 0 && shape[k] != 1);
    const ptrdiff_t *const gate_strides = call.gate.strides;   // as given: a copy of the gate below is not broadcast any more
    // the innermost dim with more than one element decides: the axis itself, or a lane dim
    size_t inner = rank;
    for (size_t k = rank; k-- > 0;)
        if (shape[k] != 1) {
            inner = k;
            break;
        }
    const bool along_axis = inner >= rank || inner == axis;
    ScanArgs<T> p{};
    Temp tg(c), tb(c), tx(c), sums(c);
    int rc;
    for (int pass = 0;; ++pass) {
        const bool copy = pass == 1;   // too many lane dims: dense copies have two at most
        if ((rc = in_place_or_copy(c, dtype, rank, shape, inner, copy && !tg.p, total, dense, &call.gate, &tg))) return rc;
        if ((rc = in_place_or_copy(c, dtype, rank, shape, inner, copy && !tb.p, total, dense, &call.b, &tb))) return rc;
        if (need_x && (rc = in_place_or_copy(c, dtype, rank, shape, inner, copy && !tx.p, total, dense, &call.x, &tx))) return rc;
        const ptrdiff_t *const in[5] = {dense, call.gate.strides, call.b.strides, need_x ? call.x.strides : nullptr, dense};
        if (lane_dims(rank, shape, axis, in, &p.dims)) break;
    }
    const int64_t steps = (int64_t)shape[axis];
    const bool down = ((flags & RTB_SCAN_REVERSE) != 0) != call.back;   // processing order runs towards lower indices
    auto place = [&](const View &v, int64_t *step) {
        const int64_t s = (int64_t)v.strides[axis];
        *step = down ? -s : s;
        return (const T *)v.p + (int64_t)v.offset + (down ? (steps - 1) * s : 0);
    };
    p.steps = (uint64_t)steps;
    p.lanes = total / shape[axis];
    p.g = place(call.gate, &p.tg);
    p.b = place(call.b, &p.tb);
    if (need_x) p.x = place(call.x, &p.tx);
    p.to = p.td = down ? -(int64_t)dense[axis] : (int64_t)dense[axis];
    p.o0 = p.d0 = down ? (steps - 1) * (int64_t)dense[axis] : 0;
    p.h0 = (const T *)call.h0, p.h = (const T *)call.h;
    p.codes = (const int8_t *)call.codes, p.mags = (const T *)call.mags;
    p.out = (T *)call.out, p.dg = (T *)call.dg, p.dh0 = (T *)call.dh0;
    bool vec = !along_axis && (call.back ? (call.codes ? lanes_vector<T, kBackCodes>(p) : lanes_vector<T, kBackDense>(p)) : lanes_vector<T, kForward>(p));
    SharedGate share;
    if (shared) {
        const int in_dim = p.dims.nd - 1;
        const bool segments = vec && p.dims.sg[in_dim] == 0;
        share = shared_gate(rank, shape, gate_strides, axis, segments ? p.dims.n[in_dim] : 0, !segments ? 1 : 16 / sizeof(T) * (walks<T, 16 / sizeof(T)>(ctx, p, true) ? 32 : side_by_side<T, 16 / sizeof(T)>(ctx, p, true)));
        if (share.seg_shift) {
            p.seg_shift = share.seg_shift;
            const ptrdiff_t *const in[5] = {dense, call.gate.strides, call.b.strides, need_x ? call.x.strides : nullptr, share.strides.data()};
            if (!lane_dims(rank, shape, axis, in, &p.dims)) return fail(RTB_ERR_TOO_LARGE, "gated scan: more than %d dims", kMaxLaneDims);
            p.td = down ? -(int64_t)share.strides[axis] : (int64_t)share.strides[axis];
            p.d0 = down ? (steps - 1) * (int64_t)share.strides[axis] : 0;
        }
        if (share.rest) {
            size_t n = 1;
            for (size_t v : share.shape) n *= v;
            if ((rc = rtb_alloc(c, n * sizeof(T), &sums.p))) return rc;
            p.dg = (T *)sums.p;
        }
    }
    if (!call.back) rc = pick<T, kForward>(ctx, p, along_axis, coupled, vec);
    else if (call.codes) rc = pick<T, kBackCodes>(ctx, p, along_axis, coupled, vec);
    else rc = pick<T, kBackDense>(ctx, p, along_axis, coupled, vec);
    if (rc || !sums.p) return rc;
    // only a short innermost dim is left: one thread for each sum (a row each is what the axis reduction is built for)
    size_t left = 1, n_out = 1;
    bool inner_only = true;
    for (size_t k = 0; k < share.shape.size(); ++k) {
        if (share.gate_strides[k] == 0 && share.shape[k] != 1) {
            inner_only = inner_only && left == 1 && k + 1 == share.shape.size();
            left *= share.shape[k];
        } else {
            n_out *= share.shape[k];
        }
    }
    if (inner_only && left <= 64 && n_out / kThreads < kMaxGrid) {
        launch_dep(ctx, (unsigned)((n_out + kThreads - 1) / kThreads), kThreads, neighbour_sum_kernel<T>, (const T *)sums.p, (uint64_t)n_out,
                   (unsigned)left, (T *)call.dg);
        return check_launch(ctx, "neighbour_sum_kernel");
    }
    std::vector<size_t> out_shape(share.shape.size());
    return rtb_reduce_to_shape(c, dtype, sums.p, share.shape.size(), share.shape.data(), share.gate_strides.data(), call.dg, out_shape.data());
}

template <typename T, bool COUPLED> int run_step(Ctx *ctx, const LaneDims &d, uint64_t lanes, T *state, const T *g, const T *x) {
    constexpr int V = 16 / sizeof(T);
    const int in = d.nd - 1;
    const bool gvec = d.sg[in] == 1;
    bool vec = d.n[in] % V == 0 && d.so[in] == 1 && d.sb[in] == 1 && (gvec || d.sg[in] == 0) && strides_whole<V>(d, d.so, 0) &&
               strides_whole<V>(d, d.sb, 0) && aligned16(state) && aligned16(x);
    if (gvec) vec = vec && strides_whole<V>(d, d.sg, 0) && aligned16(g);
    const uint64_t per = (uint64_t)kThreads * (vec ? V : 1), grid = (lanes + per - 1) / per;
    if (grid > kMaxGrid) return fail(RTB_ERR_TOO_LARGE, "gated step: %zu elements are beyond one launch", (size_t)lanes);
    if (vec && gvec) launch_dep(ctx, (unsigned)grid, kThreads, step_kernel<T, V, COUPLED, true>, d, lanes, state, g, x);
    else if (vec) launch_dep(ctx, (unsigned)grid, kThreads, step_kernel<T, V, COUPLED, false>, d, lanes, state, g, x);
    else launch_dep(ctx, (unsigned)grid, kThreads, step_kernel<T, 1, COUPLED, false>, d, lanes, state, g, x);
    return check_launch(ctx, "step_kernel");
}

template <typename T> int step_any(Ctx *ctx, int flags, T *state, const ptrdiff_t *ss, const T *g, const ptrdiff_t *sg, const T *x,
                                   const ptrdiff_t *sx, size_t rank, const size_t *shape) {
    LaneDims d;
    uint64_t lanes = 1;
    for (size_t k = 0; k < rank; ++k) lanes *= shape[k];
    const ptrdiff_t *const in[5] = {ss, sg, sx, nullptr, nullptr};
    if (lane_dims(rank, shape, rank, in, &d))
        return flags & RTB_SCAN_COUPLED ? run_step<T, true>(ctx, d, lanes, state, g, x) : run_step<T, false>(ctx, d, lanes, state, g, x);
    // more dims than one launch takes: peel the outermost one that has extent
    size_t k0 = 0;
    while (shape[k0] == 1) ++k0;
    for (size_t i = 0; i < shape[k0]; ++i) {
        const ptrdiff_t k = (ptrdiff_t)i;
        int rc = step_any<T>(ctx, flags, state + k * ss[k0], ss + k0 + 1, g + k * sg[k0], sg + k0 + 1, x + k * sx[k0], sx + k0 + 1,
                             rank - k0 - 1, shape + k0 + 1);
        if (rc) return rc;
    }
    return RTB_OK;
}

}  // namespace
}  // namespace rtb

using namespace rtb;

static inline Ctx *C(rtb_ctx *c) { return reinterpret_cast<Ctx *>(c); }

static size_t count_of(size_t rank, const size_t *shape) {
    size_t n = 1;
    for (size_t k = 0; k < rank; ++k) n *= shape[k];
    return n;
}

RTB_API int rtb_gated_scan(rtb_ctx *c, int dtype, int flags, const void *gate, const ptrdiff_t *stride_g, size_t off_g, const void *x,
                           const ptrdiff_t *stride_x, size_t off_x, const void *h0, void *h, size_t rank, const size_t *shape, size_t axis) {
    return guarded([&]() -> int {
        int rc = check_scan(c, dtype, flags, rank, shape, axis);
        if (rc) return rc;
        const size_t total = count_of(rank, shape);
        if (total == 0) return RTB_OK;
        if (!gate || !x || !h || !stride_g || !stride_x) return fail(RTB_ERR_INVALID, "null argument");
        Ctx *ctx = C(c);
        if ((rc = use_device(ctx))) return rc;
        ScanCall call{};
        call.gate = View{gate, stride_g, off_g};
        call.b = View{x, stride_x, off_x};
        call.h0 = h0, call.out = h;
        return dtype == RTB_F32 ? run_scan<float>(c, ctx, dtype, flags, call, rank, shape, axis, total)
                                : run_scan<double>(c, ctx, dtype, flags, call, rank, shape, axis, total);
    });
}

RTB_API int rtb_gated_scan_backward(rtb_ctx *c, int dtype, int flags, const void *up, const ptrdiff_t *stride_u, size_t off_u,
                                    const void *gate, const ptrdiff_t *stride_g, size_t off_g, const void *x, const ptrdiff_t *stride_x,
                                    size_t off_x, const void *h, const int8_t *codes, const void *mags, const void *h0, void *d_x,
                                    void *d_gate, void *d_h0, size_t rank, const size_t *shape, size_t axis) {
    return guarded([&]() -> int {
        int rc = check_scan(c, dtype, flags, rank, shape, axis);
        if (rc) return rc;
        const size_t total = count_of(rank, shape), es = dtype_size(dtype);
        Ctx *ctx = C(c);
        if (!stride_g) return fail(RTB_ERR_INVALID, "null argument");
        if (total == 0) {
            // no step and no upstream: what is left of the gradients is zero
            if ((rc = use_device(ctx))) return rc;
            size_t lanes = 1, gate_n = 1;
            for (size_t k = 0; k < rank; ++k) {
                if (k != axis) lanes *= shape[k];
                if (stride_g[k] != 0) gate_n *= shape[k];   // the dims it is broadcast along are summed
            }
            if (d_h0 && lanes) RTB_CUDA(cudaMemsetAsync(d_h0, 0, lanes * es, ctx->stream));
            if (d_gate && gate_n) RTB_CUDA(cudaMemsetAsync(d_gate, 0, gate_n * es, ctx->stream));
            return RTB_OK;
        }
        if (!up || !gate || !stride_u) return fail(RTB_ERR_INVALID, "null argument");
        if (d_gate && !h && (!codes || !mags)) return fail(RTB_ERR_INVALID, "the gate's gradient needs the states or their checkpoint");
        if (h && codes) return fail(RTB_ERR_INVALID, "states and a checkpoint of them at once");
        if (d_gate && (flags & RTB_SCAN_COUPLED) && (!x || !stride_x)) return fail(RTB_ERR_INVALID, "the coupled gate's gradient needs x");
        if (!d_x && !d_gate && !d_h0) return RTB_OK;
        if ((rc = use_device(ctx))) return rc;
        ScanCall call{};
        call.back = true;
        call.gate = View{gate, stride_g, off_g};
        call.b = View{up, stride_u, off_u};
        call.x = View{x, stride_x, off_x};
        call.h0 = h0, call.h = h, call.codes = codes, call.mags = mags;
        call.out = d_x, call.dg = d_gate, call.dh0 = d_h0;
        return dtype == RTB_F32 ? run_scan<float>(c, ctx, dtype, flags, call, rank, shape, axis, total)
                                : run_scan<double>(c, ctx, dtype, flags, call, rank, shape, axis, total);
    });
}

RTB_API int rtb_gated_step(rtb_ctx *c, int dtype, int flags, void *state, const ptrdiff_t *stride_s, size_t off_s, const void *gate,
                           const ptrdiff_t *stride_g, size_t off_g, const void *x, const ptrdiff_t *stride_x, size_t off_x, size_t rank,
                           const size_t *shape) {
    return guarded([&]() -> int {
        if (!c) return fail(RTB_ERR_INVALID, "null ctx");
        if (dtype != RTB_F32 && dtype != RTB_F64) return fail(RTB_ERR_DTYPE, "the gated step is defined for f32 and f64 only");
        if (flags & ~RTB_SCAN_COUPLED) return fail(RTB_ERR_INVALID, "unknown step flags %d", flags);
        if (rank > RTB_MAX_RANK) return fail(RTB_ERR_DIM, "rank %zu exceeds %d", rank, RTB_MAX_RANK);
        if (rank && (!shape || !stride_s || !stride_g || !stride_x)) return fail(RTB_ERR_INVALID, "null shape or strides");
        if (count_of(rank, shape) == 0) return RTB_OK;
        if (!state || !gate || !x) return fail(RTB_ERR_INVALID, "null argument");
        for (size_t k = 0; k < rank; ++k)
            if (stride_s[k] == 0 && shape[k] != 1) return fail(RTB_ERR_SHAPE, "the state's dim %zu is broadcast: it cannot be written", k);
        Ctx *ctx = C(c);
        if (int rc = use_device(ctx)) return rc;
        if (dtype == RTB_F32)
            return step_any<float>(ctx, flags, (float *)state + off_s, stride_s, (const float *)gate + off_g, stride_g, (const float *)x + off_x,
                                   stride_x, rank, shape);
        return step_any<double>(ctx, flags, (double *)state + off_s, stride_s, (const double *)gate + off_g, stride_g, (const double *)x + off_x,
                                stride_x, rank, shape);
    });
}
