// Selective recurrence, backward (sm_100a).
//
// With dy = dout silu(z) and g_t the gradient of h_t,
//     g_t[n] = C_t[n] dy_t + a_{t+1}[n] g_{t+1}[n]             a = exp(s A)
//     dC_t[n] = sum_d dy_t h_t[n]        dB_t[n] = sum_d g_t[n] s_t x_t
//     dx_t = s_t sum_n g_t[n] B_t[n] + D dy_t
//     ds_t = sum_n g_t[n] a_t[n] h_{t-1}[n] A[n] + x_t sum_n g_t[n] B_t[n]
//     dA[n] = sum_t g_t[n] a_t[n] h_{t-1}[n] s_t
// and ddelta = ds sigmoid(delta + bias), dz = dout y silu'(z).
//
// A CTA owns the channels that a forward CTA owns, with half the threads: a thread holds four states
// of two neighbouring channels, so that the sums of dB and dC start in its registers.  It goes through
// the tiles from the last one back.  From the state that the forward kept before a tile it runs
// forward, keeping the state before every fourth position, then takes the groups of four positions
// from the last one back: states again, then gradients.  dB and dC are summed over a thread's two
// channels, over the warp's by exchanges between lanes, over the CTA's warps in shared memory and
// over CTAs by a second kernel, all in a fixed order: two calls give the same bits.
//
// What bounds it: an element takes two exponentials (238 us for the 537 M elements of 4 x 4096 x 2048
// x 16, which takes 1188; its memory 82) and 28 instructions, most of them the gradients' FMAs and the
// exchanges that sum dB, dC over channels and ds, dx over states.  Eight warps an SM are what the
// registers leave (above 16 states shared memory leaves six to two); a scheduler issues .35 a cycle.  Of the 1188 us the pass to the states takes 180,
// the gradients 570 (their sums over channels 180, over states 100), and what is done once per
// position and channel (step sizes, gates, loads, stores) 440.
//
// Sums straight to memory for each warp and half the groups took 1372 us, loads ahead of the tile
// 1266, B and C doubled in shared memory 2107, prefetches of the next tile into L2 1217.
#include "cc1d_selective.cuh"

namespace cc1d {
namespace {

constexpr int kSelThreads = 64, kWarps = kSelThreads / 32, kHalf = kSelThreads * 4;
// CTAs of an SM: all 255 registers of a thread are in use.  With 168, and six CTAs, 1550 us.
constexpr int kBwdCtas = 4;

// Shared memory: flags; (s, x) of a pair by position, replaced by (dx, ddelta), and (dy, slope of the
// step size), replaced by (y, -), and dout silu'(z); the states before every fourth position; each
// warp's sums of dB and dC; B and C; of each pass g carried, dA and its low part; with several passes
// three sums by position and pair.
template <int LN>
struct BwdSmem {
  static constexpr int T = sel_tile(LN), PAIRS = kSelThreads / LN, PITCH = PAIRS + 1;
  static constexpr int kFlags = 256, kIo = T * PITCH * 16, kDz = (T * PITCH * 8 + 15) / 16 * 16, kSub = T / 4 * kSelThreads * 32;
  static constexpr int kSlab = T * 8 * LN * 4;  // one warp's
  static constexpr int kThree = T * PITCH * 24;
  static int64_t bytes(const SelArgs& a) {
    return kFlags + 2 * kIo + kDz + kSub + kWarps * kSlab + T * 8 * LN * a.blocks * 4 + 3ll * a.blocks * kSelThreads * 32 +
           (a.blocks > 1 ? kThree : 0);
  }
};

// Adds v to the sum hi + lo, which together hold twice the bits (Knuth's two-sum).
__device__ __forceinline__ void add_to(float& hi, float& lo, float v) {
  const float s = hi + v;
  const float w = s - hi;
  lo += (hi - (s - w)) + (v - w);
  hi = s;
}
__device__ __forceinline__ void add_to(float2& hi, float2& lo, float2 v) {
  add_to(hi.x, lo.x, v.x);
  add_to(hi.y, lo.y, v.y);
}

// The sums of eight values over the channels of a warp.  A lane ends with kLeft<LN> of them, the
// first of which summed() tells; lanes that differ in further bits hold the same ones.
template <int LN>
constexpr int kLeft = LN >= 4 ? LN / 4 : 1;
template <int LN>
__device__ __forceinline__ void sum_channels(float (&v)[8], int lane) {
#pragma unroll
  for (int half = 4; half >= kLeft<LN>; half /= 2) {
    const int bit = 4 * half;
    const bool hi = lane & bit;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float send = hi ? v[i] : v[half + i];
      v[i] = (hi ? v[half + i] : v[i]) + __shfl_xor_sync(~0u, send, bit);
    }
  }
#pragma unroll
  for (int bit = 2; bit >= LN; bit /= 2) v[0] += __shfl_xor_sync(~0u, v[0], bit);
}
template <int LN>
__device__ __forceinline__ int summed(int lane) {
  return (lane >> 4 & 1) * 4 + (LN <= 8 ? (lane >> 3 & 1) * 2 : 0) + (LN <= 4 ? lane >> 2 & 1 : 0);
}

// ENDS: only the gradient that each segment hands to the one before it.
template <typename T, int LN, bool ROWS, bool MULTI, bool ENDS>
__global__ void __launch_bounds__(kSelThreads, kBwdCtas) sel_bwd_kernel(const __grid_constant__ SelArgs a) {
  using Smem = BwdSmem<LN>;
  constexpr int TT = Smem::T, PITCH = Smem::PITCH;
  using Where = Tile<kSelThreads, LN, ROWS>;
  constexpr int K = Where::K;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float biases[2 * Where::PAIRS];
  SelFlags& flags = *reinterpret_cast<SelFlags*>(smem);
  float4* io = reinterpret_cast<float4*>(smem + Smem::kFlags);
  float4* io2 = reinterpret_cast<float4*>(smem + Smem::kFlags + Smem::kIo);
  float2* dzfs = reinterpret_cast<float2*>(smem + Smem::kFlags + 2 * Smem::kIo);  // dout silu'(z)
  float* sub = reinterpret_cast<float*>(smem + Smem::kFlags + 2 * Smem::kIo + Smem::kDz) + threadIdx.x * 4;
  float* slabs = reinterpret_cast<float*>(smem + Smem::kFlags + 2 * Smem::kIo + Smem::kDz + Smem::kSub);
  float* bc = slabs + kWarps * Smem::kSlab / 4;
  const int np = static_cast<int>(a.padded), blocks = MULTI ? a.blocks : 1, wide = 4 * LN * blocks;
  float* held = bc + TT * 2 * wide + threadIdx.x * 4;  // of each pass: g carried, dA, its low part
  float2* sums = reinterpret_cast<float2*>(bc + TT * 2 * wide + blocks * 6 * kHalf);

  const SelPlace p = sel_place<LN>(a);
  if (ENDS && p.seg == 0) return;  // nothing is before it
  const int tid = threadIdx.x, sl = tid % LN, c = tid / LN, lane = tid & 31, warp = tid >> 5;
  const int mine = p.channels - 2 * c;  // of the thread's two channels, those that exist
  const int64_t ch = p.ch0 + (mine > 0 ? 2 * c : 0);
  grid_dependency_wait();
  for (int i = tid; i < 2 * Where::PAIRS; i += kSelThreads)
    biases[i] = i < p.channels && a.bias.data ? load_any(a.bias.data, a.bias.dtype, (p.ch0 + i) * a.bias.s0) : 0.f;
  __syncthreads();
  auto of_pair = [](const float* v, int k) { return make_float2(v[2 * Where::c(k)], v[2 * Where::c(k) + 1]); };
  const float2 bias = of_pair(biases, 0);  // unless along the sequence
  float2 skip = both(0.f);
  if (a.D.data && mine > 0) skip.x = load_any(a.D.data, a.D.dtype, ch * a.D.s0);
  if (a.D.data && mine > 1) skip.y = load_any(a.D.data, a.D.dtype, (ch + 1) * a.D.s0);

  Eight rate, carry;
  float2 dbias = both(0.f), dbias_low = both(0.f), dskip = both(0.f), dskip_low = both(0.f);
  float2 total = both(0.f);
  for (int nb = 0; nb < blocks; ++nb) {
    const int n0 = nb * 4 * LN + sl * kSelStates, n = n0 < np ? mine : 0;
    rate = load_rates(a, ch, n0, n);
    carry = ENDS ? zero8() : handed_over(a, p.b, a.segments - 1, p.seg, -1, ch, n0, n, rate);
    if constexpr (MULTI) put8(held + nb * 6 * kHalf, kHalf, carry);
    put8(held + (nb * 6 + 2) * kHalf, kHalf, zero8());
    put8(held + (nb * 6 + 4) * kHalf, kHalf, zero8());
  }

  // where this lane's sums over channels of the first position go
  const int which = summed<LN>(lane);
  float* slab = slabs + warp * (Smem::kSlab / 4) + (which >> 2) * 4 * LN + sl * 4 + (which & 3);
  const Walk<T, Where> xs(a.x, p), deltas(a.delta, p), zs(a.z.data ? a.z : a.x, p), douts(a.dout, p);
  const Walk<T, Where> dxs(a.dx, p), ddeltas(a.ddelta, p), dzs(a.z.data ? a.dz : a.dx, p);
  const bool all_channels = p.channels == 2 * Where::PAIRS, packed = a.seq_idx.data != nullptr;
  Raw next_x[K], next_delta[K], next_z[K], next_dout[K];
  FlagFeed<TT> feed;
  Coefficients<T, kSelThreads, LN, MULTI> next_bc(a, p);
  auto inside = [&](int64_t i) { return all_channels && (i + 1) * TT <= a.seqlen; };
  auto fetch = [&](int64_t i) {
    const bool whole = inside(i);
    xs.load(a, a.x, p, i, whole, next_x);
    deltas.load(a, a.delta, p, i, whole, next_delta);
    douts.load(a, a.dout, p, i, whole, next_dout);
    if (a.z.data) zs.load(a, a.z, p, i, whole, next_z);
    feed.load(a, p.b, i * TT);
    next_bc.load(a, i * TT, whole);
  };
  for (int64_t i = p.chunk1 - 1; i >= p.chunk0; --i) {
    // one latency of memory for 32 positions, which the CTAs beside this one fill: registers for
    // inputs that are loaded ahead would cost more
    fetch(i);
    const int64_t t0 = i * TT;
    const bool whole = inside(i), checked = packed || !whole;
    feed.store(a, p.b, t0, flags);
    if (checked || MULTI) __syncthreads();  // flags are there
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float2 u = fadd2(pair_of<T>(next_delta[k], a.pairs), ROWS ? of_pair(biases, k) : bias), x = pair_of<T>(next_x[k], a.pairs);
      float2 slope = both(1.f), dzf = both(0.f), dy = pair_of<T>(next_dout[k], a.pairs);
      const float2 s = a.softplus ? step_size<T>(u, &slope) : u;
      if (a.z.data) {
        // silu(z) = z r and silu'(z) = r + z r (1 - r)
        float2 r, less;
        const float2 z = pair_of<T>(next_z[k], a.pairs);
        sigmoid_pair_of<T>(z.x, r.x, less.x);
        sigmoid_pair_of<T>(z.y, r.y, less.y);
        const float2 zr = fmul2(z, r);
        dzf = fmul2(dy, ffma2(zr, less, r));
        dy = fmul2(dy, zr);
      }
      float4 v = make_float4(s.x, s.y, x.x, x.y), w = make_float4(dy.x, dy.y, slope.x, slope.y);
      if (checked) {
        const int has = flags.valid(Where::t(k)) ? p.channels - 2 * Where::c(k) : 0;
        if (has < 1) v.x = v.z = w.x = w.z = dzf.x = 0.f;
        if (has < 2) v.y = v.w = w.y = w.w = dzf.y = 0.f;
      }
      io[Where::t(k) * PITCH + Where::c(k)] = v;
      io2[Where::t(k) * PITCH + Where::c(k)] = w;
      if (a.z.data) dzfs[Where::t(k) * PITCH + Where::c(k)] = dzf;
    }
    next_bc.store(a, p, t0, checked, flags, bc);
    __syncthreads();

    for (int nb = 0; nb < blocks; ++nb) {
      const int n0 = nb * 4 * LN + sl * kSelStates, n = n0 < np ? mine : 0;
      if constexpr (MULTI) {
        carry = take8(held + nb * 6 * kHalf, kHalf);
        rate = load_rates(a, ch, n0, n);
      }
      const float* row = bc + nb * 4 * LN + sl * 4;
      Eight h;
      auto advance = [&](int t) {
        const float4 v = io[t * PITCH + c];
        const float2 s = make_float2(v.x, v.y), sx = fmul2(s, make_float2(v.z, v.w));
        const Eight decay = decays8(s, rate);
        const Quad B = quad(row + t * 2 * wide);
#pragma unroll
        for (int e = 0; e < 4; ++e) h.v[e] = ffma2(decay.v[e], h.v[e], fmul2(both(B.v[e]), sx));
      };
      if constexpr (!ENDS) {
        h = load8(a.checkpoints + ((p.b * a.nchunks + i) * a.dim + ch) * np + n0, np, n);
#pragma unroll 1
        for (int q = 0; q < TT / 4; ++q) {
          put8(sub + q * 2 * kHalf, kHalf, h);
          if (q == TT / 4 - 1) break;
          const uint32_t f = flags.word[q];
          if (f == kAllInside) {
#pragma unroll
            for (int j = 0; j < 4; ++j) advance(q * 4 + j);
          } else {
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
              if (f >> (8 * j) & kFirst) h = load_states(a.init, flags.row[q * 4 + j], ch, n0, a.dstate, n);
              advance(q * 4 + j);
            }
          }
        }
      }
      Eight da = zero8();  // of this tile
      float2 tile_bias = both(0.f), tile_skip = both(0.f);
      // The sums of a position's dB and dC over the warp's channels, to the warp's slab.
      auto keep_channels = [&](int t, float2 (&b)[8]) {
        if (!all_channels) {  // so that 0 * infinity of no channel does not count
#pragma unroll
          for (int e = 0; e < 8; ++e) b[e] = make_float2(mine > 0 ? b[e].x : 0.f, mine > 1 ? b[e].y : 0.f);
        }
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = b[e].x + b[e].y;
        sum_channels<LN>(v, lane);
#pragma unroll
        for (int e = 0; e < kLeft<LN>; ++e)
          if ((lane & 3) < LN) slab[t * 8 * LN + e] = v[e];
      };
      // One position, from the gradient carried to it: h before it in `kept` times its decay.
      // y, sa, sb: the thread's parts of the sums over the states of C h, g a h_{t-1} A and g B.
      auto retreat = [&](int t, const Eight& decay, const Eight& kept, float2& y, float2& sa, float2& sb, float2 (&v)[8]) {
        const float4 in = io[t * PITCH + c];
        const float2 s = make_float2(in.x, in.y), x = make_float2(in.z, in.w);
        const float2 dy = *reinterpret_cast<const float2*>(&io2[t * PITCH + c]);
        const Quad B = quad(row + t * 2 * wide), C = quad(row + t * 2 * wide + wide);
        const float2 sx = fmul2(s, x);
        y = sa = sb = both(0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 g = ffma2(both(C.v[e]), dy, carry.v[e]);
          const float2 now = ffma2(both(B.v[e]), sx, kept.v[e]);
          const float2 w = fmul2(g, kept.v[e]);
          carry.v[e] = fmul2(decay.v[e], g);
          v[e] = fmul2(g, sx);
          v[4 + e] = fmul2(now, dy);
          y = ffma2(both(C.v[e]), now, y);
          sb = ffma2(both(B.v[e]), g, sb);
          sa = ffma2(w, rate.v[e], sa);
          da.v[e] = ffma2(w, s, da.v[e]);
        }
      };
#pragma unroll 1
      for (int q = TT / 4 - 1; q >= 0; --q) {
        const uint32_t f = flags.word[q];
        float2 y[4], sa[4], sb[4];
        if (f == kAllInside) {
          Eight decay[4], kept[4];  // a and a h_{t-1} of the four positions
          if (!ENDS) h = take8(sub + q * 2 * kHalf, kHalf);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 v = io[(q * 4 + j) * PITCH + c];
            const float2 s = make_float2(v.x, v.y), sx = fmul2(s, make_float2(v.z, v.w));
            decay[j] = decays8(s, rate);
            if constexpr (!ENDS) {
              const Quad B = quad(row + (q * 4 + j) * 2 * wide);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                kept[j].v[e] = fmul2(decay[j].v[e], h.v[e]);
                h.v[e] = ffma2(both(B.v[e]), sx, kept[j].v[e]);
              }
            }
          }
#pragma unroll
          for (int j = 3; j >= 0; --j) {
            const int t = q * 4 + j;
            if constexpr (!ENDS) {
              float2 v[8];
              retreat(t, decay[j], kept[j], y[j], sa[j], sb[j], v);
              keep_channels(t, v);
            } else {
              const float4 in = io[t * PITCH + c];
              const float2 dy = *reinterpret_cast<const float2*>(&io2[t * PITCH + c]);
              const Quad C = quad(row + t * 2 * wide + wide);
#pragma unroll
              for (int e = 0; e < 4; ++e) carry.v[e] = fmul2(decay[j].v[e], ffma2(both(C.v[e]), dy, carry.v[e]));
              if (nb == 0) total = fadd2(total, make_float2(in.x, in.y));
            }
          }
        } else {
          // ends of sequences or padding: one position at a time, its state anew from the group's
#pragma unroll 1
          for (int j = 3; j >= 0; --j) {
            const int t = q * 4 + j, r = flags.row[t];
            const uint32_t fj = f >> (8 * j);
            float2 yj = both(0.f), saj = both(0.f), sbj = both(0.f);
            float2 v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = both(0.f);
            if (fj & kValid) {
              const float4 in = io[t * PITCH + c];
              const Eight decay = decays8(make_float2(in.x, in.y), rate);
              if (fj & kLast) carry = load_states(a.dfinal, r, ch, n0, a.dstate, n);
              if constexpr (!ENDS) {
                h = take8(sub + q * 2 * kHalf, kHalf);
#pragma unroll 1
                for (int k = 0; k < j; ++k) {
                  if (f >> (8 * k) & kFirst) h = load_states(a.init, flags.row[q * 4 + k], ch, n0, a.dstate, n);
                  advance(q * 4 + k);
                }
                if (fj & kFirst) h = load_states(a.init, r, ch, n0, a.dstate, n);
                Eight kept;
#pragma unroll
                for (int e = 0; e < 4; ++e) kept.v[e] = fmul2(decay.v[e], h.v[e]);
                retreat(t, decay, kept, yj, saj, sbj, v);
              } else {
                const float2 dy = *reinterpret_cast<const float2*>(&io2[t * PITCH + c]);
                const Quad C = quad(row + t * 2 * wide + wide);
#pragma unroll
                for (int e = 0; e < 4; ++e) carry.v[e] = fmul2(decay.v[e], ffma2(both(C.v[e]), dy, carry.v[e]));
                if (nb == 0) total = fadd2(total, make_float2(in.x, in.y));
              }
              if (fj & kFirst) {
                if (!ENDS) store_states(a.dinit, r, ch, n0, a.dstate, n, carry);
                if (ENDS) total = both(INFINITY);
                carry = zero8();
              }
            }
            if constexpr (!ENDS) {
              keep_channels(t, v);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (e == j) y[e] = yj, sa[e] = saj, sb[e] = sbj;
            }
          }
        }
        if constexpr (!ENDS) {
          float l[3][2][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            l[0][0][j] = y[j].x, l[0][1][j] = y[j].y;
            l[1][0][j] = sa[j].x, l[1][1][j] = sa[j].y;
            l[2][0][j] = sb[j].x, l[2][1][j] = sb[j].y;
          }
#pragma unroll
          for (int e = 0; e < 6; ++e) sum_lanes<LN>(l[e / 2][e % 2], sl);
#pragma unroll
          for (int j = 0; j < kSums<LN>; ++j) {
            if (sl >= 4) break;
            const int t = q * 4 + first_sum<LN>(sl) + j;
            float2 yt = make_float2(l[0][0][j], l[0][1][j]), sat = make_float2(l[1][0][j], l[1][1][j]), sbt = make_float2(l[2][0][j], l[2][1][j]);
            if constexpr (MULTI) {
              float2* s = sums + (t * PITCH + c) * 3;
              if (nb > 0) yt = fadd2(yt, s[0]), sat = fadd2(sat, s[1]), sbt = fadd2(sbt, s[2]);
              if (nb + 1 < blocks) {
                s[0] = yt, s[1] = sat, s[2] = sbt;
                continue;
              }
            }
            const float4 in = io[t * PITCH + c], in2 = io2[t * PITCH + c];
            const float2 s = make_float2(in.x, in.y), x = make_float2(in.z, in.w), dy = make_float2(in2.x, in2.y);
            const float2 du = fmul2(ffma2(sat, both(0.693147181f), fmul2(x, sbt)), make_float2(in2.z, in2.w));
            const float2 dx = ffma2(s, sbt, fmul2(skip, dy));
            io[t * PITCH + c] = make_float4(dx.x, dx.y, du.x, du.y);
            *reinterpret_cast<float2*>(&io2[t * PITCH + c]) = ffma2(skip, x, yt);
            tile_bias = fadd2(tile_bias, du);
            tile_skip = ffma2(dy, x, tile_skip);
          }
        }
      }
      if constexpr (MULTI) put8(held + nb * 6 * kHalf, kHalf, carry);
      if constexpr (!ENDS) {
        add_to(dbias, dbias_low, tile_bias);
        add_to(dskip, dskip_low, tile_skip);
        Eight hi = take8(held + (nb * 6 + 2) * kHalf, kHalf), lo = take8(held + (nb * 6 + 4) * kHalf, kHalf);
#pragma unroll
        for (int e = 0; e < 4; ++e) add_to(hi.v[e], lo.v[e], da.v[e]);
        put8(held + (nb * 6 + 2) * kHalf, kHalf, hi);
        put8(held + (nb * 6 + 4) * kHalf, kHalf, lo);
        __syncthreads();
        // this pass's states of dB and dC: the warps' sums to the CTA's.  A thread has the same values
        // of every STEP-th position, one or two of them.
        constexpr int STEP = 8 * LN < kSelThreads ? kSelThreads / (8 * LN) : 1;
        const int count = static_cast<int>(a.seqlen - t0 < TT ? a.seqlen - t0 : TT);
#pragma unroll
        for (int more = 0; more < 8 * LN; more += kSelThreads) {
          const int v = tid % (8 * LN) + more, m = nb * 4 * LN + v % (4 * LN), first = tid / (8 * LN);
          if (m >= np) continue;
          const float* from = slabs + first * 8 * LN + v;
          const int64_t row_size = a.tiles * 2 * np;
          float* to = a.parts_bc + ((p.b - a.row0) * a.seqlen + t0 + first) * row_size + (p.tile * 2 + v / (4 * LN)) * np + m;
#pragma unroll 4
          for (int t = first; t < count; t += STEP, to += STEP * row_size, from += STEP * 8 * LN) {
            float r = from[0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) r += from[w * (Smem::kSlab / 4)];
            *to = r;
          }
        }
        if (nb + 1 < blocks) __syncthreads();
      }
    }
    if constexpr (!ENDS) {
      float2 o[K];
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        if (part == 2 && !a.z.data) break;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int at = Where::t(k) * PITCH + Where::c(k);
          const float4* from = part == 2 ? &io2[at] : &io[at];
          o[k] = reinterpret_cast<const float2*>(from)[part == 1];
          if (part == 2) o[k] = fmul2(o[k], dzfs[at]);
        }
        if (packed)
#pragma unroll
          for (int k = 0; k < K; ++k)
            if (!flags.valid(Where::t(k))) o[k] = both(0.f);
        if (part == 0) dxs.store(a, a.dx, p, i, whole, o);
        else if (part == 1) ddeltas.store(a, a.ddelta, p, i, whole, o);
        else dzs.store(a, a.dz, p, i, whole, o);
      }
    }
    __syncthreads();
  }

  const int64_t part = p.b * a.segments + p.seg;
  for (int nb = 0; nb < blocks; ++nb) {
    const int n0 = nb * 4 * LN + sl * kSelStates, n = n0 < np ? mine : 0;
    if constexpr (ENDS) {
      if constexpr (MULTI) carry = take8(held + nb * 6 * kHalf, kHalf);
      store8(a.ends + (part * a.dim + ch) * np + n0, np, n, carry);
    } else {
      Eight hi = take8(held + (nb * 6 + 2) * kHalf, kHalf);
      const Eight lo = take8(held + (nb * 6 + 4) * kHalf, kHalf);
#pragma unroll
      for (int e = 0; e < 4; ++e) hi.v[e] = fadd2(hi.v[e], lo.v[e]);
      store8(a.parts_a + (part * a.dim + ch) * np + n0, np, n, hi);
    }
  }
  float2 one = total, two = both(0.f);
  if constexpr (!ENDS) {
    one = fadd2(dskip, dskip_low);
    two = fadd2(dbias, dbias_low);
#pragma unroll
    for (int bit = 1; bit < LN; bit *= 2) {
      one = fadd2(one, make_float2(__shfl_xor_sync(~0u, one.x, bit), __shfl_xor_sync(~0u, one.y, bit)));
      two = fadd2(two, make_float2(__shfl_xor_sync(~0u, two.x, bit), __shfl_xor_sync(~0u, two.y, bit)));
    }
  }
  if (sl != 0) return;
  float* d = ENDS ? a.steps + part * a.dim + ch : a.parts_d + part * 2 * a.dim + ch;
  if (mine > 0) d[0] = one.x;
  if (mine > 1) d[1] = one.y;
  if (!ENDS && mine > 0) d[a.dim] = two.x;
  if (!ENDS && mine > 1) d[a.dim + 1] = two.y;
}

// dB and dC: the sums over a group's CTAs.  Four threads take four states of a position, each of them
// every fourth CTA, in loads of 16 bytes of which eight are on their way.  One state and all CTAs a
// thread made the backward of 4 x 4096 x 1024 x 16 take 613 us, this 599.
constexpr int kSumQuads = kThreads / 4;
template <typename T>
__global__ void __launch_bounds__(kThreads) sel_sum_bc_kernel(const __grid_constant__ SelArgs a) {
  grid_dependency_wait();
  const int64_t per = 2 * a.padded, quads = per / 4, rows = a.group_tiles;
  const int lane = threadIdx.x & 31, share = lane >> 3;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kSumQuads + (threadIdx.x >> 5) * 8 + (lane & 7);
  const bool is = i < a.launch_rows * a.seqlen * a.groups * quads;
  const int64_t v = is ? i % quads * 4 : 0, r = is ? i / quads : 0, g = r % a.groups, bt = r / a.groups;
  const float* part = a.parts_bc + (bt * a.tiles + g * rows) * per + v;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (is) {
#pragma unroll 8
    for (int64_t k = share; k < rows; k += 4) {
      const float4 p = *reinterpret_cast<const float4*>(part + k * per);
      s[0] += p.x;
      s[1] += p.y;
      s[2] += p.z;
      s[3] += p.w;
    }
  }
  float sum = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    s[e] += __shfl_xor_sync(~0u, s[e], 8);
    s[e] += __shfl_xor_sync(~0u, s[e], 16);
    if (e == share) sum = s[e];
  }
  const bool is_c = v >= a.padded;
  const int64_t n = (is_c ? v - a.padded : v) + share;
  if (!is || n >= a.dstate) return;
  const TensorArg& t = is_c ? a.dC : a.dB;
  static_cast<T*>(t.data)[(a.row0 + bt / a.seqlen) * t.s0 + g * (is_c ? a.dC_group : a.dB_group) + n * t.s1 + (bt % a.seqlen) * t.s2] = from_f32<T>(sum);
}

// dA, dD and dbias: the sums over batch rows and segments.
__global__ void __launch_bounds__(kThreads) sel_sum_params_kernel(const __grid_constant__ SelArgs a) {
  grid_dependency_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t na = a.dim * a.padded, rows = a.batch * a.segments;
  if (i >= na + 2 * a.dim) return;
  const bool is_a = i < na;
  const float* part = is_a ? a.parts_a + i : a.parts_d + (i - na);
  const int64_t step = is_a ? na : 2 * a.dim;
  float s = 0.f, low = 0.f;
#pragma unroll 4
  for (int64_t k = 0; k < rows; ++k) add_to(s, low, part[k * step]);
  s += low;
  if (is_a) {
    const int64_t d = i / a.padded, n = i - d * a.padded;
    if (a.dA && n < a.dstate) a.dA[d * a.dstate + n] = s;
  } else if (i - na < a.dim) {
    if (a.dD) a.dD[i - na] = s;
  } else if (a.dbias) {
    a.dbias[i - na - a.dim] = s;
  }
}

template <typename T, int LN, bool ROWS, bool MULTI, bool ENDS>
cudaError_t launch(const SelArgs& a, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(BwdSmem<LN>::bytes(a));
  const auto kernel = sel_bwd_kernel<T, LN, ROWS, MULTI, ENDS>;
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(a.launch_rows * a.segments * a.tiles)), dim3(kSelThreads), smem, s, a);
}

template <typename T, int LN, bool ROWS, bool MULTI = false>
cudaError_t walk(const SelArgs& a, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (a.segments > 1) e = launch<T, LN, ROWS, MULTI, true>(a, s);
  return e == cudaSuccess ? launch<T, LN, ROWS, MULTI, false>(a, s) : e;
}
template <typename T>
cudaError_t walk(const SelArgs& a, cudaStream_t s) {
  if (a.blocks > 1) return a.rows ? walk<T, kSelLanes, true, true>(a, s) : walk<T, kSelLanes, false, true>(a, s);
  switch (a.lanes) {
    case 1: return a.rows ? walk<T, 1, true>(a, s) : walk<T, 1, false>(a, s);
    case 2: return a.rows ? walk<T, 2, true>(a, s) : walk<T, 2, false>(a, s);
    case 4: return a.rows ? walk<T, 4, true>(a, s) : walk<T, 4, false>(a, s);
    case 8: return a.rows ? walk<T, 8, true>(a, s) : walk<T, 8, false>(a, s);
    default: return a.rows ? walk<T, 16, true>(a, s) : walk<T, 16, false>(a, s);
  }
}

template <typename T>
cudaError_t run(const SelArgs& all, cudaStream_t s) {
  SelArgs a = all;
  cudaError_t e = cudaSuccess;
  const int64_t params = a.dim * (a.padded + 2);
  for (a.row0 = 0; e == cudaSuccess && a.row0 < a.batch; a.row0 += all.launch_rows) {
    if (a.launch_rows > a.batch - a.row0) a.launch_rows = a.batch - a.row0;
    const int64_t quads = a.launch_rows * a.seqlen * a.groups * a.padded / 2;
    if (a.dim > 0) e = walk<T>(a, s);
    if (e == cudaSuccess)
      e = launch_dependent(sel_sum_bc_kernel<T>, dim3(static_cast<unsigned>((quads + kSumQuads - 1) / kSumQuads)), dim3(kThreads), 0, s, a);
  }
  if (e == cudaSuccess && a.dim > 0)
    e = launch_dependent(sel_sum_params_kernel, dim3(static_cast<unsigned>((params + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
  return e;
}

}  // namespace

cudaError_t CC1D_DT_NAME(sel_bwd)(const SelArgs& a, cudaStream_t s) { return run<CC1D_DT_TYPE>(a, s); }

}  // namespace cc1d
