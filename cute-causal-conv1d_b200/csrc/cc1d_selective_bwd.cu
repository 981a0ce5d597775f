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
// CTAs, threads and tiles are the forward's; a CTA goes through its tiles from the last one back.
// From the state that the forward kept before a tile it runs forward, keeping the state before
// every fourth position, then takes the groups of four positions from the last one back: states
// again, then gradients.  dB and dC are summed over the warp's channels by exchanges between
// lanes, over the CTA's warps in shared memory and over CTAs by a second kernel, all in a fixed
// order.
#include "cc1d_selective.cuh"

namespace cc1d {
namespace {

constexpr int kWarps = kSelThreads / 32;
#ifndef BWDC
#define BWDC 3
#endif
constexpr int kBwdCtas = BWDC;

// Shared memory: flags; (s, x, dy, slope of the step size), replaced by (dx, ddelta, y), by position
// and channel; the states before every fourth position; each warp's sums of dB and dC; B and C;
// with several passes three sums by position and channel, and the states between two tiles.
template <typename T, int LN>
struct BwdSmem {
  static constexpr int kFlags = 256, TT = Tile<LN, false>::T, PITCH = Tile<LN, false>::PITCH;
  static constexpr int kIo = TT * PITCH * 16;
  static constexpr int kSums = (TT * PITCH * 12 + 15) / 16 * 16;
  static constexpr int kSub = TT / 4 * kSelThreads * 16;
  static constexpr int kSlab = TT * 8 * LN * 4;  // one warp's
  static int64_t bytes(const SelArgs& a) {
    return kFlags + kIo + kSub + kWarps * kSlab + TT * 8 * LN * a.blocks * static_cast<int>(sizeof(T)) +
           (a.blocks > 1 ? kSums + 3ll * a.blocks * kSelThreads * 16 : 0);
  }
};

// Adds v to the sum hi + lo, which together hold twice the bits (Knuth's two-sum).
__device__ __forceinline__ void add_to(float& hi, float& lo, float v) {
  const float s = hi + v;
  const float w = s - hi;
  lo += (hi - (s - w)) + (v - w);
  hi = s;
}
__device__ __forceinline__ void add_to(Four& hi, Four& lo, const Four& v) {
  add_to(hi.lo.x, lo.lo.x, v.lo.x);
  add_to(hi.lo.y, lo.lo.y, v.lo.y);
  add_to(hi.hi.x, lo.hi.x, v.hi.x);
  add_to(hi.hi.y, lo.hi.y, v.hi.y);
}

// The sums of a's and b's four values over the channels of a warp.  A lane ends with one of the
// eight, the number of which summed() tells; lanes that differ in further bits hold the same one.
template <int LN>
__device__ __forceinline__ float sum_channels(const Four& a, const Four& b, int lane) {
  float v[8] = {a.lo.x, a.lo.y, a.hi.x, a.hi.y, b.lo.x, b.lo.y, b.hi.x, b.hi.y};
#pragma unroll
  for (int half = 4; half >= 1; half /= 2) {
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
  return v[0];
}
__device__ __forceinline__ int summed(int lane) { return (lane >> 4 & 1) * 4 + (lane >> 3 & 1) * 2 + (lane >> 2 & 1); }

// ENDS: only the gradient that each segment hands to the one before it.
template <typename T, int LN, bool ROWS, bool MULTI, bool ENDS>
__global__ void __launch_bounds__(kSelThreads, ENDS ? 4 : kBwdCtas) sel_bwd_kernel(const __grid_constant__ SelArgs a) {
  using Where = Tile<LN, ROWS>;
  using Smem = BwdSmem<T, LN>;
  constexpr int PITCH = Where::PITCH, TT = Where::T;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float biases[Where::CH];
  SelFlags& flags = *reinterpret_cast<SelFlags*>(smem);
  float4* io = reinterpret_cast<float4*>(smem + Smem::kFlags);
  float* sub = reinterpret_cast<float*>(smem + Smem::kFlags + Smem::kIo);
  float* slabs = reinterpret_cast<float*>(smem + Smem::kFlags + Smem::kIo + Smem::kSub);
  T* bc = reinterpret_cast<T*>(slabs + kWarps * Smem::kSlab / 4);
  const int np = static_cast<int>(a.padded), blocks = MULTI ? a.blocks : 1, wide = 4 * LN * blocks;
  float* held = reinterpret_cast<float*>(bc + TT * 2 * wide);  // several passes: g carried, dA and its low part
  float* sums = held + 3 * blocks * kSelThreads * 4;

  const SelPlace p = sel_place<LN>(a);
  const int tid = threadIdx.x, sl = tid % LN, c = tid / LN, lane = tid & 31, warp = tid >> 5;
  const bool mine = c < p.channels;
  const int64_t ch = p.ch0 + (mine ? c : 0);
  grid_dependency_wait();
  for (int i = tid; i < Where::CH; i += kSelThreads)
    biases[i] = i < p.channels && a.bias.data ? load_any(a.bias.data, a.bias.dtype, (p.ch0 + i) * a.bias.s0) : 0.f;

  __syncthreads();
  const float bias = biases[Where::c()];  // of the thread's channel, unless along the sequence
  const float skip = a.D.data && mine ? load_any(a.D.data, a.D.dtype, ch * a.D.s0) : 0.f;
  Four rate = zero4(), carry = zero4(), da = zero4(), da_low = zero4();
  float dbias = 0.f, dbias_low = 0.f, dskip = 0.f, dskip_low = 0.f;
  float total = 0.f;
  const int64_t ends_at = (p.b * a.segments * a.dim + ch) * np;
  for (int nb = 0; nb < blocks; ++nb) {
    const int n0 = nb * kSelBlock + sl * kSelStates;
    const bool has = n0 < np;
    rate = mine && has ? load_rates(a, ch, n0) : zero4();
    carry = zero4();
    if (!ENDS && mine && has)
      for (int64_t s = a.segments - 1; s > p.seg; --s)
        carry = handed_on(carry, rate, a.steps[(p.b * a.segments + s) * a.dim + ch], load4(a.ends + ends_at + s * a.dim * np + n0));
    if constexpr (MULTI) {
      store4(held + (nb * 3 * kSelThreads + tid) * 4, carry);
      store4(held + ((nb * 3 + 1) * kSelThreads + tid) * 4, zero4());
      store4(held + ((nb * 3 + 2) * kSelThreads + tid) * 4, zero4());
    }
  }

  // where this lane's sums over channels of the first position go
  const int which = summed(lane);
  float* slab = slabs + warp * (Smem::kSlab / 4) + (which >> 2) * 4 * LN + sl * 4 + (which & 3);
  const Walk<T, LN, ROWS> xs(a.x, p), deltas(a.delta, p), zs(a.z.data ? a.z : a.x, p), douts(a.dout, p);
  const Walk<T, LN, ROWS> dxs(a.dx, p), ddeltas(a.ddelta, p), dzs(a.z.data ? a.dz : a.dx, p);
  const bool all_channels = p.channels == Where::CH, packed = a.seq_idx.data != nullptr;
  T next_x[8], next_delta[8], next_z[8], next_dout[8];
  float dzf[8];  // dout silu'(z)
  FlagFeed<TT> feed;
  Coefficients<T, LN, MULTI> next_bc(a, p);
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
  fetch(p.chunk1 - 1);
  for (int64_t i = p.chunk1 - 1; i >= p.chunk0; --i) {
    const int64_t t0 = i * TT;
    const bool whole = inside(i);
    feed.store(a, p.b, t0, flags);
    __syncthreads();
    const bool checked = packed || !whole;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int t = Where::t() + k * Where::DT, cc = Where::c() + k * Where::DC;
      const float u = to_f32(next_delta[k]) + (ROWS ? biases[cc] : bias);
      float slope = 1.f, dy = to_f32(next_dout[k]);
      const float s = a.softplus ? step_size<T>(u, &slope) : u;
      if (a.z.data) {
        // silu(z) = z r and silu'(z) = r + z r (1 - r)
        float r, less;
        const float z = to_f32(next_z[k]);
        sigmoid_pair_of<T>(z, r, less);
        dzf[k] = dy * fmaf(z * r, less, r);
        dy *= z * r;
      }
      io[t * PITCH + cc] = make_float4(s, to_f32(next_x[k]), dy, slope);
    }
    if (checked)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int t = Where::t() + k * Where::DT, cc = Where::c() + k * Where::DC;
        if (!flags.valid(t) || cc >= p.channels) {
          io[t * PITCH + cc] = make_float4(0.f, 0.f, 0.f, 0.f);
          dzf[k] = 0.f;
        }
      }
    next_bc.store(a, p, t0, checked, flags, bc);
    __syncthreads();
    if (i > p.chunk0) fetch(i - 1);

    for (int nb = 0; nb < blocks; ++nb) {
      const int n0 = nb * kSelBlock + sl * kSelStates;
      const bool has = n0 < np;
      if constexpr (MULTI) {
        carry = load4(held + (nb * 3 * kSelThreads + tid) * 4);
        rate = mine && has ? load_rates(a, ch, n0) : zero4();
      }
      const T* row = bc + nb * 4 * LN + sl * 4;
      Four h = zero4();
      auto start = [&](int t) {
        const int r = flags.row[t];
        h = a.init.data && r >= 0 && mine && has ? load_state(a.init, r, ch, n0, a.dstate) : zero4();
      };
      auto advance = [&](int t) {
        const float4 v = io[t * PITCH + c];
        const float sx = v.x * v.y;
        h = fma4(decays4(make_float2(v.x, v.x), rate), h, mul4(load4_of(row + t * 2 * wide), make_float2(sx, sx)));
      };
      if constexpr (!ENDS) {
        if (mine && has) h = load4(a.checkpoints + ((p.b * a.nchunks + i) * a.dim + ch) * np + n0);
#pragma unroll 1
        for (int q = 0; q < TT / 4; ++q) {
          store4(sub + (q * kSelThreads + tid) * 4, h);
          if (q == TT / 4 - 1) break;
          const uint32_t f = flags.word[q];
          if (f == kAllInside) {
#pragma unroll
            for (int j = 0; j < 4; ++j) advance(q * 4 + j);
          } else {
#pragma unroll 1
            for (int j = 0; j < 4; ++j) {
              if (f >> (8 * j) & kFirst) start(q * 4 + j);
              advance(q * 4 + j);
            }
          }
        }
      }
      Four da_tile = zero4();
      // The sums of a position's dB and dC over the warp's channels, to the warp's slab.
      auto keep_channels = [&](int t, Four dB, Four dC) {
        if (!all_channels && !mine) dB = dC = zero4();  // so that 0 * infinity of no channel does not count
        const float v = sum_channels<LN>(dB, dC, lane);
        if ((lane & 3) < LN) slab[t * 8 * LN] = v;
      };
#pragma unroll 1
      for (int q = TT / 4 - 1; q >= 0; --q) {
        const uint32_t f = flags.word[q];
        float y[4], sa[4], sb[4];  // sums over the states of C h, g a h_{t-1} A and g B
        if (f == kAllInside) {
          Four decay[4], kept[4], now[4];  // a, a h_{t-1} and h of the four positions
          if (!ENDS) h = load4(sub + (q * kSelThreads + tid) * 4);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int t = q * 4 + j;
            const float4 v = io[t * PITCH + c];
            decay[j] = decays4(make_float2(v.x, v.x), rate);
            if constexpr (!ENDS) {
              const float sx = v.x * v.y;
              kept[j] = mul4(decay[j], h);
              h = now[j] = fma4(load4_of(row + t * 2 * wide), make_float2(sx, sx), kept[j]);
            }
          }
#pragma unroll
          for (int j = 3; j >= 0; --j) {
            const int t = q * 4 + j;
            const float4 v = io[t * PITCH + c];
            const float2 dy = make_float2(v.z, v.z);
            const Four C = load4_of(row + t * 2 * wide + wide);
            const Four g = fma4(C, dy, carry);
            carry = mul4(decay[j], g);
            if constexpr (!ENDS) {
              const float sx = v.x * v.y;
              const Four w = mul4(g, kept[j]);
              y[j] = dot4(C, now[j]);
              sb[j] = dot4(load4_of(row + t * 2 * wide), g);
              sa[j] = dot4(w, rate);
              da_tile = fma4(w, make_float2(v.x, v.x), da_tile);
              keep_channels(t, mul4(g, make_float2(sx, sx)), mul4(now[j], dy));
            } else {
              if (nb == 0) total += v.x;
            }
          }
        } else {
          // ends of sequences or padding: one position at a time, its state anew from the group's
#pragma unroll 1
          for (int j = 3; j >= 0; --j) {
            const int t = q * 4 + j, r = flags.row[t];
            const uint32_t fj = f >> (8 * j);
            float yj = 0.f, saj = 0.f, sbj = 0.f;
            Four dB = zero4(), dC = zero4();
            if (fj & kValid) {
              const float4 v = io[t * PITCH + c];
              const Four decay = decays4(make_float2(v.x, v.x), rate), C = load4_of(row + t * 2 * wide + wide);
              if (fj & kLast) carry = a.dfinal.data && r >= 0 && mine && has ? load_state(a.dfinal, r, ch, n0, a.dstate) : zero4();
              const Four g = fma4(C, make_float2(v.z, v.z), carry);
              if constexpr (!ENDS) {
                h = load4(sub + (q * kSelThreads + tid) * 4);
#pragma unroll 1
                for (int k = 0; k < j; ++k) {
                  if (f >> (8 * k) & kFirst) start(q * 4 + k);
                  advance(q * 4 + k);
                }
                if (fj & kFirst) start(t);
                const float sx = v.x * v.y;
                const Four B = load4_of(row + t * 2 * wide), kept = mul4(decay, h), now = fma4(B, make_float2(sx, sx), kept), w = mul4(g, kept);
                yj = dot4(C, now);
                sbj = dot4(B, g);
                saj = dot4(w, rate);
                da_tile = fma4(w, make_float2(v.x, v.x), da_tile);
                dB = mul4(g, make_float2(sx, sx));
                dC = mul4(now, make_float2(v.z, v.z));
              } else {
                if (nb == 0) total += v.x;
              }
              carry = mul4(decay, g);
              if (fj & kFirst) {
                if (!ENDS && a.dinit.data && r >= 0 && mine && has) store_state(a.dinit, r, ch, n0, a.dstate, carry);
                if (ENDS) total = INFINITY;
                carry = zero4();
              }
            }
            if constexpr (!ENDS) {
              keep_channels(t, dB, dC);
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (e == j) y[e] = yj, sa[e] = saj, sb[e] = sbj;
            }
          }
        }
        if constexpr (!ENDS) {
          sum_lanes<LN>(y, sl);
          sum_lanes<LN>(sa, sl);
          sum_lanes<LN>(sb, sl);
#pragma unroll
          for (int j = 0; j < 4 / LN; ++j) {
            const int t = q * 4 + sl * (4 / LN) + j;
            float* s = sums + (t * PITCH + c) * 3;
            if (MULTI && nb > 0) {
              y[j] += s[0];
              sa[j] += s[1];
              sb[j] += s[2];
            }
            if (MULTI && nb + 1 < blocks) {
              s[0] = y[j];
              s[1] = sa[j];
              s[2] = sb[j];
              continue;
            }
            const float4 v = io[t * PITCH + c];
            const float du = fmaf(sa[j], 0.693147181f, v.y * sb[j]) * v.w;
            io[t * PITCH + c] = make_float4(fmaf(v.x, sb[j], skip * v.z), du, fmaf(skip, v.y, y[j]), 0.f);
            add_to(dbias, dbias_low, du);
            add_to(dskip, dskip_low, v.z * v.y);
          }
        }
      }
      if constexpr (MULTI) store4(held + (nb * 3 * kSelThreads + tid) * 4, carry);
      if constexpr (!ENDS) {
        if constexpr (MULTI) {
          da = load4(held + ((nb * 3 + 1) * kSelThreads + tid) * 4);
          da_low = load4(held + ((nb * 3 + 2) * kSelThreads + tid) * 4);
        }
        add_to(da, da_low, da_tile);
        if constexpr (MULTI) {
          store4(held + ((nb * 3 + 1) * kSelThreads + tid) * 4, da);
          store4(held + ((nb * 3 + 2) * kSelThreads + tid) * 4, da_low);
        }
        __syncthreads();
        // this pass's states of dB and dC: the warps' sums to the CTA's
        for (int e = tid; e < TT * 8 * LN; e += kSelThreads) {
          const int t = e / (8 * LN), v = e % (8 * LN), n = nb * kSelBlock + v % (4 * LN);
          if (t0 + t >= a.seqlen || n >= np) continue;
          float s = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) s += slabs[w * (Smem::kSlab / 4) + e];
          a.parts_bc[(((p.b * a.seqlen + t0 + t) * a.tiles + p.tile) * 2 + v / (4 * LN)) * np + n] = s;
        }
        if (nb + 1 < blocks) __syncthreads();
      }
    }
    if constexpr (!ENDS) {
      float o[8];
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        if (part == 2 && !a.z.data) break;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int t = Where::t() + k * Where::DT, cc = Where::c() + k * Where::DC;
          const float4 v = io[t * PITCH + cc];
          o[k] = part == 0 ? v.x : part == 1 ? v.y : dzf[k] * v.z;
        }
        if (packed)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (!flags.valid(Where::t() + k * Where::DT)) o[k] = 0.f;
        if (part == 0) dxs.store(a, a.dx, p, i, whole, o);
        else if (part == 1) ddeltas.store(a, a.ddelta, p, i, whole, o);
        else dzs.store(a, a.dz, p, i, whole, o);
      }
    }
    __syncthreads();
  }

  for (int nb = 0; nb < blocks; ++nb) {
    const int n0 = nb * kSelBlock + sl * kSelStates;
    if (n0 >= np || !mine) continue;
    if constexpr (ENDS) {
      if constexpr (MULTI) carry = load4(held + (nb * 3 * kSelThreads + tid) * 4);
      store4(a.ends + ends_at + p.seg * a.dim * np + n0, carry);
    } else {
      if constexpr (MULTI) {
        da = load4(held + ((nb * 3 + 1) * kSelThreads + tid) * 4);
        da_low = load4(held + ((nb * 3 + 2) * kSelThreads + tid) * 4);
      }
      store4(a.parts_a + ((p.b * a.segments + p.seg) * a.dim + ch) * np + n0,
             Four{fadd2(da.lo, da_low.lo), fadd2(da.hi, da_low.hi)});
    }
  }
  if constexpr (ENDS) {
    if (mine && sl == 0) a.steps[(p.b * a.segments + p.seg) * a.dim + ch] = total;
    return;
  }
  dskip += dskip_low;
  dbias += dbias_low;
#pragma unroll
  for (int bit = 1; bit < LN; bit *= 2) {
    dskip += __shfl_xor_sync(~0u, dskip, bit);
    dbias += __shfl_xor_sync(~0u, dbias, bit);
  }
  if (mine && sl == 0) {
    float* d = a.parts_d + (p.b * a.segments + p.seg) * 2 * a.dim + ch;
    d[0] = dskip;
    d[a.dim] = dbias;
  }
}

// dB and dC: the sums over a group's CTAs.  A thread takes one state of one position.
template <typename T>
__global__ void __launch_bounds__(kThreads) sel_sum_bc_kernel(const __grid_constant__ SelArgs a) {
  grid_dependency_wait();
  const int64_t per = 2 * a.padded;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= a.batch * a.seqlen * a.groups * per) return;
  const int64_t v = i % per, r = i / per, g = r % a.groups, bt = r / a.groups;
  const float* part = a.parts_bc + (bt * a.tiles + g * a.group_tiles) * per + v;
  float s = 0.f;
#pragma unroll 4
  for (int64_t k = 0; k < a.group_tiles; ++k) s += part[k * per];
  const bool is_c = v >= a.padded;
  const int64_t n = is_c ? v - a.padded : v;
  if (n >= a.dstate) return;
  const TensorArg& t = is_c ? a.dC : a.dB;
  static_cast<T*>(t.data)[(bt / a.seqlen) * t.s0 + g * (is_c ? a.dC_group : a.dB_group) + n * t.s1 + (bt % a.seqlen) * t.s2] = from_f32<T>(s);
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
  const size_t smem = static_cast<size_t>(BwdSmem<T, LN>::bytes(a));
  const auto kernel = sel_bwd_kernel<T, LN, ROWS, MULTI, ENDS>;
  const cudaError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), smem);
  if (e != cudaSuccess) return e;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(a.batch * a.segments * a.tiles)), dim3(kSelThreads), smem, s, a);
}

template <typename T, int LN, bool ROWS, bool MULTI = false>
cudaError_t walk(const SelArgs& a, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  if (a.segments > 1) e = launch<T, LN, ROWS, MULTI, true>(a, s);
  return e == cudaSuccess ? launch<T, LN, ROWS, MULTI, false>(a, s) : e;
}
template <typename T>
cudaError_t walk(const SelArgs& a, cudaStream_t s) {
  if (a.blocks > 1) return a.rows ? walk<T, 4, true, true>(a, s) : walk<T, 4, false, true>(a, s);
  switch (a.lanes) {
    case 1: return a.rows ? walk<T, 1, true>(a, s) : walk<T, 1, false>(a, s);
    case 2: return a.rows ? walk<T, 2, true>(a, s) : walk<T, 2, false>(a, s);
    default: return a.rows ? walk<T, 4, true>(a, s) : walk<T, 4, false>(a, s);
  }
}

template <typename T>
cudaError_t run(const SelArgs& a, cudaStream_t s) {
  cudaError_t e = walk<T>(a, s);
  const int64_t bc = a.batch * a.seqlen * a.groups * 2 * a.padded, params = a.dim * (a.padded + 2);
  if (e == cudaSuccess)
    e = launch_dependent(sel_sum_bc_kernel<T>, dim3(static_cast<unsigned>((bc + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
  if (e == cudaSuccess)
    e = launch_dependent(sel_sum_params_kernel, dim3(static_cast<unsigned>((params + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, a);
  return e;
}

}  // namespace

cudaError_t CC1D_DT_NAME(sel_bwd)(const SelArgs& a, cudaStream_t s) { return run<CC1D_DT_TYPE>(a, s); }

}  // namespace cc1d
