// Attention of few query rows over many keys: one new token (or a few) per sequence, over a paged
// BF16 or E4M3 cache or over contiguous K/V.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m), s_j = scale log2(e) q.k_j, in one pass over
// the keys with a running maximum m.  Bound by the K/V bytes (every byte is used for at most 16
// rows), so the kernel is built around loads in flight: a CTA of 4 warps takes a tile of 16 rows of
// one (sequence, K/V head) and a share of its keys; each warp streams its own 16-key chunks through
// its own cp.async ring (no CTA barrier in the loop) and keeps its own m, l and O in registers; the
// warps merge at the end.  The products run on mma.sync m16n8k16: with 16 rows the tensor work is a
// few per cent of the time that the bytes take, and the fragments need no shared-memory round trip
// of S and P.  Long sequences are split over several CTAs (`unit` chunks each), whose partial
// results a second kernel joins in a fixed order.
//
// Keys that a row does not see have no influence whatever they hold: S is replaced by -inf, and a
// chunk with a non-finite V (where P = 0 times V would be NaN) goes through exact_pv, which adds
// only what each row sees.
#include "join.cuh"

namespace solattn {

namespace {

constexpr int kTileRows = 16;   // rows of a CTA
constexpr int kChunk = 16;      // keys of a chunk
constexpr int kWarps = 4;
constexpr int kRowThreads = kWarps * 32;

template <int D, int KV>
struct RowsCfg {
  static constexpr int kElt = KV == kPagedE4m3 ? 1 : 2;
  static constexpr int kRowB = D * kElt;          // bytes of a K or V row
  static constexpr int kCpr = kRowB / 16;         // 16-byte pieces of a row
  static constexpr int kPart = kChunk * kRowB;    // K or V of a chunk
  static constexpr int kStage = 2 * kPart + (KV == kPagedE4m3 ? 32 : 0);  // + 16 K and V scales
  // About 24 KB of ring per warp, so that two CTAs share an SM.
  static constexpr int kStages = 24576 / kStage > 8 ? 8 : 24576 / kStage;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kMerge = kWarps * kTileRows * (D + 2) * 4;  // m, l, O of every warp
  static constexpr int kSmem = kWarps * kRing > kMerge ? kWarps * kRing : kMerge;
};

// Shared-memory offsets of the 16-byte piece c of row r, chosen so that the reads below have no bank
// conflicts: K is read as 16 bytes by lane (row = lane / 4, piece = 4 i + lane % 4); BF16 V by
// ldmatrix (8 rows, one piece); E4M3 V as 4 bytes (rows 2 t, t = lane % 4; 32 bytes by lane / 4).
template <int D, int KV>
__device__ __forceinline__ uint32_t k_off(int r, int c) {
  using C = RowsCfg<D, KV>;
  return (uint32_t)(r * C::kRowB + ((C::kCpr >= 8 ? c ^ ((r & 1) << 2) : c) << 4));
}
template <int D, int KV>
__device__ __forceinline__ uint32_t v_off(int r, int c) {
  using C = RowsCfg<D, KV>;
  if (KV != kPagedE4m3) return (uint32_t)(r * C::kRowB + ((c ^ (r & 7)) << 4));
  if (D == 128) return (uint32_t)(r * C::kRowB + ((c ^ (((r >> 1) & 3) << 1)) << 4));
  const int phys = (r & 12) | ((r & 1) << 1) | ((r >> 1) & 1);
  return (uint32_t)(phys * C::kRowB + ((c ^ (((r >> 2) & 1) << 1)) << 4));
}

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a));
  return v;
}

// The head dim of column `col` (0 or 1) of this lane's pair in output tile nt (8 columns).  BF16: the
// tile's own.  E4M3: a lane's 4-byte read covers four tiles' columns, so that tile (4 j + i) holds the
// dims 32 j + 4 g + i, g = 0..7.
template <int KV>
__device__ __forceinline__ int out_dim(int nt, int t, int col) {
  return KV == kPagedE4m3 ? 32 * (nt >> 2) + 8 * t + 4 * col + (nt & 3) : 8 * nt + 2 * t + col;
}

template <int D, int KV>
__device__ __forceinline__ float v_at(uint32_t sv, int key, int d) {
  if (KV == kPagedE4m3) {
    const uint32_t w = lds32(sv + v_off<D, KV>(key, d >> 4) + (uint32_t)(d & 12));
    return e4m3_value((w >> (8 * (d & 3))) & 0xffu);
  }
  const uint32_t w = lds32(sv + v_off<D, KV>(key, d >> 3) + (uint32_t)(2 * (d & 6)));
  return __uint_as_float((d & 1) ? (w & 0xffff0000u) : (w << 16));
}

// O += P V of one chunk with a non-finite V, key by key and only where the row sees the key.
// `scales` is the chunk's 16 V exponents (E4M3).
template <int D, int KV>
__device__ __forceinline__ void exact_pv(float (&o)[D / 8][4], const float (&pr)[2][4],
                                         const bool (&vis)[2][4], uint32_t sv, uint32_t scales,
                                         int lane) {
  const int t = lane & 3;
#pragma unroll 1
  for (int key = 0; key < kChunk; ++key) {
    const int owner = (lane & ~3) | ((key & 7) >> 1);
    float p0 = 0.f, p1 = 0.f;
    bool s0 = false, s1 = false;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if ((key >> 3) == nt && (key & 1) == c) {
          p0 = pr[nt][c];
          p1 = pr[nt][2 + c];
          s0 = vis[nt][c];
          s1 = vis[nt][2 + c];
        }
    p0 = __shfl_sync(0xffffffffu, p0, owner);
    p1 = __shfl_sync(0xffffffffu, p1, owner);
    s0 = __shfl_sync(0xffffffffu, (int)s0, owner) != 0;
    s1 = __shfl_sync(0xffffffffu, (int)s1, owner) != 0;
    const float f =
        KV == kPagedE4m3 ? e8m0_value((lds32(scales + (key & 12)) >> (8 * (key & 3))) & 0xffu) : 1.f;
#pragma unroll
    for (int nt = 0; nt < D / 8; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float x = v_at<D, KV>(sv, key, out_dim<KV>(nt, t, c)) * f;
        if (s0) o[nt][c] += p0 * x;
        if (s1) o[nt][2 + c] += p1 * x;
      }
    }
  }
}

}  // namespace

template <int D, int KV>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(const SeqParams p) {
  using C = RowsCfg<D, KV>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = (int)(blockIdx.x % p.splits);
  const int h = (int)((blockIdx.x / p.splits) % p.Hkv);
  const int slot = (int)(blockIdx.x / ((unsigned)p.splits * p.Hkv));
  if (split == 0 && h == 0 && p.zero_tail) zero_tail<D>(p, slot, p.slots, tid, kRowThreads);
  const Seq sq = find_seq<kTileRows>(p, slot, lane);
  if (sq.b < 0 || !p.takes(sq.n)) return;
  const int rows = min(kTileRows, sq.n * p.G - sq.tile * kTileRows);
  const int r_base = sq.tile * kTileRows;  // first (token, head) row of the tile
  const int off = sq.L - sq.n;             // position of token 0
  const int pos0 = off + r_base / p.G, pos1 = off + (r_base + rows - 1) / p.G;
  const KeyTiles kt = key_tiles<kChunk>(p, sq.L, pos0, pos1);
  const int total = kt.count();
  const int ns = max(1, min(p.splits, (total + p.unit - 1) / p.unit));
  if (split >= ns) return;
  const int c0 = (int)((int64_t)total * split / ns), c1 = (int)((int64_t)total * (split + 1) / ns);
  const int mine = c1 - c0 > warp ? (c1 - c0 - warp + kWarps - 1) / kWarps : 0;  // this warp's chunks

  // Q fragments: the contraction order over the head dim is free, so lane t of a row group holds the
  // dims that its 16-byte K reads deliver: k-step ks takes 4 consecutive dims of piece 4 (ks / S) + t.
  constexpr int kS = C::kElt == 1 ? 4 : 2;  // k-steps of a 16-byte piece
  uint32_t qa[D / 16][4];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = g + 8 * half;
    const bool in = r < rows;
    const int tok = (r_base + (in ? r : 0)) / p.G, head = (r_base + (in ? r : 0)) % p.G;
    const __nv_bfloat16* src = p.q + (p.table ? (int64_t)(sq.start + tok) * p.q_sT
                                              : (int64_t)sq.b * p.q_sB + (int64_t)tok * p.q_sT) +
                               (int64_t)(h * p.G + head) * p.q_sH;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      const int d = (16 / C::kElt) * (4 * (ks / kS) + t) + 4 * (ks % kS);
      const uint2 w = in ? __ldg(reinterpret_cast<const uint2*>(src + d)) : make_uint2(0u, 0u);
      qa[ks][half] = w.x;
      qa[ks][2 + half] = w.y;
    }
  }
  int hi[2], lo[2];  // what rows g and g + 8 see
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = g + 8 * half;
    const int pos = off + (r_base + r) / p.G;
    hi[half] = r < rows ? key_high(p, sq.L, pos) : -1;
    lo[half] = key_low(p, pos);
  }
  const int all_hi = key_high(p, sq.L, pos0), all_lo = key_low(p, pos1);  // what every row sees

  // This lane's page of every 32nd chunk of the warp, fetched ahead of the loop.
  int my_page = 0;
  auto fetch_pages = [&](int i0) {
    const int i = i0 + lane;
    if (KV != kStrided && i < mine) my_page = page_of(p, sq.b, kChunk * kt.at(c0 + warp + i * kWarps));
  };
  const uint32_t ring = smem_u32(smem) + (uint32_t)(warp * C::kRing);
  auto load = [&](int i) {
    const int key0 = kChunk * kt.at(c0 + warp + i * kWarps);
    const uint32_t st = ring + (uint32_t)((i % C::kStages) * C::kStage);
    int64_t ko, vo, kstep, vstep;  // byte offsets of the chunk's first row, and of a row
    int64_t row0 = 0;
    if (KV == kStrided) {
      ko = ((int64_t)sq.b * p.k_sB + (int64_t)key0 * p.k_sT + (int64_t)h * p.k_sH) * 2;
      vo = ((int64_t)sq.b * p.v_sB + (int64_t)key0 * p.v_sT + (int64_t)h * p.v_sH) * 2;
      kstep = p.k_sT * 2;
      vstep = p.v_sT * 2;
    } else {
      const int page = __shfl_sync(0xffffffffu, my_page, i & 31);
      row0 = (((int64_t)page * p.Hkv + h) << p.page_shift) + (key0 & ((1 << p.page_shift) - 1));
      ko = vo = row0 * C::kRowB;
      kstep = vstep = C::kRowB;
    }
#pragma unroll
    for (int j = 0; j < C::kPart / 512; ++j) {
      const int r = j * (32 / C::kCpr) + lane / C::kCpr, c = lane % C::kCpr;
      const bool in = key0 + r < sq.L;  // rows behind the last key: zeros, nothing is read
      const int64_t rr = in ? r : 0;
      cp_async16(st + k_off<D, KV>(r, c), p.k + ko + rr * kstep + 16 * c, in ? 16 : 0);
      cp_async16(st + C::kPart + v_off<D, KV>(r, c), p.v + vo + rr * vstep + 16 * c, in ? 16 : 0);
    }
    if (KV == kPagedE4m3 && lane < 2)
      cp_async16(st + 2 * C::kPart + 16 * lane, (lane ? p.v_scale : p.k_scale) + row0, 16);
  };

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  fetch_pages(0);
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) {
    if (i < mine) load(i);
    cp_async_commit();
  }
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    cp_async_wait<C::kStages - 2>();
    __syncwarp();  // every lane's pieces of chunk i have landed, and chunk i - 1 has been read
    const int ahead = i + C::kStages - 1;
    if (ahead < mine) {
      if ((ahead & 31) == 0) fetch_pages(ahead);
      load(ahead);
    }
    cp_async_commit();
    const int key0 = kChunk * kt.at(c0 + warp + i * kWarps);
    const uint32_t st = ring + (uint32_t)((i % C::kStages) * C::kStage);
    const uint32_t sv = st + C::kPart;

    // ---- S = Q K^T: 16 rows, two tiles of 8 keys
    float s[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    uint32_t k_nan = 0u;  // E4M3: a NaN code in this lane's part of key g (bit 0) or g + 8 (bit 1)
#pragma unroll
    for (int hh = 0; hh < C::kCpr / 4; ++hh) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const uint4 w4 = lds128(st + k_off<D, KV>(8 * nt + g, 4 * hh + t));
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        if (KV == kPagedE4m3) {
          uint32_t bad = 0u;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            bad |= e4m3_nan_bytes(w[x]);
            const uint32_t b0 = bf16x2_mul(e4m3_fields(__byte_perm(w[x], 0u, 0x1404)), kTwo120x2);
            const uint32_t b1 = bf16x2_mul(e4m3_fields(__byte_perm(w[x], 0u, 0x3424)), kTwo120x2);
            mma_bf16_16816(s[nt], qa[4 * hh + x], b0, b1);
          }
          if (bad) k_nan |= 1u << nt;
        } else {
          mma_bf16_16816(s[nt], qa[2 * hh], w[0], w[1]);
          mma_bf16_16816(s[nt], qa[2 * hh + 1], w[2], w[3]);
        }
      }
    }
    float vs[2][2];  // V scales of this lane's keys 8 nt + 2 t + c
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      if (KV == kPagedE4m3) {
        const uint32_t kw = lds32(st + 2 * C::kPart + 8 * nt + 4 * (t >> 1)) >> (16 * (t & 1));
        const uint32_t vw = lds32(st + 2 * C::kPart + 16 + 8 * nt + 4 * (t >> 1)) >> (16 * (t & 1));
        const float k0 = e8m0_value(kw & 0xffu) * p.scale_log2;
        const float k1 = e8m0_value((kw >> 8) & 0xffu) * p.scale_log2;
        s[nt][0] *= k0;
        s[nt][1] *= k1;
        s[nt][2] *= k0;
        s[nt][3] *= k1;
        vs[nt][0] = e8m0_value(vw & 0xffu);
        vs[nt][1] = e8m0_value((vw >> 8) & 0xffu);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) s[nt][c] *= p.scale_log2;
        vs[nt][0] = vs[nt][1] = 1.f;
      }
    }
    if (KV == kPagedE4m3 && __any_sync(0xffffffffu, k_nan != 0u)) {
      k_nan |= __shfl_xor_sync(0xffffffffu, k_nan, 1);
      k_nan |= __shfl_xor_sync(0xffffffffu, k_nan, 2);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const uint32_t f = __shfl_sync(0xffffffffu, k_nan, 4 * (2 * t + c));  // flags of keys 2 t + c
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
          if ((f >> nt) & 1u) s[nt][c] = s[nt][2 + c] = __uint_as_float(0x7fc00000u);
      }
    }
    // ---- visibility
    bool vis[2][4];
    const bool full = key0 + kChunk - 1 <= all_hi && (key0 >= all_lo || key0 + kChunk <= p.sinks);
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) vis[nt][c] = true;
    if (!full) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int key = key0 + 8 * nt + 2 * t + (c & 1), half = c >> 1;
          vis[nt][c] = key <= hi[half] && (key >= lo[half] || key < p.sinks);
          if (!vis[nt][c]) s[nt][c] = -INFINITY;
        }
    }
    // ---- online softmax.  The running maximum moves only when it grows by more than 8 (a factor
    // 256), so that O is rarely rescaled; P stays at most 256.
    float mt[2], al[2] = {1.f, 1.f};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x = fmaxf(fmaxf(s[0][2 * half], s[0][2 * half + 1]), fmaxf(s[1][2 * half], s[1][2 * half + 1]));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      mt[half] = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
    }
    bool need = false;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      if (m[half] == -INFINITY) {
        m[half] = fmaxf(m[half], mt[half]);  // nothing accumulated yet
      } else if (mt[half] > m[half] + 8.f) {
        al[half] = fast_exp2(m[half] - mt[half]);
        m[half] = mt[half];
        need = true;
      }
    }
    if (__any_sync(0xffffffffu, need)) {
#pragma unroll
      for (int x = 0; x < D / 8; ++x) {
        o[x][0] *= al[0];
        o[x][1] *= al[0];
        o[x][2] *= al[1];
        o[x][3] *= al[1];
      }
      l[0] *= al[0];
      l[1] *= al[1];
    }
    float pr[2][4];
    bool scale_nan = false;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float mm = m[c >> 1] == -INFINITY ? 0.f : m[c >> 1];
        pr[nt][c] = fast_exp2(s[nt][c] - mm);
        l[c >> 1] += pr[nt][c];
        scale_nan = scale_nan || vs[nt][c & 1] != vs[nt][c & 1];
      }
    // P as the A operand: rounded to BF16 (relative error at most 2^-9 each; l keeps FP32), E4M3 with
    // V's power-of-two scale folded in, which rounds the same.
    uint32_t pa[4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      pa[2 * nt] = pack_bf16(pr[nt][0] * vs[nt][0], pr[nt][1] * vs[nt][1]);
      pa[2 * nt + 1] = pack_bf16(pr[nt][2] * vs[nt][0], pr[nt][3] * vs[nt][1]);
    }
    // ---- O += P V
    uint32_t vb[D / 8][2];
    bool bad = false;
    if (KV == kPagedE4m3) {
      uint32_t acc = 0u;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        uint32_t w[4];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9; dims 32 j + 4 g..
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int key = 2 * t + (x & 1) + 8 * (x >> 1);
          w[x] = lds32(sv + v_off<D, KV>(key, 2 * j + (g >> 2)) + (uint32_t)(4 * (g & 3)));
          acc |= e4m3_nan_bytes(w[x]);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          // Byte x of two keys' words into the high bytes of a pair; the fields mask drops the rest.
          const uint32_t sel = (uint32_t)(x << 4) | (uint32_t)((4 + x) << 12);
          vb[4 * j + x][0] = bf16x2_mul(e4m3_fields(__byte_perm(w[0], w[1], sel)), kTwo120x2);
          vb[4 * j + x][1] = bf16x2_mul(e4m3_fields(__byte_perm(w[2], w[3], sel)), kTwo120x2);
        }
      }
      bad = acc != 0u || scale_nan;
    } else {
      uint32_t acc = 0u;  // V * 0 summed: NaN where a V is not finite
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        ldsm_x4_t(sv + v_off<D, KV>(lane & 15, 2 * dt + (lane >> 4)), vb[2 * dt][0], vb[2 * dt][1],
                  vb[2 * dt + 1][0], vb[2 * dt + 1][1]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          acc = bf16x2_fma(vb[2 * dt + x][0], 0u, acc);
          acc = bf16x2_fma(vb[2 * dt + x][1], 0u, acc);
        }
      }
      bad = (acc & 0x7fff7fffu) != 0u;
    }
    if (__any_sync(0xffffffffu, bad)) {
      exact_pv<D, KV>(o, pr, vis, sv, st + 2 * C::kPart + 16, lane);
    } else {
#pragma unroll
      for (int nt = 0; nt < D / 8; ++nt) mma_bf16_16816(o[nt], pa, vb[nt][0], vb[nt][1]);
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- the warps' results through shared memory (over the rings, which are drained)
  float* sO = reinterpret_cast<float*>(smem);                       // [warp][row][D]
  float* sM = sO + kWarps * kTileRows * D;                          // [warp][row][2]
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
    const int r = g + 8 * half;
    if (r < rows) {
      float* dst = sO + (warp * kTileRows + r) * D;
#pragma unroll
      for (int nt = 0; nt < D / 8; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) dst[out_dim<KV>(nt, t, c)] = o[nt][2 * half + c];
      if (t == 0) {
        sM[(warp * kTileRows + r) * 2] = m[half];
        sM[(warp * kTileRows + r) * 2 + 1] = l[half];
      }
    }
  }
  __syncthreads();
  const int64_t unit = ((int64_t)slot * p.Hkv + h) * p.splits + split;
  for (int i = tid; i < rows * (D / 4); i += kRowThreads) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sM[(w * kTileRows + r) * 2]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = fast_exp2(sM[(w * kTileRows + r) * 2] - base);
      sum += sM[(w * kTileRows + r) * 2 + 1] * f;
      const float4 x = *reinterpret_cast<const float4*>(sO + (w * kTileRows + r) * D + d);
      a.x += x.x * f;
      a.y += x.y * f;
      a.z += x.z * f;
      a.w += x.w * f;
    }
    if (ns > 1) {
      *reinterpret_cast<float4*>(p.part + (unit * kTileRows + r) * D + d) = a;
      if (d == 0) {
        float* ml = p.part + (int64_t)p.slots * p.Hkv * p.splits * kTileRows * D + (unit * kTileRows + r) * 2;
        ml[0] = mx;
        ml[1] = sum;
      }
    } else {
      const int tok = (r_base + r) / p.G, head = (r_base + r) % p.G, pos = off + tok;
      // A row that sees no key gives zeros.
      const int high = key_high(p, sq.L, pos);
      const bool any = high >= 0 && (high >= key_low(p, pos) || p.sinks > 0);
      const float inv = any ? 1.f / sum : 0.f;
      uint2 w;
      w.x = any ? pack_bf16(a.x * inv, a.y * inv) : 0u;
      w.y = any ? pack_bf16(a.z * inv, a.w * inv) : 0u;
      *reinterpret_cast<uint2*>(p.out + ((int64_t)(sq.start + tok) * p.Hq + h * p.G + head) * D + d) = w;
    }
  }
}

namespace {

template <int D, int KV>
cudaError_t launch_rows_kv(const SeqParams& p, cudaStream_t stream) {
  constexpr int smem = RowsCfg<D, KV>::kSmem;
  static_assert(smem <= 113 * 1024, "two CTAs share an SM");
  cudaError_t err = cudaFuncSetAttribute(rows_kernel<D, KV>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (err != cudaSuccess) return err;
  const int64_t ctas = (int64_t)p.slots * p.Hkv * p.splits;
  rows_kernel<D, KV><<<(unsigned)ctas, kRowThreads, smem, stream>>>(p);
  err = cudaGetLastError();
  if (err != cudaSuccess || p.splits == 1) return err;
  join_kernel<D, kTileRows, kChunk><<<(unsigned)((int64_t)p.slots * p.Hkv), kJoinThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_rows(const SeqParams& p, int D, int kv, cudaStream_t stream) {
  if (D == 128) {
    if (kv == kStrided) return launch_rows_kv<128, kStrided>(p, stream);
    if (kv == kPagedBf16) return launch_rows_kv<128, kPagedBf16>(p, stream);
    return launch_rows_kv<128, kPagedE4m3>(p, stream);
  }
  if (kv == kStrided) return launch_rows_kv<64, kStrided>(p, stream);
  if (kv == kPagedBf16) return launch_rows_kv<64, kPagedBf16>(p, stream);
  return launch_rows_kv<64, kPagedE4m3>(p, stream);
}

}  // namespace solattn
