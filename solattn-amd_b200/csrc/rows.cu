// Attention of few query rows over many keys: one new token (or a few) per sequence, over a paged
// BF16 or E4M3 cache or over contiguous K/V.
//
// o = sum_j p_j v_j / sum_j p_j with p_j = 2^(s_j - m), s_j = scale log2(e) q.k_j, in one pass over
// the keys with a running maximum m.  Bound by the K/V bytes (every byte is used for at most 16
// rows), so the kernel is built around loads in flight: a CTA of 4 warps takes a tile of 8 or 16 rows
// of one (sequence, K/V head) and a share of its keys; each warp streams its own chunks of 16 or 32 keys through
// its own cp.async ring (no CTA barrier in the loop) and keeps its own m, l and O in registers; the
// warps merge at the end.  The products run on mma.sync m16n8k16: with so few rows the tensor work is a
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

constexpr int kWarps = 4;
constexpr float kTwo60 = 1152921504606846976.f, kTwoM60 = 1.f / kTwo60;
constexpr int kRowThreads = kWarps * 32;

// R rows of a tile: 8 or 16 (of the 16 rows of an MMA).  A chunk has 16 keys per MMA step, two steps
// where a step is small, so that what a chunk costs besides its bytes is spread over more of them.
template <int D, int KV, int R>
struct RowsCfg {
  static constexpr int kElt = KV == kPagedE4m3 ? 1 : 2;
  static constexpr int kRowB = D * kElt;          // bytes of a K or V row
  static constexpr int kSteps = D == 64 ? 2 : 1;
  static constexpr int kChunk = 16 * kSteps;      // keys of a chunk
  static constexpr int kCpr = kRowB / 16;         // 16-byte pieces of a row
  static constexpr int kPart = kChunk * kRowB;    // K or V of a chunk
  static constexpr int kStage = 2 * kPart + (KV == kPagedE4m3 ? 2 * kChunk : 0);  // + K and V scales
  // BF16: 24 KB of ring per warp and two CTAs per SM (the bytes in flight are what counts); E4M3, which
  // also has codes to convert: three or four CTAs, as many as the registers allow.
  static constexpr int kStages = KV == kPagedE4m3 && D == 128 ? 4 : 3;
  static constexpr int kCtas = KV != kPagedE4m3 ? 2 : D == 64 ? 4 : 3;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kMerge = kWarps * R * (D + 2) * 4;  // m, l, O of every warp
  static constexpr int kSmem = kWarps * kRing > kMerge ? kWarps * kRing : kMerge;
  static constexpr int kHalves = R / 8;  // row groups g and g + 8 of the MMA
};

// Shared-memory offsets of the 16-byte piece c of row r, chosen so that the reads below have no bank
// conflicts: K is read as 16 bytes by lane (row = lane / 4, piece = 4 i + lane % 4); BF16 V by
// ldmatrix (8 rows, one piece); E4M3 V as 4 bytes (rows 2 t, t = lane % 4; 32 bytes by lane / 4).
template <int D, int KV>
__device__ __forceinline__ uint32_t k_off(int r, int c) {
  constexpr int kRowB = KV == kPagedE4m3 ? D : 2 * D;
  return (uint32_t)(r * kRowB + ((kRowB >= 128 ? c ^ ((r & 1) << 2) : c) << 4));
}
template <int D, int KV>
__device__ __forceinline__ uint32_t v_off(int r, int c) {
  constexpr int kRowB = KV == kPagedE4m3 ? D : 2 * D;
  if (KV != kPagedE4m3) return (uint32_t)(r * kRowB + ((c ^ (r & 7)) << 4));
  if (D == 128) return (uint32_t)(r * kRowB + ((c ^ (((r >> 1) & 3) << 1)) << 4));
  const int phys = (r & ~3) | ((r & 1) << 1) | ((r >> 1) & 1);
  return (uint32_t)(phys * kRowB + ((c ^ (((r >> 2) & 1) << 1)) << 4));
}

__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a));
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

// E4M3 codes 2 x and 2 x + 1 of a word as FP16, exactly (NaN stays NaN).
__device__ __forceinline__ uint32_t codes_to_f16(uint32_t w, int x) {
  uint32_t d;
  const uint16_t two = (uint16_t)(x ? w >> 16 : w);
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"(two));
  return d;
}

// D = A(16x16 FP16, row) * B(16x8 FP16, col) + D, FP32 accumulate.
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Whether a pair of code fields (see e4m3_fields; signs cleared) is at E4M3's NaN: the largest pair so
// far is kept, one instruction for two pairs.
__device__ __forceinline__ bool nan_fields(uint32_t top) { return (top >> 16) == 0x7f0u || (top & 0xffffu) == 0x7f0u; }

// O += P V of one chunk with a non-finite V, key by key and only where the row sees the key.
// `scales` is the chunk's V exponents (E4M3).
template <int D, int KV, int R>
__device__ __forceinline__ void exact_pv(float (&o)[D / 8][4], const float (&pr)[2 * RowsCfg<D, KV, R>::kSteps][4],
                                         const bool (&vis)[2 * RowsCfg<D, KV, R>::kSteps][4], uint32_t sv,
                                         uint32_t scales, int lane) {
  const int t = lane & 3;
#pragma unroll 1
  for (int key = 0; key < RowsCfg<D, KV, R>::kChunk; ++key) {
    const int owner = (lane & ~3) | ((key & 7) >> 1);
    float p0 = 0.f, p1 = 0.f;
    bool s0 = false, s1 = false;
#pragma unroll
    for (int nt = 0; nt < 2 * RowsCfg<D, KV, R>::kSteps; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        if ((key >> 3) == nt && (key & 1) == c) {
          p0 = pr[nt][c];
          s0 = vis[nt][c];
          if (R == 16) {
            p1 = pr[nt][2 + c];
            s1 = vis[nt][2 + c];
          }
        }
    p0 = __shfl_sync(0xffffffffu, p0, owner);
    s0 = __shfl_sync(0xffffffffu, (int)s0, owner) != 0;
    if (R == 16) {
      p1 = __shfl_sync(0xffffffffu, p1, owner);
      s1 = __shfl_sync(0xffffffffu, (int)s1, owner) != 0;
    }
    const float f = KV == kPagedE4m3 ? e8m0_value(lds8(scales + key)) * kTwoM60 : 1.f;
#pragma unroll
    for (int nt = 0; nt < D / 8; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float x = v_at<D, KV>(sv, key, out_dim<KV>(nt, t, c)) * f;  // (O holds 2^-60 of it, E4M3)
        if (s0) o[nt][c] += p0 * x;
        if (s1) o[nt][2 + c] += p1 * x;
      }
    }
  }
}

}  // namespace

template <int D, int KV, int R>
__global__ void __launch_bounds__(kRowThreads, RowsCfg<D, KV, R>::kCtas) rows_kernel(const SeqParams p) {
  using C = RowsCfg<D, KV, R>;
  constexpr int kNt = 2 * C::kSteps;  // 8-key columns of a chunk
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int split = (int)(blockIdx.x % p.splits);
  const int h = (int)((blockIdx.x / p.splits) % p.Hkv);
  const int slot = (int)(blockIdx.x / ((unsigned)p.splits * p.Hkv));
  if (split == 0 && h == 0 && p.zero_tail) zero_tail<D>(p, slot, p.slots, tid, kRowThreads);
  const Seq sq = find_seq<R>(p, slot, lane);
  if (sq.b < 0 || !p.takes(sq.n)) return;
  const int rows = min(R, sq.n * p.G - sq.tile * R);
  const int r_base = sq.tile * R;  // first (token, head) row of the tile
  const int off = sq.L - sq.n;     // position of token 0
  const int pos0 = off + r_base / p.G, pos1 = off + (r_base + rows - 1) / p.G;
  const KeyTiles kt = key_tiles<C::kChunk>(p, sq.L, pos0, pos1);
  const int total = kt.count();
  const int ns = max(1, min(p.splits, (total + p.unit - 1) / p.unit));
  if (split >= ns) return;
  const int c0 = (int)((int64_t)total * split / ns), c1 = (int)((int64_t)total * (split + 1) / ns);
  const int mine = c1 - c0 > warp ? (c1 - c0 - warp + kWarps - 1) / kWarps : 0;  // this warp's chunks
  // Keys that some row sees: [low, high] and those below the sinks.
  const int low = key_low(p, pos0), high = key_high(p, sq.L, pos1);

  // This lane's page of the warp's chunks, a page of every 16 keys, fetched ahead of the loop: lane l has
  // that of 16-key step l % steps of chunk i0 + l / steps.  -1: nobody sees it, so it is not loaded,
  // whatever the page table says.
  constexpr int kAhead = 32 / C::kSteps;  // chunks that a fetch covers
  int my_page = 0;
  auto fetch_pages = [&](int i0) {
    const int i = i0 + lane / C::kSteps;
    if (KV == kStrided || i >= mine) return;
    const int key = C::kChunk * kt.at(c0 + warp + i * kWarps) + 16 * (lane % C::kSteps);
    my_page = key > high || (key + 16 <= low && key >= p.sinks) ? -1 : page_of(p, sq.b, key);
  };
  const uint32_t ring = smem_u32(smem) + (uint32_t)(warp * C::kRing);
  constexpr int kPass = 32 / C::kCpr;  // rows of a warp instruction
  const int lr = lane / C::kCpr, lc = lane % C::kCpr;
  auto load = [&](int i) {
    const int key0 = C::kChunk * kt.at(c0 + warp + i * kWarps);
    const uint32_t st = ring + (uint32_t)((i % C::kStages) * C::kStage);
    // Pieces of each 16-key step; rows behind the last key, and steps that nobody sees, become zeros
    // without a read.
#pragma unroll
    for (int u = 0; u < C::kSteps; ++u) {
      const int key = key0 + 16 * u;
      int page = 0;
      if (KV != kStrided) page = __shfl_sync(0xffffffffu, my_page, (i % kAhead) * C::kSteps + u);
      const int valid = page < 0 ? 0 : min(16, sq.L - key);
      const uint8_t *kp, *vp;
      int64_t kstep = C::kRowB, vstep = C::kRowB, row0 = 0;
      if (KV == kStrided) {
        kp = p.k + ((int64_t)sq.b * p.k_sB + (int64_t)key * p.k_sT + (int64_t)h * p.k_sH) * 2;
        vp = p.v + ((int64_t)sq.b * p.v_sB + (int64_t)key * p.v_sT + (int64_t)h * p.v_sH) * 2;
        kstep = p.k_sT * 2;
        vstep = p.v_sT * 2;
      } else {
        row0 = (((int64_t)max(page, 0) * p.Hkv + h) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
        kp = p.k + row0 * C::kRowB;
        vp = p.v + row0 * C::kRowB;
      }
      kp += lr * kstep + 16 * lc;
      vp += lr * vstep + 16 * lc;
      const uint32_t dk = st + k_off<D, KV>(16 * u + lr, lc), dv = st + C::kPart;
      if (valid == 16) {
#pragma unroll
        for (int j = 0; j < 16 / kPass; ++j) {
          // (k_off only looks at r mod 2, which a pass keeps.)
          cp_async16(dk + (uint32_t)(j * kPass * C::kRowB), kp + j * kPass * kstep, 16);
          cp_async16(dv + v_off<D, KV>(16 * u + j * kPass + lr, lc), vp + j * kPass * vstep, 16);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 16 / kPass; ++j) {
          const bool in = j * kPass + lr < valid;
          cp_async16(dk + (uint32_t)(j * kPass * C::kRowB), in ? kp + j * kPass * kstep : p.k, in ? 16 : 0);
          cp_async16(dv + v_off<D, KV>(16 * u + j * kPass + lr, lc), in ? vp + j * kPass * vstep : p.v, in ? 16 : 0);
        }
      }
      if (KV == kPagedE4m3 && lane < 2)
        cp_async16(st + 2 * C::kPart + C::kChunk * lane + 16 * u, (lane ? p.v_scale : p.k_scale) + row0, 16);
    }
  };
  fetch_pages(0);
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) {
    if (i < mine) load(i);
    cp_async_commit();
  }

  // Q fragments: the contraction order over the head dim is free, so lane t of a row group holds the
  // dims that its 16-byte K reads deliver: k-step ks takes 4 consecutive dims of piece 4 (ks / S) + t.
  // E4M3: S on FP16, in which codes are exact and cheap to make.  A row of Q is scaled by a power of two
  // that puts its largest value below 2^15; BF16's 8 significant bits fit in FP16's 11, and what falls
  // below FP16's range is 2^-39 of that value.
  constexpr int kS = C::kElt == 1 ? 4 : 2;  // k-steps of a 16-byte piece
  uint32_t qa[D / 16][4];
  int hi[C::kHalves], lo[C::kHalves];  // what rows g and g + 8 see
  float qf[C::kHalves];                // S in log2 units = qf * (Q K^T)
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
      uint2 w = make_uint2(0u, 0u);
      if (half < C::kHalves && in) w = __ldg(reinterpret_cast<const uint2*>(src + d));
      qa[ks][half] = w.x;
      qa[ks][2 + half] = w.y;
    }
    if (half < C::kHalves) {
      qf[half] = p.scale_log2;
      if (KV == kPagedE4m3) {
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t w = qa[ks][2 * x + half];
            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w << 16)), fabsf(__uint_as_float(w & 0xffff0000u))));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // top < 2^(e + 1): Q * 2^(14 - e) < 2^15.
        const int e = min(127, max(-100, (int)(__float_as_uint(top) >> 23) - 127));
        const float f = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
        qf[half] *= __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint32_t w = qa[ks][2 * x + half];
            const __half2 y = __floats2half2_rn(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xffff0000u) * f);
            qa[ks][2 * x + half] = *reinterpret_cast<const uint32_t*>(&y);
          }
      }
      const int pos = off + (r_base + r) / p.G;
      hi[half] = in ? key_high(p, sq.L, pos) : -1;
      lo[half] = key_low(p, pos);
    }
  }
  const int all_hi = key_high(p, sq.L, pos0), all_lo = key_low(p, pos1);  // what every row sees

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[C::kHalves], l[C::kHalves];
#pragma unroll
  for (int half = 0; half < C::kHalves; ++half) {
    m[half] = -INFINITY;
    l[half] = 0.f;
  }

#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    cp_async_wait<C::kStages - 2>();
    __syncwarp();  // every lane's pieces of chunk i have landed, and chunk i - 1 has been read
    const int ahead = i + C::kStages - 1;
    if (ahead < mine) {
      if (ahead % kAhead == 0) fetch_pages(ahead);
      load(ahead);
    }
    cp_async_commit();
    const int key0 = C::kChunk * kt.at(c0 + warp + i * kWarps);
    const uint32_t st = ring + (uint32_t)((i % C::kStages) * C::kStage);
    const uint32_t sv = st + C::kPart;

    // ---- S = Q K^T: 16 rows, tiles of 8 keys
    float s[kNt][4];
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int hh = 0; hh < C::kCpr / 4; ++hh) {
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) {
        const uint4 w4 = lds128(st + k_off<D, KV>(8 * nt + g, 4 * hh + t));
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        if (KV == kPagedE4m3) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            mma_f16_16816(s[nt], qa[4 * hh + x], codes_to_f16(w[x], 0), codes_to_f16(w[x], 1));
        } else {
          mma_bf16_16816(s[nt], qa[2 * hh], w[0], w[1]);
          mma_bf16_16816(s[nt], qa[2 * hh + 1], w[2], w[3]);
        }
      }
    }
    // Scales: lane l converts those of key l, then each lane takes its columns' (keys 8 nt + 2 t + c).
    float vs[kNt][2];
    bool odd_scale = false;
    if (KV == kPagedE4m3) {
      const int key = lane & (C::kChunk - 1);
      const float ks_l = e8m0_value(lds8(st + 2 * C::kPart + key));
      const float vs_l = e8m0_value(lds8(st + 2 * C::kPart + C::kChunk + key));
      odd_scale = !(vs_l < kTwo60 / 2);  // (or one that P cannot take, see below)
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float f = __shfl_sync(0xffffffffu, ks_l, 8 * nt + 2 * t + c);
          vs[nt][c] = __shfl_sync(0xffffffffu, vs_l, 8 * nt + 2 * t + c);
#pragma unroll
          for (int half = 0; half < C::kHalves; ++half) s[nt][2 * half + c] *= f;
        }
    } else {
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt) vs[nt][0] = vs[nt][1] = 1.f;
    }
    // ---- visibility
    bool vis[kNt][4];
    const bool full = key0 + C::kChunk - 1 <= all_hi && (key0 >= all_lo || key0 + C::kChunk <= p.sinks);
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) vis[nt][c] = true;
    if (!full) {
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
        for (int c = 0; c < 2 * C::kHalves; ++c) {
          const int key = key0 + 8 * nt + 2 * t + (c & 1), half = c >> 1;
          vis[nt][c] = key <= hi[half] && (key >= lo[half] || key < p.sinks);
          if (!vis[nt][c]) s[nt][c] = -INFINITY;
        }
    }
    // ---- online softmax.  The running maximum moves only when it grows by more than 8 (a factor
    // 256), so that O is rarely rescaled; P stays at most 256.
    float al[2] = {1.f, 1.f};
    bool need = false;
#pragma unroll
    for (int half = 0; half < C::kHalves; ++half) {
      float x = fmaxf(s[0][2 * half], s[0][2 * half + 1]);
#pragma unroll
      for (int nt = 1; nt < kNt; ++nt) x = fmaxf(x, fmaxf(s[nt][2 * half], s[nt][2 * half + 1]));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2)) * qf[half];
      if (m[half] == -INFINITY) {
        m[half] = fmaxf(m[half], x);  // nothing accumulated yet
      } else if (x > m[half] + 8.f) {
        al[half] = fast_exp2(m[half] - x);
        m[half] = x;
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
#pragma unroll
      for (int half = 0; half < C::kHalves; ++half) l[half] *= al[half];
    }
    float pr[kNt][4];
#pragma unroll
    for (int half = 0; half < C::kHalves; ++half) {
      const float mm = m[half] == -INFINITY ? 0.f : m[half];
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          pr[nt][2 * half + c] = fast_exp2(fmaf(s[nt][2 * half + c], qf[half], -mm));
          l[half] += pr[nt][2 * half + c];
        }
    }
    // P as the A operand: rounded to BF16 (relative error at most 2^-8 each; l keeps FP32), E4M3 with
    // V's power-of-two scale folded in, which rounds the same, and 2^60 of the 2^120 that V's code
    // fields lack (O takes the rest at the end; the products then lie well inside FP32's range).
    uint32_t pa[C::kSteps][4];
    if (KV == kPagedE4m3) {
#pragma unroll
      for (int nt = 0; nt < kNt; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) vs[nt][c] *= kTwo60;
    }
#pragma unroll
    for (int nt = 0; nt < kNt; ++nt) {
      pa[nt >> 1][2 * (nt & 1)] = pack_bf16(pr[nt][0] * vs[nt][0], pr[nt][1] * vs[nt][1]);
      pa[nt >> 1][2 * (nt & 1) + 1] =
          R == 16 ? pack_bf16(pr[nt][2] * vs[nt][0], pr[nt][3] * vs[nt][1]) : 0u;
    }
    // ---- O += P V, once V is known to be finite
    uint32_t vb[C::kSteps][D / 8][2];
    bool bad = false;
    if (KV == kPagedE4m3) {
      uint32_t top = 0u;
#pragma unroll
      for (int u = 0; u < C::kSteps; ++u)
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          uint32_t w[4];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of the step; dims 32 j + 4 g..
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int key = 16 * u + 2 * t + (x & 1) + 8 * (x >> 1);
            w[x] = lds32(sv + v_off<D, KV>(key, 2 * j + (g >> 2)) + (uint32_t)(4 * (g & 3)));
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            // Byte x of two keys' words into the high bytes of a pair; the fields mask drops the rest.
            const uint32_t sel = (uint32_t)(x << 4) | (uint32_t)((4 + x) << 12);
            const uint32_t a = __byte_perm(w[0], w[1], sel), b = __byte_perm(w[2], w[3], sel);
            const uint32_t fa = (a >> 4) & 0x07f007f0u, fb = (b >> 4) & 0x07f007f0u;
            top = __vimax3_u16x2(top, fa, fb);
            vb[u][4 * j + x][0] = fa | (a & 0x80008000u);
            vb[u][4 * j + x][1] = fb | (b & 0x80008000u);
          }
        }
      bad = nan_fields(top) || odd_scale;
    } else {
      uint32_t acc = 0u;  // V * 0 summed: NaN where a V is not finite
#pragma unroll
      for (int u = 0; u < C::kSteps; ++u)
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          ldsm_x4_t(sv + v_off<D, KV>(16 * u + (lane & 15), 2 * dt + (lane >> 4)), vb[u][2 * dt][0],
                    vb[u][2 * dt][1], vb[u][2 * dt + 1][0], vb[u][2 * dt + 1][1]);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            acc = bf16x2_fma(vb[u][2 * dt + x][0], 0u, acc);
            acc = bf16x2_fma(vb[u][2 * dt + x][1], 0u, acc);
          }
        }
      bad = (acc & 0x7fff7fffu) != 0u;
    }
    if (__any_sync(0xffffffffu, bad)) {
      exact_pv<D, KV, R>(o, pr, vis, sv, st + 2 * C::kPart + C::kChunk, lane);
    } else {
#pragma unroll
      for (int u = 0; u < C::kSteps; ++u)
#pragma unroll
        for (int nt = 0; nt < D / 8; ++nt) mma_bf16_16816(o[nt], pa[u], vb[u][nt][0], vb[u][nt][1]);
    }
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- the warps' results through shared memory (over the rings, which are drained)
  float* sO = reinterpret_cast<float*>(smem);  // [warp][row][D]
  float* sM = sO + kWarps * R * D;             // [warp][row][2]
#pragma unroll
  for (int half = 0; half < C::kHalves; ++half) {
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
    const int r = g + 8 * half;
    if (r < rows) {
      float* dst = sO + (warp * R + r) * D;
#pragma unroll
      for (int nt = 0; nt < D / 8; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          dst[out_dim<KV>(nt, t, c)] = KV == kPagedE4m3 ? o[nt][2 * half + c] * kTwo60 : o[nt][2 * half + c];
      if (t == 0) {
        sM[(warp * R + r) * 2] = m[half];
        sM[(warp * R + r) * 2 + 1] = l[half];
      }
    }
  }
  __syncthreads();
  const int64_t unit = ((int64_t)slot * p.Hkv + h) * p.splits + split;
  for (int i = tid; i < rows * (D / 4); i += kRowThreads) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sM[(w * R + r) * 2]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = fast_exp2(sM[(w * R + r) * 2] - base);
      sum += sM[(w * R + r) * 2 + 1] * f;
      const float4 x = *reinterpret_cast<const float4*>(sO + (w * R + r) * D + d);
      a.x += x.x * f;
      a.y += x.y * f;
      a.z += x.z * f;
      a.w += x.w * f;
    }
    if (ns > 1) {
      *reinterpret_cast<float4*>(p.part + (unit * R + r) * D + d) = a;
      if (d == 0) {
        float* ml = p.part + (int64_t)p.slots * p.Hkv * p.splits * R * D + (unit * R + r) * 2;
        ml[0] = mx;
        ml[1] = sum;
      }
    } else {
      const int tok = (r_base + r) / p.G, head = (r_base + r) % p.G, pos = off + tok;
      // A row that sees no key gives zeros.
      const int top = key_high(p, sq.L, pos);
      const bool any = top >= 0 && (top >= key_low(p, pos) || p.sinks > 0);
      const float inv = any ? 1.f / sum : 0.f;
      uint2 w;
      w.x = any ? pack_bf16(a.x * inv, a.y * inv) : 0u;
      w.y = any ? pack_bf16(a.z * inv, a.w * inv) : 0u;
      *reinterpret_cast<uint2*>(p.out + ((int64_t)(sq.start + tok) * p.Hq + h * p.G + head) * D + d) = w;
    }
  }
}

namespace {

template <int D, int KV, int R>
cudaError_t launch_rows_kv(const SeqParams& p, cudaStream_t stream) {
  using C = RowsCfg<D, KV, R>;
  static_assert(C::kCtas * (C::kSmem + 1024) <= 227 * 1024, "CTAs that share an SM");
  cudaError_t err = cudaFuncSetAttribute(rows_kernel<D, KV, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (err != cudaSuccess) return err;
  const int64_t tiles = (int64_t)p.slots * p.Hkv;
  rows_kernel<D, KV, R><<<(unsigned)(tiles * p.splits), kRowThreads, C::kSmem, stream>>>(p);
  err = cudaGetLastError();
  if (err != cudaSuccess || p.splits == 1) return err;
  join_kernel<D, R, C::kChunk><<<(unsigned)tiles, kJoinThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

template <int D, int R>
cudaError_t launch_rows_d(const SeqParams& p, int kv, cudaStream_t stream) {
  if (kv == kStrided) return launch_rows_kv<D, kStrided, R>(p, stream);
  if (kv == kPagedBf16) return launch_rows_kv<D, kPagedBf16, R>(p, stream);
  return launch_rows_kv<D, kPagedE4m3, R>(p, stream);
}

}  // namespace

// `rows`: of a tile, 8 or 16.
cudaError_t launch_rows(const SeqParams& p, int D, int kv, int rows, cudaStream_t stream) {
  if (D == 128) return rows == 8 ? launch_rows_d<128, 8>(p, kv, stream) : launch_rows_d<128, 16>(p, kv, stream);
  return rows == 8 ? launch_rows_d<64, 8>(p, kv, stream) : launch_rows_d<64, 16>(p, kv, stream);
}

}  // namespace solattn
