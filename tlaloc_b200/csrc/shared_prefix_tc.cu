// Records of shared prefixes on the tensor cores: bf16 pools, head sizes of multiples of 8 up to 128, pages of multiples of 8 positions.
//
// The (row, head) pairs that read one KV head of a prefix are the rows of a matrix product: S = Q K^T over tiles of 128 pairs x 128 keys, O += P V, both tcgen05.mma
// kind::f16 with f32 accumulators in TMEM, keys and values by TMA out of their pages.  A CTA runs two streams of tiles, each with its own scores, weights (in the scores'
// place), outputs and running maximum, so that one's products run under the other's softmax:
//   a unit of more than 128 pairs    a stream takes 128 pairs and every tile of keys: a tile is fetched once for both
//   a unit of up to 128 pairs        the streams take the same pairs and every second tile of keys, and merge their results in the end
//   producer warp   a tile's boxes (64 channels x as many positions as lie in one page), each lane some of them, onto a ring of slots
//   MMA lane        in turn for the streams: O += P(j) V(j), S(j + 1)
//   eight warps     softmax, stream w by warps 4 w .. 4 w + 3, a thread a pair; before that the queries into shared memory, at the end the records
// An f32 query enters as two bf16 parts.  Where the result is f32 the weights do as well (2^-17 of them is lost); for a bf16 result one part is enough: what is lost
// (2^-9 of each weight, at random) is less than the result's own rounding.
// Every mbarrier wait is bounded.
#include <cuda.h>

#include <algorithm>

#include "shared_prefix.cuh"
#include "tc_common.cuh"

namespace tlaloc_b200 {
namespace {

using namespace tc;

constexpr int kRows = 128, kKeys = kPrefixTcKeys;
constexpr int kAtom = kRows * 64 * 2;  // 128 rows x 64 channels
constexpr int kWarps = 8, kThreads = kWarps * 32 + 64;
constexpr int kBudget = 224 * 1024;    // queries and ring; a KB to align them and static shared memory come on top
constexpr int kMaxSlots = 8;
constexpr float kLazy = 8.f;           // how far (log2) a row's maximum may grow past the reference in use
constexpr float kLn2 = 0.6931471805599453f;

__device__ int g_prefix_status = 0;

__host__ __device__ constexpr uint32_t InstrDesc(int n, bool b_mn_major)  // f32 accumulator, bf16, A K-major, M = 128
{
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void TmaBox(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar)
{
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
               : "memory");
}
__device__ __forceinline__ float Exp2(float x)
{
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t Pack(float a, float b)
{
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float Low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float High(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ void Store32(uint32_t dst, uint4 v)
{
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// Eight values as one 32-byte word: a thread writes a row of a record by itself, and whole sectors are all that counts.
__device__ __forceinline__ void StoreSector(float* dst, const float* v)
{
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]),
               "f"(v[7])
               : "memory");
}
__device__ __forceinline__ void FenceAsync() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void SoftmaxWarpsSync() { asm volatile("bar.sync 1, 256;\n" ::: "memory"); }

// ATOMS: 64-channel blocks of a head.  PLO: the weights in two parts.
template <typename QT, int ATOMS>
struct PrefixTcLayout {
  static constexpr bool kQLo = sizeof(QT) == 4;
  static constexpr int kPart = ATOMS * kAtom;               // 128 pairs of queries (one part of them), or 128 keys or values
  static constexpr int kQTile = kPart * (kQLo ? 2 : 1);
  static constexpr int kSlots = (kBudget - 2 * kQTile) / kPart < kMaxSlots ? (kBudget - 2 * kQTile) / kPart : kMaxSlots;
  static constexpr int kBytes = 2 * kQTile + kSlots * kPart + 1024;
};

// The order in which a segment's n tiles of keys (0, 2, ..) and values (1, 3, ..) are used, as places in the ring's sequence.  One stream takes tiles one after the other
// (K0 V0 K1 V1 ..); two streams of alternate tiles want both first scores ahead (K0 K1 V0 K2 V1 ..).
__device__ __forceinline__ int KeyItem(bool split, int t) { return !split ? 2 * t : (t == 0 ? 0 : 2 * t - 1); }
__device__ __forceinline__ int ValueItem(bool split, int n, int t) { return !split ? 2 * t + 1 : (t == n - 1 ? 2 * n - 1 : 2 * t + 2); }

template <typename QT, int ATOMS, bool PLO>
__global__ void __launch_bounds__(kThreads, 1)
    PrefixTc(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ PrefixArgs a, const int box)
{
  using Layout = PrefixTcLayout<QT, ATOMS>;
  constexpr int kSlots = Layout::kSlots, kPart = Layout::kPart;
  extern __shared__ unsigned char smem_raw[];
  __shared__ alignas(8) uint64_t bars[2 * kMaxSlots + 7];
  __shared__ uint32_t slot_store[2];
  const uint32_t base = (SmemAddr(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - SmemAddr(smem_raw));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // full: a slot's tile has landed; empty: its products are done.  Per stream, sfull: scores are there; pfull: weights are; odone: the last product of a segment is done.
  const uint32_t full = SmemAddr(bars), empty = full + 8 * kMaxSlots, sfull = empty + 8 * kMaxSlots, pfull = sfull + 16, odone = pfull + 16, qfull = odone + 16;
  const uint32_t ring = base + 2 * Layout::kQTile;
  volatile uint32_t* slot = slot_store;
  volatile uint32_t* abort_word = slot_store + 1;
  if (tid == 0) {
    *abort_word = 0u;
    for (int i = 0; i < kSlots; ++i) {
      MbarInit(full + 8 * i, 1);
      MbarInit(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      MbarInit(sfull + 8 * i, 1);
      MbarInit(pfull + 8 * i, 4);
      MbarInit(odone + 8 * i, 1);
    }
    MbarInit(qfull, kWarps);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(SmemAddr(slot_store)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
  const uint32_t tmem = *slot;  // S of stream w at column 128 w, O at 256 + 128 w
  GridDependencySync();
  bool ok = true;
  long long total;
  const long long run = PrefixRun(a.plan, &total);
  long long at = blockIdx.x * run;
  const long long end = min(at + run, total);
  PrefixSegment s;
  int items = 0;  // of the ring, in front of this segment

  if (warp == kWarps) {
    const int boxes = kKeys / box, atom = lane / boxes, mine = lane - atom * boxes;  // up to 32 boxes an item: 16 of 8 positions by two atoms
    while (PrefixNext(a.plan, run, end, &at, &s)) {
      const int n = s.tile1 - s.tile0;
      const bool split = s.pairs <= kRows && n > 1;
      const int* table = a.tables + static_cast<size_t>(s.index) * a.M;
      auto tile_of = [&](int i, bool* value) {
        if (!split) {
          *value = (i & 1) != 0;
          return i >> 1;
        }
        *value = i == 2 * n - 1 || (i > 0 && (i & 1) == 0);
        return i == 0 ? 0 : i == 2 * n - 1 ? n - 1 : (i & 1) != 0 ? (i + 1) >> 1 : (i >> 1) - 1;
      };
      auto row_of = [&](int i) {  // the first pool row of this lane's box, -1 if it lies past the prefix's end
        bool value;
        const int pos = (s.tile0 + tile_of(i, &value)) * kKeys + mine * box;
        if (atom >= ATOMS || pos >= s.len) return -1;
        const int page = min(max(__ldg(table + pos / a.bs), 0), a.P - 1);
        return page * a.bs + pos % a.bs;
      };
      int row = row_of(0);
      for (int i = 0; i < 2 * n; ++i) {
        const int it = items + i, sl = it % kSlots, use = it / kSlots;
        const int next = i + 1 < 2 * n ? row_of(i + 1) : -1;  // on its way while the slot is waited for
        if (use > 0) ok = MbarWaitWarp(empty + 8 * sl, (use - 1) & 1, lane, abort_word) && ok;
        const unsigned live = __ballot_sync(0xffffffffu, row >= 0);
        bool value;
        tile_of(i, &value);
        if (lane == 0) MbarExpectTx(full + 8 * sl, __popc(live) * box * 128);
        __syncwarp();
        if (row >= 0) TmaBox(ring + sl * kPart + atom * kAtom + mine * box * 128, value ? &map_v : &map_k, atom * 64, s.kv, row, full + 8 * sl);
        row = next;
      }
      items += 2 * n;
    }
    if (!ok) {  // given up: let the copies in flight land before the CTA's shared memory goes away
      volatile uint32_t never = 0;
      for (int it = max(0, items - kSlots); it < items; ++it) MbarWaitWarp(full + 8 * (it % kSlots), (it / kSlots) & 1, lane, &never);
    }
  } else if (warp == kWarps + 1) {
    const uint32_t s_idesc = InstrDesc(kKeys, false), o_idesc = InstrDesc((a.D + 15) / 16 * 16, true);
    const uint64_t qd = SmemDesc(base, 16, 1024), kd = SmemDesc(ring, 16, 1024), vd = SmemDesc(ring, kAtom, 1024);
    const int steps = (a.D + 15) / 16;  // of 16 channels
    int segment = 0, done[2] = {0, 0};
    while (PrefixNext(a.plan, run, end, &at, &s)) {
      const int n = s.tile1 - s.tile0;
      const bool pair_tiles = s.pairs > kRows, split = !pair_tiles && n > 1;
      const int count[2] = {pair_tiles ? n : (n + 1) / 2, pair_tiles ? n : n / 2};
      if (ElectOne()) {
        ok = MbarWait(qfull, segment & 1, abort_word) && ok;
        auto scores = [&](int w, int j) {
          const int t = pair_tiles ? j : 2 * j + w, it = items + KeyItem(split, t), sl = it % kSlots;
          ok = MbarWait(full + 8 * sl, (it / kSlots) & 1, abort_word) && ok;
          asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
          // The stream's last weights lay here; their product is in front of these MMAs in the same queue.
          const uint32_t acc = tmem + w * 128;
#pragma unroll
          for (int part = 0; part < (Layout::kQLo ? 2 : 1); ++part) {
            const uint64_t qa = qd + static_cast<uint64_t>(((pair_tiles ? w : 0) * Layout::kQTile + part * kPart) >> 4);
            const uint64_t ka = kd + static_cast<uint64_t>((sl * kPart) >> 4);
#pragma unroll
            for (int k = 0; k < 4 * ATOMS; ++k)
              if (k < steps) TcMmaBf16(acc, qa + (k >> 2) * (kAtom >> 4) + 2 * (k & 3), ka + (k >> 2) * (kAtom >> 4) + 2 * (k & 3), s_idesc, part > 0 || k > 0 ? 1u : 0u);
          }
          TcCommit(sfull + 8 * w);
          if (!pair_tiles || w == 1) TcCommit(empty + 8 * sl);
        };
        scores(0, 0);
        if (count[1] > 0) scores(1, 0);
        for (int j = 0; j < count[0]; ++j) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (j >= count[w]) continue;
            const int t = pair_tiles ? j : 2 * j + w, it = items + ValueItem(split, n, t), sl = it % kSlots;
            const int live = min(kKeys, s.len - (s.tile0 + t) * kKeys);
            ok = MbarWait(full + 8 * sl, (it / kSlots) & 1, abort_word) && ok;
            ok = MbarWait(pfull + 8 * w, (done[w] + j) & 1, abort_word) && ok;
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            // P: eight columns per 16 keys; V: keys are its rows, 16 of them per step; those that hold none are left out
            const uint32_t pa = tmem + w * 128, acc = tmem + 256 + w * 128;
            const uint64_t va = vd + static_cast<uint64_t>((sl * kPart) >> 4);
#pragma unroll
            for (int part = 0; part < (PLO ? 2 : 1); ++part) {
#pragma unroll
              for (int k = 0; k < kKeys / 16; ++k)
                if (16 * k < live) TcMmaTmemA(acc, pa + 64 * part + 8 * k, va + ((k * 16 * 128) >> 4), o_idesc, j > 0 || part > 0 || k > 0 ? 1u : 0u);
            }
            if (!pair_tiles || w == 1) TcCommit(empty + 8 * sl);
            if (j + 1 == count[w]) TcCommit(odone + 8 * w);
            else scores(w, j + 1);
          }
        }
      }
      __syncwarp();
      items += 2 * n;
      done[0] += count[0];
      done[1] += count[1];
      ++segment;
    }
  } else {
    const int w = warp >> 2, quad = warp & 3, r = quad * 32 + lane;  // this thread's stream and TMEM lane
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16, sa = tmem + lanes + w * 128, oa = tmem + lanes + 256;
    // The scale's sign (or its being zero) goes into the queries: the largest score is the largest scaled one, and no masked score is multiplied by zero.
    const float scale_log2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * 1.4426950408889634f, sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f;
    int tiles_done = 0, segments = 0;
    while (PrefixNext(a.plan, run, end, &at, &s)) {
      const int n = s.tile1 - s.tile0;
      const bool pair_tiles = s.pairs > kRows, split = !pair_tiles && n > 1;
      const int count = pair_tiles ? n : (n + 1 - w) / 2;
      // Queries: rows of 128 bytes an atom, swizzled as TMA would; zeros for pairs and channels that are not there.
      constexpr int kChunks = ATOMS * 8;
      for (int i = tid; i < (pair_tiles ? 2 * kRows : kRows) * kChunks; i += kWarps * 32) {
        const int pair = i / kChunks, c = i % kChunks;
        float v[8] = {};
        if (pair < s.pairs && c * 8 < a.D) {
          const int p = s.pair0 + pair;
          const QT* src = static_cast<const QT*>(a.q) + (static_cast<size_t>(s.row0 + p / a.plan.group) * a.H + s.kv * a.plan.group + p % a.plan.group) * a.D + c * 8;
          if constexpr (Layout::kQLo) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(src)), y = __ldcg(reinterpret_cast<const float4*>(src) + 1);
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
          } else {
            const uint4 x = __ldcg(reinterpret_cast<const uint4*>(src));
            v[0] = Low(x.x), v[1] = High(x.x), v[2] = Low(x.y), v[3] = High(x.y), v[4] = Low(x.z), v[5] = High(x.z), v[6] = Low(x.w), v[7] = High(x.w);
          }
        }
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = v[2 * e] * sign, y = v[2 * e + 1] * sign;
          hi[e] = Pack(x, y);
          lo[e] = Pack(x - Low(hi[e]), y - High(hi[e]));
        }
        const uint32_t dst = base + (pair >> 7) * Layout::kQTile + (c >> 3) * kAtom + (pair & 127) * 128 + (((c & 7) ^ (pair & 7)) << 4);
        Store32(dst, make_uint4(hi[0], hi[1], hi[2], hi[3]));
        if constexpr (Layout::kQLo) Store32(dst + kPart, make_uint4(lo[0], lo[1], lo[2], lo[3]));
      }
      FenceAsync();
      __syncwarp();
      if (lane == 0) MbarArrive(qfull);
      const bool live_warp = (pair_tiles ? w * kRows : 0) + quad * 32 < s.pairs;
      float top = -INFINITY, sum = 0.f;
      for (int j = 0; j < count; ++j) {
        const int t = pair_tiles ? j : 2 * j + w, live = min(kKeys, s.len - (s.tile0 + t) * kKeys);
        ok = MbarWaitWarp(sfull + 8 * w, tiles_done & 1, lane, abort_word) && ok;
        ++tiles_done;
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        if ((live & 15) != 0 && (split || w == 0)) {
          // Values behind the end in the last 16 that are multiplied: 0 times whatever the page holds there must stay 0.
          const int it = items + ValueItem(split, n, t), sl = it % kSlots;
          ok = MbarWaitWarp(full + 8 * sl, (it / kSlots) & 1, lane, abort_word) && ok;
          const int dead = 16 - (live & 15);
          for (int i = r; i < dead * kChunks; i += kRows) {
            const int c = i / dead, row = live + i % dead;
            Store32(ring + sl * kPart + (c >> 3) * kAtom + row * 128 + ((c & 7) << 4), make_uint4(0u, 0u, 0u, 0u));
          }
          FenceAsync();
        }
        if (live_warp) {
          uint32_t x[kKeys];
#pragma unroll
          for (int c = 0; c < kKeys; c += 32) TcLd32(sa + c, x + c);
          asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
          if (live < kKeys) {
#pragma unroll
            for (int e = 0; e < kKeys; ++e)
              if (e >= live) x[e] = 0xff800000u;
          }
          float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < kKeys; ++e) t4[e & 3] = fmaxf(t4[e & 3], __uint_as_float(x[e]));
          const float tile_top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * scale_log2;
          if (__any_sync(0xffffffffu, tile_top > top + kLazy || (top == -INFINITY && tile_top > -INFINITY))) {
            const float next = fmaxf(top, tile_top), keep = top == -INFINITY ? 0.f : Exp2(top - next);
            if (j > 0) {  // O has every tile before this one in it: their products were ahead of these scores
#pragma unroll
              for (int c = 0; c < ATOMS * 64; c += 32) {
                uint32_t o[32];
                TcLd32(oa + w * 128 + c, o);
                asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                TcSt32(oa + w * 128 + c, o);
              }
            }
            sum *= keep;
            top = next;
          }
          const float ref = top == -INFINITY ? 0.f : top;
          float s4[4] = {};
#pragma unroll
          for (int half = 0; half < 2; ++half) {  // 64 keys: 32 columns of weights, and 32 of what they lose as bf16
            uint32_t hi[32], lo[PLO ? 32 : 1];
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const float p0 = Exp2(fmaf(__uint_as_float(x[64 * half + e]), scale_log2, -ref)), p1 = Exp2(fmaf(__uint_as_float(x[64 * half + e + 1]), scale_log2, -ref));
              s4[e & 2] += p0;
              s4[(e & 2) + 1] += p1;
              hi[e / 2] = Pack(p0, p1);
              if constexpr (PLO) lo[e / 2] = Pack(p0 - Low(hi[e / 2]), p1 - High(hi[e / 2]));
            }
            TcSt32(sa + 32 * half, hi);
            if constexpr (PLO) TcSt32(sa + 64 + 32 * half, lo);
          }
          sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
          asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
        }
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) MbarArrive(pfull + 8 * w);
      }
      if (count > 0) {
        ok = MbarWaitWarp(odone + 8 * w, segments & 1, lane, abort_word) && ok;
        ++segments;
      }
      asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
      const size_t rec = static_cast<size_t>(max(s.block, 0)) * kPrefixTcPairs + (pair_tiles ? w * kRows : 0) + r;
      const bool mine = s.block >= 0 && (pair_tiles ? w * kRows : 0) + r < s.pairs;
      float* out = a.acc + rec * a.d8;
      if (!split) {
        if (mine && (pair_tiles || w == 0)) *reinterpret_cast<float2*>(a.heads + 2 * rec) = make_float2(RecordMax(top * kLn2, sum), sum);
        if (live_warp && (pair_tiles || w == 0)) {
#pragma unroll
          for (int c = 0; c < ATOMS * 64; c += 32) {
            float o[32];
            TcLd32(oa + w * 128 + c, reinterpret_cast<uint32_t*>(o));
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (mine && c + e < a.d8) StoreSector(out + c + e, o + e);
          }
        }
      } else {
        // Both streams have these pairs: each takes half of the channels of both.  They meet where a second tile of queries would lie.
        float2* both = reinterpret_cast<float2*>(smem + Layout::kQTile);
        if (sum != sum) top = sum;  // no score was a number: the record is not one either
        both[w * kRows + r] = make_float2(top, sum);
        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
        SoftmaxWarpsSync();
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        const float2 other = both[(w ^ 1) * kRows + r];
        const float ref = fmaxf(top, other.x);
        const float f_mine = top == -INFINITY ? 0.f : Exp2(top - ref), f_other = other.x == -INFINITY ? 0.f : Exp2(other.x - ref);
        const float f0 = w == 0 ? f_mine : f_other, f1 = w == 0 ? f_other : f_mine;
        const float all = sum * f_mine + other.y * f_other;
        if (mine && w == 0) *reinterpret_cast<float2*>(a.heads + 2 * rec) = make_float2(RecordMax(ref * kLn2, all), all);
        if (live_warp) {
#pragma unroll
          for (int c = 0; c < ATOMS * 32; c += 32) {
            const int col = w * ATOMS * 32 + c;
            float o[32], o1[32];
            TcLd32(oa + col, reinterpret_cast<uint32_t*>(o));
            TcLd32(oa + 128 + col, reinterpret_cast<uint32_t*>(o1));
            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = o[e] * f0 + o1[e] * f1;
#pragma unroll
            for (int e = 0; e < 32; e += 8)
              if (mine && col + e < a.d8) StoreSector(out + col + e, o + e);
          }
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
      SoftmaxWarpsSync();  // accumulators and queries of this segment are read: the next one's may come
      items += 2 * n;
    }
  }
  if (!ok) atomicExch(&g_prefix_status, 1);
  __syncthreads();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
  }
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A bf16 pool [positions][kv heads][channels], boxes of 64 channels of one head x `box` positions.
bool Encode(CUtensorMap* map, const void* pool, const PrefixArgs& a, int box)
{
  auto encode = reinterpret_cast<EncodeTiledFn>(TensorMapEncoder());
  if (encode == nullptr) return false;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(a.D), static_cast<cuuint64_t>(a.plan.Hkv), static_cast<cuuint64_t>(a.P) * a.bs};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(a.D) * 2, static_cast<cuuint64_t>(a.plan.Hkv) * a.D * 2};
  const cuuint32_t boxes[3] = {64, 1, static_cast<cuuint32_t>(box)};
  const cuuint32_t elem[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(pool), dims, strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename QT, int ATOMS, bool PLO>
cudaError_t Prepare()
{
  return cudaFuncSetAttribute(PrefixTc<QT, ATOMS, PLO>, cudaFuncAttributeMaxDynamicSharedMemorySize, PrefixTcLayout<QT, ATOMS>::kBytes);
}
template <typename QT>
cudaError_t PrepareBoth()
{
  cudaError_t e = Prepare<QT, 1, false>();
  if (e == cudaSuccess) e = Prepare<QT, 1, true>();
  if (e == cudaSuccess) e = Prepare<QT, 2, false>();
  if (e == cudaSuccess) e = Prepare<QT, 2, true>();
  return e;
}
cudaError_t PreparePrefixTc()
{
  static OncePerDevice once;
  return once.Run([](int) {
    TensorMapEncoder();
    const cudaError_t e = PrepareBoth<float>();
    return e == cudaSuccess ? PrepareBoth<__nv_bfloat16>() : e;
  });
}
int ReadPrefixStatus()
{
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_prefix_status, sizeof(int)) != cudaSuccess) return -1;
  if (v != 0) {
    const int zero = 0;
    cudaMemcpyToSymbol(g_prefix_status, &zero, sizeof(int));
  }
  return v;
}
KernelSetup g_setup(PreparePrefixTc, ReadPrefixStatus);

// Positions of a box: the most that always lie in one page.
int BoxOf(int block_size) { return std::min(block_size & -block_size, kKeys); }

template <typename QT, int ATOMS>
cudaError_t Launch(const PrefixArgs& a, bool plo, cudaStream_t st)
{
  CUtensorMap map_k, map_v;
  const int box = BoxOf(a.bs);
  if (!Encode(&map_k, a.kc, a, box) || !Encode(&map_v, a.vc, a, box)) return cudaErrorInvalidValue;
  const int smem = PrefixTcLayout<QT, ATOMS>::kBytes;
  return plo ? LaunchChained(PrefixTc<QT, ATOMS, true>, a.plan.grid, kThreads, smem, st, map_k, map_v, a, box)
             : LaunchChained(PrefixTc<QT, ATOMS, false>, a.plan.grid, kThreads, smem, st, map_k, map_v, a, box);
}

}  // namespace

bool PrefixTcApplies(const PrefixArgs& a, int q_dtype, int kv_dtype)
{
  return kv_dtype == TLALOC_B200_BF16 && IsFloatType(q_dtype) && a.D >= 8 && a.D <= 128 && a.D % 8 == 0 && a.bs % 8 == 0 && Aligned16(a.q) && Aligned16(a.kc) &&
         Aligned16(a.vc) && static_cast<long long>(a.P) * a.bs < (1ll << 31) && TensorMapEncoder() != nullptr;
}

cudaError_t LaunchPrefixTc(const PrefixArgs& a, int q_dtype, int kv_dtype, int out_dtype, cudaStream_t st)
{
  (void)kv_dtype;
  const cudaError_t e = PreparePrefixTc();
  if (e != cudaSuccess) return e;
  const bool plo = out_dtype == TLALOC_B200_F32;
  if (q_dtype == TLALOC_B200_F32) return a.D <= 64 ? Launch<float, 1>(a, plo, st) : Launch<float, 2>(a, plo, st);
  return a.D <= 64 ? Launch<__nv_bfloat16, 1>(a, plo, st) : Launch<__nv_bfloat16, 2>(a, plo, st);
}

}  // namespace tlaloc_b200
