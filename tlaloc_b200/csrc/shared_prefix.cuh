// How the work of attention over shared prefixes is cut: the same arithmetic on the device for the kernel that leaves records and the one that merges them.
//
// A unit is up to `unit_rows` (query row, head) pairs of one prefix that read one KV head; its work is the prefix's key tiles.  The tiles of all units laid
// end to end are cut into runs of equal length, one for each CTA, whatever units they fall in.  CTA c leaves one record {max, sum, acc[D]} per pair of every unit that
// its run touches, at block c + u of the records (u: the unit's number): each step along the line moves on to the next CTA, the next unit or both, so no block is
// used twice.  Nothing about the cut lies in memory: lengths and row ranges are read from the device, so a captured launch follows them.
#pragma once

#include "common.cuh"

namespace tlaloc_b200 {

struct PrefixPlan {
  const int* lens;    // [G]
  const int* starts;  // [G + 1]
  int G, R, group, Hkv;
  int max_len;        // positions that a prefix table holds
  int unit_rows, tile;
  int grid;           // CTAs of the record kernel
  int min_run;        // tiles, at least, of a CTA's run
  int max_blocks;     // blocks of records that there is room for
};

struct PrefixGroup {
  int row0, rows, len, units, tiles;  // units of one KV head; key tiles
  long long unit0, work0;             // units and tiles in front of it
};

__device__ __forceinline__ void PrefixGroupAt(const PrefixPlan& p, int g, PrefixGroup& r)
{
  r.row0 = r.rows = r.len = r.units = r.tiles = 0;
  if (g >= p.G) return;
  const int a = min(max(__ldcg(p.starts + g), 0), p.R), b = min(max(__ldcg(p.starts + g + 1), 0), p.R);
  r.row0 = a;
  r.rows = max(b - a, 0);
  r.len = min(max(__ldcg(p.lens + g), 0), p.max_len);
  r.units = r.len > 0 ? (r.rows * p.group + p.unit_rows - 1) / p.unit_rows : 0;
  r.tiles = (r.len + p.tile - 1) / p.tile;
}

__device__ __forceinline__ long long WarpSum(long long v)
{
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Tiles of a run.  The whole warp.
__device__ __forceinline__ long long PrefixRun(const PrefixPlan& p, long long* total)
{
  long long w = 0;
  const int lane = threadIdx.x & 31;
  for (int g = lane; g < p.G; g += 32) {
    PrefixGroup r;
    PrefixGroupAt(p, g, r);
    w += static_cast<long long>(r.units) * p.Hkv * r.tiles;
  }
  w = WarpSum(w);
  *total = w;
  return max((w + p.grid - 1) / p.grid, static_cast<long long>(p.min_run));
}

// The group that holds tile `work` of the line (by_row false), or query row `row` (by_row true).  The whole warp; false if there is none.
__device__ __forceinline__ bool PrefixFind(const PrefixPlan& p, bool by_row, long long at, PrefixGroup* found, int* index)
{
  const int lane = threadIdx.x & 31;
  long long unit_base = 0, work_base = 0;
  for (int g0 = 0; g0 < p.G; g0 += 32) {
    PrefixGroup r;
    PrefixGroupAt(p, g0 + lane, r);
    const long long units = static_cast<long long>(r.units) * p.Hkv, work = units * r.tiles;
    long long u = units, w = work;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long uu = __shfl_up_sync(0xffffffffu, u, o), ww = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) {
        u += uu;
        w += ww;
      }
    }
    r.unit0 = unit_base + u - units;
    r.work0 = work_base + w - work;
    const bool here = by_row ? at >= r.row0 && at < r.row0 + r.rows : at >= r.work0 && at < r.work0 + work;
    const unsigned any = __ballot_sync(0xffffffffu, here);
    if (any != 0u) {
      const int src = __ffs(any) - 1;
      found->row0 = __shfl_sync(0xffffffffu, r.row0, src);
      found->rows = __shfl_sync(0xffffffffu, r.rows, src);
      found->len = __shfl_sync(0xffffffffu, r.len, src);
      found->units = __shfl_sync(0xffffffffu, r.units, src);
      found->tiles = __shfl_sync(0xffffffffu, r.tiles, src);
      found->unit0 = __shfl_sync(0xffffffffu, r.unit0, src);
      found->work0 = __shfl_sync(0xffffffffu, r.work0, src);
      *index = g0 + src;
      return true;
    }
    unit_base += __shfl_sync(0xffffffffu, u, 31);
    work_base += __shfl_sync(0xffffffffu, w, 31);
  }
  return false;
}

// What one CTA does of one unit: pairs [pair0, pair0 + pairs) of the group's (row, head of the KV head) pairs, key tiles [tile0, tile1).
struct PrefixSegment {
  int row0, len, index, kv, pair0, pairs, tile0, tile1;
  int block;  // of the records; -1: there is no room (row ranges that overlap one another)
};

// The segment at `at` of a run that ends at `end`; moves `at` behind it.  The whole warp.
__device__ __forceinline__ bool PrefixNext(const PrefixPlan& p, long long run, long long end, long long* at, PrefixSegment* s)
{
  PrefixGroup g;
  int index = 0;
  if (*at >= end || !PrefixFind(p, false, *at, &g, &index)) return false;
  const long long in = *at - g.work0;
  const int unit = static_cast<int>(in / g.tiles);
  s->tile0 = static_cast<int>(in % g.tiles);
  s->tile1 = static_cast<int>(min(static_cast<long long>(g.tiles), s->tile0 + end - *at));
  s->row0 = g.row0;
  s->len = g.len;
  s->index = index;
  s->kv = unit / g.units;
  s->pair0 = (unit % g.units) * p.unit_rows;
  s->pairs = min(p.unit_rows, g.rows * p.group - s->pair0);
  const long long block = *at / run + g.unit0 + unit;
  s->block = block < p.max_blocks ? static_cast<int>(block) : -1;
  *at += s->tile1 - s->tile0;
  return true;
}

// The maximum as a record has it.  Where the sum is not a number the maximum is none either: of scores that are all NaN it would be -infinity, which says "no keys".
__device__ __forceinline__ float RecordMax(float top, float sum) { return sum != sum ? sum : top; }

struct PrefixArgs {
  PrefixPlan plan;
  const void* q;
  const void* kc;
  const void* vc;
  const int* tables;  // [G, M]
  float* acc;         // [max_blocks, unit_rows, d8]: weighted sums of values, rows of whole 32-byte words
  float* heads;       // [max_blocks, unit_rows, 2]: {max, sum}, the maximum in units of the natural exponential
  int H, D, d8, bs, M, P;
  float scale;
};

// The record kernel on the tensor cores (shared_prefix_tc.cu): what its units and tiles are, whether it takes a call, its launch.
constexpr int kPrefixTcPairs = 256, kPrefixTcKeys = 128, kPrefixTcGrid = 148;
bool PrefixTcApplies(const PrefixArgs& a, int q_dtype, int kv_dtype);
cudaError_t LaunchPrefixTc(const PrefixArgs& a, int q_dtype, int kv_dtype, int out_dtype, cudaStream_t st);

}  // namespace tlaloc_b200
