// How the tree attention's work is cut over its CTAs.  Plain arithmetic, the same on the host.
//
// A unit is up to kTiles query tiles (128 rows of (node, query head)) of one sequence and kv head, which
// share their keys' way through the chip; it costs `width` jobs for each chunk of 64 keys and kUnitJobs
// more.  A tree of more tiles has units of kTiles and one of what is left for each kv head (a chunk of three
// tiles takes 2820 clocks, of two 2330, of one 1040, so 3 + 1 is less than 2 + 2).  All units lie on one
// line, in order of sequence, full ones first, kv head and tiles; CTA c takes the line's piece [c per,
// (c + 1) per), cut at whole chunks.  The pieces of a unit lie in consecutive CTAs.
//
// Two ways to lay them out.  Dense: one behind the other, every CTA has the same amount of work, and most
// have pieces of two units.  Aligned: each unit begins with a CTA and is cut into equal pieces, so that
// no CTA begins twice and short units are not cut; taken where it makes the longest share little longer
// (kSlack jobs and an eighth), that is for few units.
#pragma once

#ifdef __CUDACC__
#define TI_HD __host__ __device__ __forceinline__
#else
#define TI_HD inline
#endif

namespace ti {
namespace tree {

constexpr int kChunk = 64;
constexpr int kUnitJobs = 4;             // beginning and end of a unit, in jobs
constexpr int kSnap = 2;                 // a piece has at least this many chunks (dense)
constexpr int kMinJobs = 16;             // a CTA's share: below it fewer CTAs take part
constexpr int kSlack = 10;
constexpr int kTries = 5;                // shares tried for the aligned layout

struct Units {                           // units of one width
  int chunks, width, count, jobs;        // jobs: of one
};
struct SeqWork {
  int keys, tiles, groups;               // groups: full units of a kv head
  Units full, rest;
};
struct Plan {
  unsigned per, aligned;
};

TI_HD SeqWork seq_work(int ctx, int nodes, bool known, int group, int kvh, int most_keys, int tiles_max) {
  SeqWork s{0, 0, 0, {0, 0, 0, 0}, {0, 0, 0, 0}};
  if (nodes <= 0) return s;
  const long long keys = (long long)(ctx > 0 ? ctx : 0) + nodes;
  s.keys = known ? (int)(keys < most_keys ? keys : most_keys) : 0;
  const int chunks = s.keys > 0 ? (s.keys + kChunk - 1) / kChunk : 1;
  s.tiles = (nodes * group + 127) / 128;
  s.groups = s.tiles <= tiles_max ? 1 : s.tiles / tiles_max;
  const int width = s.tiles < tiles_max ? s.tiles : tiles_max, left = s.tiles - s.groups * width;
  s.full = Units{chunks, width, s.groups * kvh, width * chunks + kUnitJobs};
  s.rest = Units{chunks, left, left > 0 ? kvh : 0, left * chunks + kUnitJobs};
  return s;
}

// The dense share of `total` jobs, and the k-th share tried for the aligned layout.
TI_HD unsigned dense_share(unsigned total, unsigned ctas) {
  const unsigned per = (total + ctas - 1) / ctas;
  return per > (unsigned)kMinJobs ? per : (unsigned)kMinJobs;
}
TI_HD unsigned tried_share(unsigned dense, int k) {
  return dense + dense * (unsigned)k / (8u * (kTries - 1)) + (unsigned)(k * kSlack / (kTries - 1));
}
// CTAs that a unit takes up in the aligned layout.
TI_HD int pieces(const Units& s, unsigned per) {
  return (unsigned)s.jobs <= per ? 1 : (int)(((unsigned)s.jobs + per - 1) / per);
}

// A unit's pieces, if the layout is aligned, and its length on the line.
TI_HD int pieces(const Units& s, const Plan& p) { return p.aligned ? pieces(s, p.per) : 1; }
TI_HD unsigned length(const Units& s, const Plan& p, int k) { return p.aligned ? (unsigned)k * p.per : (unsigned)s.jobs; }

// Jobs of all of a sequence's units; its pieces at a share of `per`; its length on the line.
TI_HD unsigned seq_jobs(const SeqWork& s) { return (unsigned)s.full.count * (unsigned)s.full.jobs + (unsigned)s.rest.count * (unsigned)s.rest.jobs; }
TI_HD unsigned seq_pieces(const SeqWork& s, unsigned per) {
  return (s.full.count ? (unsigned)(s.full.count * pieces(s.full, per)) : 0u) + (s.rest.count ? (unsigned)(s.rest.count * pieces(s.rest, per)) : 0u);
}
TI_HD unsigned seq_length(const SeqWork& s, const Plan& p) {
  return (unsigned)s.full.count * length(s.full, p, pieces(s.full, p)) + (unsigned)s.rest.count * length(s.rest, p, pieces(s.rest, p));
}

// The first chunk of a unit at [start, start + length) that lies behind place b of the line.
TI_HD int chunk_at(unsigned b, unsigned start, const Units& s, const Plan& p, int k) {
  if (b <= start) return 0;
  if (b >= start + length(s, p, k)) return s.chunks;
  if (p.aligned) {
    const int j = (int)((b - start) / p.per), each = s.chunks / k, rest = s.chunks - each * k;
    return each * j + (j < rest ? j : rest);
  }
  if (b - start < (unsigned)kUnitJobs) return 0;
  const unsigned jobs = b - start - kUnitJobs;
  const int c = (int)(s.width == 1 ? jobs : s.width == 2 ? jobs / 2 : jobs / 3);   // (three tiles at most)
  if (c < kSnap) return 0;
  return s.chunks - c < kSnap ? s.chunks : c;
}

// The CTAs that hold a unit's first and last chunk.
TI_HD int first_cta(unsigned start, const Units& s, const Plan& p, int k) {
  int c = (int)(start / p.per);
  while (chunk_at((unsigned)(c + 1) * p.per, start, s, p, k) == 0) ++c;
  return c;
}
TI_HD int last_cta(unsigned start, const Units& s, const Plan& p, int k) {
  if (p.aligned) return (int)(start / p.per) + k - 1;
  int c = (int)((start + length(s, p, k) - 1) / p.per);
  while (c > 0 && chunk_at((unsigned)c * p.per, start, s, p, k) >= s.chunks) --c;
  return c;
}

}  // namespace tree
}  // namespace ti
