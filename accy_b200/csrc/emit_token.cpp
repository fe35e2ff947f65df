// Kernels of the token side of a language model: scatter_add (the gradient of an embedding lookup) and
// the log-probabilities of given tokens with their gradient.  The lookup itself is no kernel of its own:
// a gather is an indirect row offset in whatever row kernel consumes it (emit_row.cpp).
#include <algorithm>
#include <iomanip>
#include <sstream>

#include "plan.hpp"

namespace accy {
namespace {

std::string num(int64_t v) { return std::to_string(v); }

std::string loadConv(DType d, const std::string& raw) {
  if (d == DType::bf16) return "bf16_to_f32(" + raw + ")";
  if (d == DType::f16) return "f16_to_f32(" + raw + ")";
  if (d == DType::i1) return "(" + raw + " != 0)";
  return raw;
}

std::string storeConv(DType d, const std::string& v) {
  if (d == DType::bf16) return "f32_to_bf16(" + v + ")";
  if (d == DType::f16) return "f32_to_f16(" + v + ")";
  return v;
}

// An elementwise expression evaluated at row `r` (flat over the dims below `split`) and, for nodes that
// change along the columns, at the `vec` columns from `c0` on.
struct Pointwise {
  const std::vector<ENode>& nodes;
  const std::vector<LeafRef>& leaves;
  const std::vector<int64_t>& extents;
  int split;
  int vec = 1;
  int acc = -1;               // node that stands for the enclosing kernel's own value
  std::string acc_name, prefix;

  uint32_t rowMask() const { return split >= 32 ? 0xffffffffu : ((1u << split) - 1u); }
  bool element(int i) const { return (nodes[i].vary & ~rowMask()) != 0; }
  std::string name(int i) const { return i == acc ? acc_name : prefix + num(i); }
  std::string at(int i) const { return element(i) ? name(i) + "[e]" : name(i); }
  int rank() const { return static_cast<int>(extents.size()); }

  // one run of stride 1 over the columns that `vec`-wide accesses from any column block may read
  bool wide(const LeafRef& l) const {
    int64_t expect = 1;
    for (int d = rank() - 1; d >= split; --d) {
      if (extents[d] == 1) continue;
      if (l.strides[d] != expect) return false;
      expect *= extents[d];
    }
    for (int d = 0; d < split; ++d)
      if (extents[d] != 1 && l.strides[d] % vec != 0) return false;
    return true;
  }

  // Loads of several rows ahead: the buffers' values as they are stored, `slots` of them per leaf, so that a
  // row in flight takes no more registers than its bytes; `unpacked` makes node values of slot `a`.
  bool buffered(int i) const { return nodes[i].op == ENode::Leaf && element(i); }
  void declareBuffered(int i, std::ostream& o, const std::string& ind, const std::string& slots) const {
    o << ind << "Pack<" << storageTypeOf(leaves[nodes[i].leaf].dtype) << ", " << vec << "> raw_" << name(i) << "[" << slots << "];\n";
  }
  void loadBuffered(int i, std::ostream& o, const std::string& ind) const {
    const LeafRef& l = leaves[nodes[i].leaf];
    const std::string L = "L" + num(nodes[i].leaf), st = storageTypeOf(l.dtype), row = indexExpr(extents, l.strides, 0, split, "r");
    if (vec > 1 && wide(l)) {
      o << ind << "raw_" << name(i) << "[a * COLUMNS + v] = *reinterpret_cast<const Pack<" << st << ", " << vec << ">*>(" << L << " + " << row << " + c0);\n";
    } else {
      o << ind << "#pragma unroll\n" << ind << "for (int e = 0; e < " << vec << "; ++e) raw_" << name(i) << "[a * COLUMNS + v].v[e] = " << L
        << "[" << row << " + " << indexExpr(extents, l.strides, split, rank(), "(c0 + e)") << "];\n";
    }
  }
  void unpacked(int i, std::ostream& o, const std::string& ind) const {
    o << ind << ctypeOf(nodes[i].dtype) << " " << name(i) << "[" << vec << "];\n" << ind << "#pragma unroll\n" << ind << "for (int e = 0; e < "
      << vec << "; ++e) " << name(i) << "[e] = " << loadConv(leaves[nodes[i].leaf].dtype, "raw_" + name(i) + "[a * COLUMNS + v].v[e]") << ";\n";
  }

  void leafLoad(int i, std::ostream& o, const std::string& ind) const {
    const ENode& n = nodes[i];
    const LeafRef& l = leaves[n.leaf];
    o << ind << "const " << ctypeOf(n.dtype) << " " << name(i) << " = "
      << loadConv(l.dtype, "L" + num(n.leaf) + "[" + indexExpr(extents, l.strides, 0, split, "r") + "]") << ";\n";
  }

  void emit(int i, std::ostream& o, const std::string& ind) const {
    const ENode& n = nodes[i];
    const std::string ty = ctypeOf(n.dtype);
    if (i == acc) return;
    if (n.op == ENode::Leaf) return buffered(i) ? unpacked(i, o, ind) : leafLoad(i, o, ind);
    const bool el = element(i);
    std::string value;
    if (n.op == ENode::Const) value = constLiteral(n);
    else if (n.op == ENode::Iota) {
      std::vector<int64_t> one(extents.size(), 0);
      one[n.dim] = 1;
      value = "(" + ty + ")(" + (n.dim < split ? indexExpr(extents, one, 0, split, "r") : indexExpr(extents, one, split, rank(), "(c0 + e)")) + ")";
    } else {
      auto arg = [&](int k) { return n.args[k] >= 0 ? at(n.args[k]) : std::string(); };
      value = elementwiseExpr(n, arg(0), arg(1), arg(2), nodes[n.args[n.op == ENode::Sel ? 1 : 0]].dtype);
    }
    if (!el) o << ind << "const " << ty << " " << name(i) << " = " << value << ";\n";
    else
      o << ind << ty << " " << name(i) << "[" << vec << "];\n" << ind << "#pragma unroll\n" << ind << "for (int e = 0; e < " << vec
        << "; ++e) " << name(i) << "[e] = " << value << ";\n";
  }

  std::string params() const {
    std::string out;
    for (size_t l = 0; l < leaves.size(); ++l) out += std::string(", const ") + storageTypeOf(leaves[l].dtype) + "* __restrict__ L" + num(static_cast<int64_t>(l));
    return out;
  }
};

int addKernel(Plan& plan, const std::string& name, const char* family, const std::string& source) {
  KernelSource k;
  k.name = name;
  k.family = family;
  k.source = source;
  // recorded operations keep one rounding each; the kernels' own fused steps are written out
  k.options.push_back("--fmad=false");
  plan.kernels.push_back(k);
  return static_cast<int>(plan.kernels.size()) - 1;
}

KernelArg slotArg(int slot) {
  KernelArg a;
  a.slot = slot;
  return a;
}

int scratchSlot(Plan& plan, size_t bytes) {
  Slot s;
  s.role = Slot::Scratch;
  s.bytes = bytes;
  plan.slots.push_back(s);
  return static_cast<int>(plan.slots.size()) - 1;
}

int64_t ceilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

void define(std::ostream& o, const char* name, const std::string& value) { o << "#define " << name << " " << value << "\n"; }

// ---------------------------------------------------------------------------------------------
// scatter_add
// ---------------------------------------------------------------------------------------------
// out[p, v, :] = base[p, v, :] + sum over the i with index[i] = v of update[p, i, :], in the order of i.
//
// The indices are sorted once, stably, so that every row's updates are a run of the sorted list; runs
// are then summed by walking the list in equal pieces, whatever the rows' counts are (a padding token may
// own half of a batch and most tokens own one place).  No sum is an atomic one: the result is the same on
// every run.  Three launches:
//   order  one cluster of eight CTAs sorts by least significant digits and exchanges digit counts through distributed
//          shared memory.  Meanwhile the other CTAs write the rows that no index names, which for a large
//          vocabulary is most of the traffic;
//   sum    one CTA per (piece of the list, block of columns): a thread holds its columns' running sum in
//          registers (f32 or wider) with eight rows in flight, and writes a row when its run ends.  Runs that cross the ends
//          of a piece leave partial sums;
//   join   adds the partial sums of the runs that cross, in order.
// The floor is memory: updates once, rows once.
const char* kOrderCommon = R"CUDA(
__device__ __forceinline__ unsigned int row_of(IT x) {
  const long long v = (long long)x;
  return v >= 0 && v < EXTENT ? (unsigned int)v : (unsigned int)EXTENT;
}
#define PER_LOAD (16 / (int)sizeof(IT))

// The rows that no index names: zeros, or the base's row.  Filler f of FILLERS takes every FILLERS-th group of 32
// rows, so that frequent (low) numbers, whose rows are not its work, are no filler's alone.  `bits` is a
// bitmap in shared memory of the named rows of up to WORDS groups.
#define WORDS 1024
#define GROUPS ((EXTENT + 31) / 32)
__device__ __forceinline__ void mark(IT x, unsigned int f, unsigned int first, unsigned int* bits) {
  const unsigned int v = row_of(x), group = v >> 5, turn = group / FILLERS;
  if (v < EXTENT && group - turn * FILLERS == f && turn - first < WORDS) atomicOr(&bits[turn - first], 1u << (v & 31));
}
__device__ __forceinline__ void fill_rows(const IT* __restrict__ I, OT* __restrict__ out, BASE_PARAM_ unsigned int f, unsigned int* bits) {
  const int lane = threadIdx.x & 31;
  for (long long first = 0; first * FILLERS + f < GROUPS; first += WORDS) {
    long long words = (GROUPS - f + FILLERS - 1) / FILLERS - first;
    if (words > WORDS) words = WORDS;
    __syncthreads();
    for (int w = threadIdx.x; w < words; w += THREADS) bits[w] = 0u;
    __syncthreads();
    const long long loads = COUNT / PER_LOAD;
#pragma unroll 4
    for (long long i = threadIdx.x; i < loads; i += THREADS) {
      const Pack<IT, PER_LOAD> some = reinterpret_cast<const Pack<IT, PER_LOAD>*>(I)[i];
#pragma unroll
      for (int k = 0; k < PER_LOAD; ++k) mark(some.v[k], f, (unsigned int)first, bits);
    }
    for (long long i = loads * PER_LOAD + threadIdx.x; i < COUNT; i += THREADS) mark(I[i], f, (unsigned int)first, bits);
    __syncthreads();
    for (int w = threadIdx.x >> 5; w < words; w += THREADS / 32) {
      const long long row0 = ((first + w) * FILLERS + f) * 32;
      unsigned int open = ~bits[w];
      if (EXTENT - row0 < 32) open &= (1u << (EXTENT - row0)) - 1u;
      while (open) {   // runs of rows without an index: one range of memory each
        const int from_bit = __ffs(open) - 1;
        const unsigned int after = ~(open >> from_bit);
        const int run = after ? __ffs(after) - 1 : 32;
        open &= run + from_bit >= 32 ? (1u << from_bit) - 1u : ~(((1u << run) - 1u) << from_bit);
        for (long long p = 0; p < PRE; ++p) {
          const long long begin = (p * EXTENT + row0 + from_bit) * POST, end = begin + run * POST;
#if FROM_ZEROS
          // whole 16-byte units, the elements before and after them one by one
          constexpr int U = 16 / (int)sizeof(OT);
          long long from = (begin + U - 1) / U * U, to = end / U * U;
          if (from > to) from = to = end;
          if (begin + lane < from) out[begin + lane] = (OT)0;
          if (to + lane < end) out[to + lane] = (OT)0;
          uint4* at = reinterpret_cast<uint4*>(out + from) + lane;
          uint4* const stop = reinterpret_cast<uint4*>(out + to);
#pragma unroll 1
          for (; at + 7 * 32 < stop; at += 8 * 32) {
#pragma unroll
            for (int u = 0; u < 8; ++u) at[u * 32] = make_uint4(0u, 0u, 0u, 0u);
          }
          for (; at < stop; at += 32) *at = make_uint4(0u, 0u, 0u, 0u);
#else
          for (long long q = begin + lane * FVEC; q < end; q += 32 * FVEC) {
            Pack<OT, FVEC> o;
#pragma unroll
            for (int e = 0; e < FVEC; ++e) o.v[e] = FILL_VALUE(q + e);
            *reinterpret_cast<Pack<OT, FVEC>*>(out + q) = o;
          }
#endif
        }
      }
    }
  }
}
)CUDA";

const char* kOrderTemplate = R"CUDA(
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ unsigned int peer_word(const unsigned int* p, unsigned int cta) {
  const unsigned int a = (unsigned int)__cvta_generic_to_shared(p);
  unsigned int b, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(cta));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(b) : "memory");
  return v;
}
// Keys are taken BATCH at a time per lane, all of a batch's loads before its first use.  Where a lane has no
// more than one batch, the places found while counting are kept for the second loop.
#define BATCH 8
#define ONE_BATCH (SLICE <= BATCH * 32)
extern "C" __global__ void __cluster_dims__(8, 1, 1) __launch_bounds__(THREADS, 2)
KERNEL(const IT* __restrict__ I, uint2* list_a, uint2* list_b, OT* __restrict__ out BASE_PARAM) {
  __shared__ unsigned int pool[WARPS * RADIX > WORDS ? WARPS * RADIX : WORDS];
  __shared__ unsigned int total[RADIX], start[RADIX], wsum[WARPS];
  if (blockIdx.x >= 8) {   // whole clusters take this branch
    fill_rows(I, out, BASE_ARG_ blockIdx.x - 8, pool);
    return;
  }
  unsigned int (*hist)[RADIX] = reinterpret_cast<unsigned int (*)[RADIX]>(pool);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned int cta = blockIdx.x;
  // every warp owns one run of SLICE places, in order: that is what keeps the sort stable
  const long long w0 = ((long long)cta * WARPS + warp) * SLICE, w1 = w0 + SLICE < COUNT ? w0 + SLICE : COUNT;
  for (int pass = 0; pass < PASSES; ++pass) {
    // the last pass writes list a
    const bool to_a = ((PASSES - 1 - pass) & 1) == 0;
    const uint2* from = to_a ? list_b : list_a;
    uint2* to = to_a ? list_a : list_b;
    const int shift = pass * DIGIT_BITS;
    uint2 k[BATCH];   // key and place
    unsigned int offset[BATCH];
    for (int d = threadIdx.x; d < WARPS * RADIX; d += THREADS) (&hist[0][0])[d] = 0u;
    __syncthreads();
    for (long long b = w0; b < w1; b += BATCH * 32) {
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const long long i = b + j * 32 + lane;
        if (i < w1) k[j] = pass == 0 ? make_uint2(row_of(I[i]), (unsigned int)i) : __ldcg(from + i);
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        if (b + j * 32 >= w1) break;
        const bool in = b + j * 32 + lane < w1;
        const unsigned int d = in ? (k[j].x >> shift) & (RADIX - 1) : RADIX;
        const unsigned int peers = __match_any_sync(0xffffffffu, d);
        if (in) offset[j] = hist[warp][d] + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
        if (in && lane == __ffs(peers) - 1) hist[warp][d] += __popc(peers);
        __syncwarp();
      }
    }
    __syncthreads();
    if (threadIdx.x < RADIX) {
      unsigned int sum = 0u;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const unsigned int n = hist[w][threadIdx.x];
        hist[w][threadIdx.x] = sum;
        sum += n;
      }
      total[threadIdx.x] = sum;
    }
    cluster_sync();
    unsigned int all = 0u, before = 0u;
    if (threadIdx.x < RADIX) {
#pragma unroll
      for (unsigned int c = 0; c < 8; ++c) {
        const unsigned int n = peer_word(&total[threadIdx.x], c);
        all += n;
        if (c < cta) before += n;
      }
    }
    unsigned int inc = all;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned int n = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += n;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    if (threadIdx.x < RADIX) {
      unsigned int ex = inc - all;
      for (int w = 0; w < warp; ++w) ex += wsum[w];
      start[threadIdx.x] = ex + before;
    }
    __syncthreads();
    for (long long b = w0; b < w1; b += BATCH * 32) {
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const long long i = b + j * 32 + lane;
        if (!ONE_BATCH && i < w1) k[j] = pass == 0 ? make_uint2(row_of(I[i]), (unsigned int)i) : __ldcg(from + i);
      }
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        if (b + j * 32 >= w1) break;
        const bool in = b + j * 32 + lane < w1;
        const unsigned int d = in ? (k[j].x >> shift) & (RADIX - 1) : RADIX;
        if (ONE_BATCH) {
          // hist holds what this CTA's earlier warps have of the digit
          if (in) offset[j] += hist[warp][d];
        } else {
          const unsigned int peers = __match_any_sync(0xffffffffu, d);
          if (in) offset[j] = hist[warp][d] + __popc(peers & ((1u << lane) - 1u));
          __syncwarp();
          if (in && lane == __ffs(peers) - 1) hist[warp][d] += __popc(peers);
          __syncwarp();
        }
        if (in) to[start[d] + offset[j]] = k[j];
      }
    }
    cluster_sync();   // the list is complete, and nobody reads this pass's counts any more
  }
}
)CUDA";

// A thread has COLUMNS vectors of VEC columns, THREADS vectors apart: where rows are too badly aligned for 16-byte
// accesses it takes that many narrower ones, so that what a row costs besides (its key, its place, the end of
// its run) is spread over as much data.
const char* kSumHead = R"CUDA(
// p * EXTENT + k and the like fit 32 bits in all but the largest calls; a 32-bit factor makes the offset one instruction
#define OFFSET(row) ((long long)(ROW_T)(row) * POST)
__device__ __forceinline__ void write_row(OT* __restrict__ out, BASE_PARAM_ long long off, const VT* sum) {
  Pack<OT, VEC> o;
#pragma unroll
  for (int e = 0; e < VEC; ++e) o.v[e] = WITH_BASE(off + e, sum[e]);
  *reinterpret_cast<Pack<OT, VEC>*>(out + off) = o;
}
#define EACH_COLUMN(v, c0) _Pragma("unroll") for (int v = 0; v < COLUMNS; ++v) if (const long long c0 = column + v * (THREADS * VEC); c0 < POST)
)CUDA";

const char* kSumBody = R"CUDA(
  __shared__ unsigned int key[PIECE + AHEAD + 2], pos[PIECE + AHEAD + 2];   // of place i at i + 1
  const long long begin = (long long)blockIdx.x * PIECE;
  const int n = COUNT - begin < PIECE ? (int)(COUNT - begin) : PIECE;
  // key[0] and key[n + 1] are the neighbours' keys; EXTENT + 1 stands for none
  for (int i = threadIdx.x; i < PIECE + AHEAD + 2; i += THREADS) {
    const long long at = begin + i - 1;
    const uint2 one = i < n + 2 && at >= 0 && at < COUNT ? list[at] : make_uint2((unsigned int)EXTENT + 1u, 0u);
    key[i] = one.x;
    pos[i] = one.y;
  }
  __syncthreads();
  const long long column = ((long long)blockIdx.y * (THREADS * COLUMNS) + threadIdx.x) * VEC;
  const ROW_T p_index = (ROW_T)blockIdx.z * (ROW_T)COUNT, p_row = (ROW_T)blockIdx.z * (ROW_T)EXTENT;
  VT sum[COLUMNS * VEC];
#pragma unroll
  for (int e = 0; e < COLUMNS * VEC; ++e) sum[e] = 0;
  bool first = true;   // the run that starts this piece
  for (int i = 0; i < n; i += AHEAD) {
    unsigned int k[AHEAD + 1];
#pragma unroll
    for (int a = 0; a <= AHEAD; ++a) k[a] = key[i + a + 1];
    DECLARE
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i + a >= n || k[a] >= (unsigned int)EXTENT) break;
      const ROW_T r = p_index + pos[i + a + 1];
      (void)r;
      EACH_COLUMN(v, c0) {
        LOAD
      }
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i + a >= n) break;
      if (k[a] >= (unsigned int)EXTENT) return;   // indices outside the axis come last
      const ROW_T r = p_index + pos[i + a + 1];
      (void)r;
      EACH_COLUMN(v, c0) {
        UPDATE
      }
      const bool last = i + a + 1 == n;
      if (!last && k[a + 1] == k[a]) continue;
      // the run ends here, or the piece does
      const bool from_before = first && key[0] == k[a], goes_on = last && k[a + 1] == k[a];
      first = false;
      if (from_before || goes_on) {
        VT* to = partial + (((long long)blockIdx.z * PIECES + blockIdx.x) * 2 + (from_before ? 0 : 1)) * POST;
        EACH_COLUMN(v, c0) {
          Pack<VT, VEC> part;
#pragma unroll
          for (int e = 0; e < VEC; ++e) part.v[e] = sum[v * VEC + e];
          *reinterpret_cast<Pack<VT, VEC>*>(to + c0) = part;
        }
      } else {
        EACH_COLUMN(v, c0) write_row(out, BASE_ARG_ OFFSET(p_row + k[a]) + c0, sum + v * VEC);
      }
#pragma unroll
      for (int e = 0; e < COLUMNS * VEC; ++e) sum[e] = 0;
    }
  }
}
)CUDA";

const char* kJoinBody = R"CUDA(
  const long long piece = blockIdx.x, begin = piece * PIECE, end = begin + PIECE;
  if (end >= COUNT) return;
  const unsigned int k = list[end - 1].x, next = list[end].x, before = begin > 0 ? list[begin - 1].x : (unsigned int)EXTENT + 1u;
  // the run at the end of this piece goes on, and began in it
  if (k >= (unsigned int)EXTENT || next != k || before == k) return;
  // how many of the following pieces begin with it: they are next to each other
  long long more = 0;
  for (;;) {
    const long long at = (piece + 1 + more + threadIdx.x) * PIECE;
    const int here = __syncthreads_count(at < COUNT && list[at].x == k);
    more += here;
    if (here < THREADS) break;
  }
  const long long c0 = ((long long)blockIdx.y * THREADS + threadIdx.x) * VEC;
  if (c0 >= POST) return;
  const long long p = blockIdx.z;
  const VT* from = partial + (p * PIECES + piece) * 2 * POST + c0;
  VT sum[VEC];
  {
    const Pack<VT, VEC> part = *reinterpret_cast<const Pack<VT, VEC>*>(from + POST);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = part.v[e];
  }
#pragma unroll 1
  for (long long m = 1; m <= more; m += AHEAD) {
    Pack<VT, VEC> part[AHEAD];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (m + a > more) break;
      part[a] = *reinterpret_cast<const Pack<VT, VEC>*>(from + (m + a) * 2 * POST);
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (m + a > more) break;
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] = sum[e] + part[a].v[e];
    }
  }
  write_row(out, BASE_ARG_ OFFSET((ROW_T)p * (ROW_T)EXTENT + k) + c0, sum);
}
)CUDA";

}  // namespace

void emitScatterAdd(const ScatterOp& s, const std::string& name, Plan& plan, const ScheduleOverrides& ov) {
  if (s.extent > 0x7ffffff0ll || s.count > 0x7ffffff0ll) throw PlanError("scatter_add over more than 2^31-16 rows or indices is not supported");
  if (s.pre > 65535) throw PlanError("scatter_add with more than 65535 leading blocks is not supported");
  const bool wide = s.dtype == DType::f64;
  // 16-byte accesses where every row starts on their boundary, narrower ones otherwise
  const int widest = std::max(1, 16 / static_cast<int>(std::max(dtypeSize(s.out_dtype), dtypeSize(s.dtype))));
  int vec = widest, fvec = 16 / static_cast<int>(dtypeSize(s.out_dtype));
  while (vec > 1 && s.post % vec != 0) vec /= 2;
  while (fvec > 1 && s.post % fvec != 0) fvec /= 2;
  int bits = 1;
  while ((int64_t{1} << bits) < s.extent + 1) ++bits;
  const int passes = static_cast<int>(ceilDiv(bits, 9)), digit_bits = static_cast<int>(ceilDiv(bits, passes));
  const int64_t out_bytes = s.pre * s.extent * s.post * static_cast<int64_t>(dtypeSize(s.out_dtype));
  // Fillers in whole clusters, no more than write 64 KB each.  Clusters are placed two CTAs to an SM before all SMs have
  // one, so it takes several per SM to use them all (131072 rows of 8 KB: 346 us for all three launches with 17 clusters,
  // 297 with 26, 268 with 71, 281 with 140).
  const int64_t fillers = 8 * std::max<int64_t>(1, std::min<int64_t>(ceilDiv(out_bytes, 8 * 65536), (ov.sm_count - 4) / 2));

  const int columns = static_cast<int>(std::min<int64_t>(widest / vec, ceilDiv(s.post, 32 * vec)));
  const int64_t lanes = ceilDiv(s.post, vec * columns);   // threads that a row takes
  const int64_t blocks = ceilDiv(lanes, 256);
  const int threads = static_cast<int>(ceilDiv(ceilDiv(lanes, blocks), 32) * 32);
  if (blocks > 65535) throw PlanError("scatter_add rows are too long");
  // At least four CTAs per SM while pieces are worth having: a piece is walked one place after the other, about 0.15 us
  // each, and each piece may leave two partial sums (bf16 16384 places of 4096: 104 us in pieces of 8, 86 of 32, 96 of 128;
  // f32 9999 of 513: 35, 31 and 51; bf16 2048 of 2048: 35, 41 and 68).
  int64_t piece = 8;
  while (piece < 128 && ceilDiv(s.count, piece * 2) * blocks * s.pre >= 4 * ov.sm_count) piece *= 2;
  const int64_t pieces = ceilDiv(s.count, piece);

  const int list_a = scratchSlot(plan, s.count * 8), list_b = scratchSlot(plan, s.count * 8);
  const int partial = scratchSlot(plan, static_cast<size_t>(s.pre * pieces * 2 * s.post) * (wide ? 8 : 4));

  const std::string ot = storageTypeOf(s.out_dtype), bt = storageTypeOf(s.base_dtype), vt = ctypeOf(s.dtype);
  auto head = [&](std::ostream& o) {
    o << kernelPrelude();
    define(o, "IT", storageTypeOf(s.index_dtype));
    define(o, "OT", ot);
    define(o, "VT", vt);
    define(o, "EXTENT", num(s.extent) + "ll");
    define(o, "COUNT", num(s.count) + "ll");
    define(o, "POST", num(s.post) + "ll");
    define(o, "PRE", num(s.pre) + "ll");
    if (s.base_slot >= 0) {
      const std::string load = loadConv(s.base_dtype, "base[off]");
      o << "#define BASE_PARAM , const " << bt << "* __restrict__ base\n#define BASE_PARAM_ const " << bt << "* __restrict__ base,\n#define BASE_ARG_ base,\n";
      o << "#define FILL_VALUE(at) " << storeConv(s.out_dtype, loadConv(s.base_dtype, "base[at]")) << "\n";
      o << "#define WITH_BASE(at, sum) " << storeConv(s.out_dtype, "(" + loadConv(s.base_dtype, "base[at]") + " + sum)") << "\n";
    } else {
      o << "#define BASE_PARAM\n#define BASE_PARAM_\n#define BASE_ARG_\n#define FILL_VALUE(at) (" << ot << ")0\n#define WITH_BASE(at, sum) " << storeConv(s.out_dtype, "sum") << "\n";
    }
  };
  {
    std::ostringstream o;
    head(o);
    define(o, "KERNEL", name + "_order");
    define(o, "THREADS", "512");
    define(o, "FROM_ZEROS", s.base_slot < 0 ? "1" : "0");
    define(o, "FVEC", num(fvec));
    define(o, "FILLERS", num(fillers) + "u");
    define(o, "WARPS", "16");
    define(o, "PASSES", num(passes));
    define(o, "DIGIT_BITS", num(digit_bits));
    define(o, "RADIX", num(1 << digit_bits));
    define(o, "SLICE", num(ceilDiv(s.count, 8 * 16 * 32) * 32));
    o << kOrderCommon << kOrderTemplate;
    Launch l;
    l.kernel = addKernel(plan, name + "_order", "scatter_add", o.str());
    l.grid[0] = static_cast<uint32_t>(8 + fillers);
    l.block[0] = 512;
    l.label = name + " order";
    for (int slot : {s.index_slot, list_a, list_b, s.out_slot}) l.args.push_back(slotArg(slot));
    if (s.base_slot >= 0) l.args.push_back(slotArg(s.base_slot));
    plan.launches.push_back(l);
  }
  auto sumHead = [&](std::ostream& o, const char* kernel, const std::string& more, int threads, int vec, int columns, int ahead) {
    head(o);
    define(o, "COLUMNS", num(columns));
    define(o, "ROW_T", s.pre * std::max(s.extent, s.count) < (int64_t{1} << 32) ? "unsigned int" : "long long");
    define(o, "THREADS", num(threads));
    define(o, "VEC", num(vec));
    define(o, "PIECE", num(piece));
    define(o, "PIECES", num(pieces) + "ll");
    define(o, "AHEAD", num(ahead));
    o << kSumHead << "extern \"C\" __global__ void __launch_bounds__(" << threads << ") " << name << kernel
      << "(const uint2* __restrict__ list, " << vt << "* __restrict__ partial, " << ot
      << "* __restrict__ out BASE_PARAM" << more << ") {\n";
  };
  auto sumLaunch = [&](int kernel, const char* what, int threads, int64_t blocks) {
    Launch l;
    l.kernel = kernel;
    l.grid[0] = static_cast<uint32_t>(pieces);
    l.grid[1] = static_cast<uint32_t>(blocks);
    l.grid[2] = static_cast<uint32_t>(s.pre);
    l.block[0] = static_cast<uint32_t>(threads);
    l.label = name + what;
    for (int slot : {list_a, partial, s.out_slot}) l.args.push_back(slotArg(slot));
    if (s.base_slot >= 0) l.args.push_back(slotArg(s.base_slot));
    return l;
  };
  {
    Pointwise g{s.updates.nodes, s.updates.leaves, s.updates.extents, s.updates.split, vec, -1, "", "n"};
    std::ostringstream o, declare, load, update;
    for (size_t i = 0; i < g.nodes.size(); ++i) {
      const int n = static_cast<int>(i);
      if (g.buffered(n)) {
        g.declareBuffered(n, declare, "    ", "AHEAD * COLUMNS");
        g.loadBuffered(n, load, "      ");
      }
      g.emit(n, update, "      ");
    }
    update << "#pragma unroll\n      for (int e = 0; e < VEC; ++e) sum[v * VEC + e] = sum[v * VEC + e] + " << g.at(s.result) << ";\n";
    sumHead(o, "_sum", g.params(), threads, vec, columns, 8);
    std::string body = kSumBody;
    body.replace(body.find("DECLARE"), 7, declare.str());
    body.replace(body.find("LOAD\n"), 5, load.str());
    body.replace(body.find("UPDATE\n"), 7, update.str());
    o << body;
    Launch l = sumLaunch(addKernel(plan, name + "_sum", "scatter_add", o.str()), " sum", threads, blocks);
    for (const LeafRef& leaf : s.updates.leaves) l.args.push_back(slotArg(leaf.slot));
    plan.launches.push_back(l);
  }
  if (pieces > 1) {
    // partial sums are f32 or f64: 16 bytes of them per thread, sixteen in flight
    const int join_vec = std::min(vec, wide ? 2 : 4);
    const int64_t join_lanes = ceilDiv(s.post, join_vec), join_blocks = ceilDiv(join_lanes, 256);
    const int join_threads = static_cast<int>(ceilDiv(ceilDiv(join_lanes, join_blocks), 32) * 32);
    if (join_blocks > 65535) throw PlanError("scatter_add rows are too long");
    std::ostringstream o;
    sumHead(o, "_join", "", join_threads, join_vec, 1, 16);
    o << kJoinBody;
    plan.launches.push_back(sumLaunch(addKernel(plan, name + "_join", "scatter_add", o.str()), " join", join_threads, join_blocks));
  }
}

// ---------------------------------------------------------------------------------------------
// log-probabilities of tokens
// ---------------------------------------------------------------------------------------------
namespace {

// The arithmetic.  With c = fl(m log2 e) for a reference m near the row's maximum,
//
//   e[v] = 2^(x[v] log2 e - c)    log p = (x[token] - m) - (ln(sum e) - ln 2 (m log2 e - c))    p[v] = e[v] / sum e
//
// one fused step and one ex2.approx per element.  c is the same for every element that is summed with it
// or divided by the sum, so its rounding cancels, and the fused step rounds at the size of its result: rows whose
// logits are all far from zero lose nothing.  References are combined as 2^(c1 - c2), for the same
// reason.  A reference of 1e34 or more might overflow c: such rows (logits at the type's lowest value)
// subtract first.  Where the logits are others times a number, the number goes into the constant (L2E below).
//
// An exponent is rounded at its own size, so a reference that lies d below the row's maximum costs the largest terms d times
// 2^-24 or so.  A thread moves its reference when a logit exceeds it by more than 5.5 (exponents of the largest
// terms then stay below 8), and adds what comes after a new reference to a sum of its own: the many small terms beside
// a token the model is sure of are not rounded one by one at the size of that token's.  Log-probabilities of such
// rows are within 6e-7 (the largest of 600 rows each of 32003 to 300007 logits, the token 14 to 40 above the mean; with
// a window of 40 and one sum 4e-6, some of them positive).  bf16 8192 x 131072 with the gradient 708 us, f32
// 1023 x 32003 56.0 us (with the window of 40 and one sum 712 and 55.4; with 4, which moves it more often, 720 and 57.3;
// with an exact running maximum 730 and 57.4; with compensated sums 732 and 57.4, without smaller errors).
const char* kTokenCommon = R"CUDA(
#define LN2 0.6931471805599453f
#define NEG_INF __uint_as_float(0xff800000u)
#if IN_BITS == 32
__device__ __forceinline__ float value_of(XT x) { return x; }
#define NEG_INF_WORD 0xff800000u
#elif IN_BF16
__device__ __forceinline__ float value_of(XT x) { return bf16_to_f32(x); }
#define NEG_INF_WORD 0xff80ff80u
#else
__device__ __forceinline__ float value_of(XT x) { return f16_to_f32(x); }
#define NEG_INF_WORD 0xfc00fc00u
#endif

struct Raw { unsigned int w[4]; };   // 16 bytes of a row

__device__ __forceinline__ void unpack(const Raw& v, float (&f)[E]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#if IN_BITS == 32
    f[i] = __uint_as_float(v.w[i]);
#elif IN_BF16
    f[2 * i] = __uint_as_float(v.w[i] << 16);
    f[2 * i + 1] = __uint_as_float(v.w[i] & 0xffff0000u);
#else
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}" : "=f"(f[2 * i]), "=f"(f[2 * i + 1]) : "r"(v.w[i]));
#endif
  }
}
// the larger of each pair of packed elements (a NaN loses: it shows up in the sum)
__device__ __forceinline__ unsigned int packed_max(unsigned int a, unsigned int b) {
#if IN_BITS == 32
  return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
#elif IN_BF16
  unsigned int r; asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r;
#else
  unsigned int r; asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b)); return r;
#endif
}
__device__ __forceinline__ float largest(unsigned int packed) {
#if IN_BITS == 32
  return __uint_as_float(packed);
#else
  return fmaxf(value_of((XT)(packed & 0xffffu)), value_of((XT)(packed >> 16)));
#endif
}
// whether c would overflow (f16 logits cannot get there; an infinite one gives NaN either way)
__device__ __forceinline__ bool huge_ref(float m) {
#if IN_BITS == 32 || IN_BF16
  return fabsf(m) >= 1e34f && m != NEG_INF;
#else
  return false;
#endif
}
// what to add to x log2 e: -c; nothing for a row that has no finite element yet, or that subtracts first
__device__ __forceinline__ float minus_c(float m) { return m == NEG_INF || huge_ref(m) ? 0.0f : -(m * L2E); }
// a sum relative to `from` seen relative to `to` >= from (an empty sum has from = -inf)
__device__ __forceinline__ float moved(float s, float from, float to) {
  if (to == NEG_INF) return s;
  return s * ex2_ftz(huge_ref(to) ? (from - to) * L2E : from * L2E + minus_c(to));
}
// 2^(x log2 e - c) of a vector.  HUGE, the rare case, is a template argument and not a condition here:
// the compiler would execute it under a predicate for every element.
template <bool HUGE> __device__ __forceinline__ void exps(const Raw& v, float m, float minus, float (&f)[E]) {
  unpack(v, f);
  if (HUGE) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = f[e] - m;
  }
  const unsigned long long scale = pk2(L2E, L2E), add = pk2(minus, minus);
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    float a, b;
    upk2(fma2(pk2(f[e], f[e + 1]), scale, add), a, b);
    f[e] = ex2_ftz(a);
    f[e + 1] = ex2_ftz(b);
  }
}
// a thread's share of a row's sum: s + rest relative to m.  `rest` is what was added since m last moved.
struct Sum {
  float m, s, limit, rest, minus;
  __device__ __forceinline__ Sum() : m(NEG_INF), s(0.0f), limit(NEG_INF), rest(0.0f), minus(0.0f) {}
  template <int N> __device__ __forceinline__ void fold(const Raw (&raw)[N]) {
    unsigned int top = raw[0].w[0];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) top = packed_max(top, raw[i].w[q]);
    const float t = largest(top);
    const bool top_here = t > limit;
    if (top_here) {
      s = moved(s + rest, m, t);
      rest = 0.0f;
      m = t;
      minus = minus_c(t);
      limit = t + 5.5f / SCALE;
    }
    if (huge_ref(m)) add<true>(raw, top_here);
    else add<false>(raw, top_here);
  }
  template <bool HUGE, int N> __device__ __forceinline__ void add(const Raw (&raw)[N], bool top_here) {
    unsigned long long acc;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float f[E];
      exps<HUGE>(raw[i], m, minus, f);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const unsigned long long pair = pk2(f[e], f[e + 1]);
        acc = i + e == 0 ? pair : add2(acc, pair);
      }
    }
    float lo, hi;
    upk2(acc, lo, hi);
    if (top_here) s = s + (lo + hi);
    else rest = rest + (lo + hi);
  }
  // the sum over W neighbouring lanes, in every one of them
  template <int W> __device__ __forceinline__ void across_lanes() {
    float top = m;
    if (W == 32) {
      asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(m));
    } else {
#pragma unroll
      for (int off = W / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off, W));
    }
    s = moved(s + rest, m, top);
    rest = 0.0f;
    m = top;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off, W);
  }
};
// (x - m) - log(sum of e^(x - m)): the sum is relative to c instead of m log2 e, which is off by a known residue.  The
// difference is taken before anything is rounded at the size of x.
__device__ __forceinline__ float log_prob_at(float x, float m, float total) {
  const float residue = huge_ref(m) ? 0.0f : __fmaf_rn(m, L2E, minus_c(m));
  const float log_prob = (x - m) * SCALE - (logf(total) - residue * LN2);
  return log_prob > 0.0f ? 0.0f : log_prob;   // a probability of one, rounded
}

#if GRADIENT
__device__ __forceinline__ void store_vector(GT* p, const float (&f)[E]) {
#if OUT_16
  unsigned int w[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2) asm("cvt.rn." OUT_16_NAME "x2.f32 %0, %1, %2;" : "=r"(w[e / 2]) : "f"(f[e + 1]), "f"(f[e]));
#if IN_BITS == 32
  WRITE(reinterpret_cast<uint2*>(p), make_uint2(w[0], w[1]));
#else
  WRITE(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
#endif
#else
#pragma unroll
  for (int e = 0; e < E; e += 4) WRITE(reinterpret_cast<float4*>(p + e), make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]));
#endif
}
// What a row's gradient is made of: k = -slope / sum, the slope, and the vector with the token's element.
struct Slope {
  float m, minus, k, g, x;
  long long at;
  int vector;
  __device__ __forceinline__ Slope(float m_, float total, float slope, bool known, long long tok, float x_, int lead)
      : m(m_), minus(minus_c(m_)), g(known ? slope * GRAD_SCALE : 0.0f), x(x_), at(tok), vector(known ? (int)((tok + lead) / E) : -1) {
    k = -g / total;
  }
  // rows that take the slow way: those the loss does not depend on are zero whatever their logits hold
  __device__ __forceinline__ bool special() const { return g == 0.0f || huge_ref(m); }
  template <bool SPECIAL> __device__ __forceinline__ void of(const Raw& v, float (&f)[E]) const {
    if (SPECIAL && g == 0.0f) {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = 0.0f;
      return;
    }
    if (SPECIAL && huge_ref(m)) exps<true>(v, m, minus, f);
    else exps<false>(v, m, minus, f);
    const unsigned long long kk = pk2(k, k);
#pragma unroll
    for (int e = 0; e < E; e += 2) upk2(mul2(pk2(f[e], f[e + 1]), kk), f[e], f[e + 1]);
  }
  // by the thread that wrote the vector with the token's element, after it: that element again
  __device__ __forceinline__ void token(GT* grow, int j) const {
    if (j != vector || g == 0.0f) return;
    const float e = ex2_ftz(huge_ref(m) ? (x - m) * L2E : __fmaf_rn(x, L2E, minus));
    grow[at] = STORE((e * k + g));
  }
};
// the elements of an edge vector that belong to the row
__device__ __forceinline__ void store_edge(GT* grow, int first, const float (&f)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (first + e >= 0 && first + e < VOCAB) grow[first + e] = STORE(f[e]);
}
#endif
)CUDA";

// One row of logits per TPR threads (PARTS CTAs of a cluster share a long row while there are few rows).  A
// thread holds its part of the row in registers (longer rows in chunks), and the row's sums are combined
// through shuffles, shared memory and, in a cluster, distributed shared memory.  The gradient is written
// from the registers that hold the row, so logits are read once and the gradient written once; the slope of
// each row (what the recorded program does to its log-probability on the way to the loss) is evaluated in
// between.  Rows need not be aligned: a row is covered by aligned 16-byte vectors, and the elements of the first
// and last one that belong to its neighbours are left out.
const char* kTokenTemplate = R"CUDA(
__device__ __forceinline__ float2 peer_pair(const float2* p, unsigned int cta) {
  const unsigned int a = (unsigned int)__cvta_generic_to_shared(p);
  unsigned int b;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(cta));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(b) : "memory");
  return v;
}
__device__ __forceinline__ Raw load_inner(const XT* __restrict__ at) {
  Raw v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]) : "l"(at));
  return v;
}
// vector j of a row whose first element is element `lead` of its first aligned vector; elements outside
// the row read as -inf
__device__ __forceinline__ Raw load_vector(const XT* __restrict__ row, int lead, int vectors, int j) {
  Raw v;
  const int first = j * E - lead;
  if (j < vectors && first >= 0 && first + E <= VOCAB) {
    v = load_inner(row + first);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = NEG_INF_WORD;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (j >= vectors || first + e < 0 || first + e >= VOCAB) continue;
#if IN_BITS == 32
      v.w[e] = __float_as_uint(row[first + e]);
#else
      const unsigned int bits = row[first + e];
      v.w[e / 2] = (e & 1) ? (v.w[e / 2] & 0xffffu) | (bits << 16) : (v.w[e / 2] & 0xffff0000u) | bits;
#endif
    }
  }
  return v;
}

// whether this thread's vectors of the chunk that starts at vector j1 lie in the row
__device__ __forceinline__ bool inner_chunk(int j1, int lead) {
  return j1 * E - lead >= 0 && (j1 + (VPT - 1) * TPR + 1) * E - lead <= VOCAB;
}
__device__ __forceinline__ void load_chunk(const XT* mine, const XT* row, int lead, int vectors, int j0, int ck, Raw (&raw)[VPT]) {
  const int j1 = j0 + ck * (VPT * TPR);
  if (inner_chunk(j1, lead)) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) raw[i] = load_inner(mine + (ck * VPT + i) * (TPR * E));
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) raw[i] = load_vector(row, lead, vectors, j1 + i * TPR);
  }
}

extern "C" __global__ void CLUSTER __launch_bounds__(THREADS, MIN_BLOCKS)
KERNEL(const XT* __restrict__ X, const TT* __restrict__ T, float* __restrict__ log_prob_out, float2* __restrict__ stats, GT* __restrict__ G LEAF_PARAMS) {
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int part = PARTS > 1 ? (int)(blockIdx.x % PARTS) : 0;
  long long r = (long long)(blockIdx.x / PARTS) * RPC + sub;
  const bool row_ok = r < ROWS;
  if (!row_ok) r = ROWS - 1;
  const long long tok = (long long)T[r];
  const bool known = tok >= 0 && tok < VOCAB;
  LEAVES
  const XT* row = X + r * VOCAB;
  const int lead = (int)(((unsigned long long)row & 15ull) / sizeof(XT));
  const int vectors = (lead + VOCAB + E - 1) / E;
  const int j0 = part * (CHUNKS * TPR * VPT) + t;
  const XT* mine = row + ((long long)j0 * E - lead);   // this thread's first vector
  float xt = 0.0f;
  Raw raw[VPT];
#if STATS_IN
  if (known) xt = value_of(row[tok]);
  const float2 kept = stats[r];
  const float m = kept.x, total = kept.y;
#else
  Sum sum;
  for (int ck = 0; ck < CHUNKS; ++ck) {
    load_chunk(mine, row, lead, vectors, j0, ck, raw);
    // behind the first loads: its address has to wait for the token
    if (ck == 0 && known) xt = value_of(row[tok]);
    sum.fold(raw);
  }
  // the row's threads: lanes, then warps, then CTAs
  sum.across_lanes<(TPR < 32 ? TPR : 32)>();
#if TPR > 32
  __shared__ float2 cells[RPC * (TPR / 32)];
  if ((t & 31) == 0) cells[sub * (TPR / 32) + (t >> 5)] = make_float2(sum.m, sum.s);
  __syncthreads();
  {
    const float2 cell = cells[sub * (TPR / 32) + (t & 31) % (TPR / 32)];
    sum.m = cell.x;
    sum.s = cell.y;
    sum.across_lanes<TPR / 32>();
  }
#endif
#if CLUSTERED
  __shared__ float2 whole;
  if (threadIdx.x == 0) whole = make_float2(sum.m, sum.s);
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  {
    const float2 theirs = peer_pair(&whole, (threadIdx.x & 31) % PARTS);
    sum.m = theirs.x;
    sum.s = theirs.y;
    sum.across_lanes<PARTS>();
  }
  // nobody leaves while another CTA may still read its pair; waited for at the end
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
#endif
  const float m = sum.m, total = sum.s;
#endif
  const float log_prob = known ? log_prob_at(xt, m, total) : 0.0f;
#if LOG_PROB_OUT
  if (row_ok && part == 0 && t == 0) log_prob_out[r] = log_prob;
#endif
#if STATS_OUT
  if (row_ok && part == 0 && t == 0) stats[r] = make_float2(m, total);
#endif
#if GRADIENT
  SLOPE
  const Slope grad(m, total, slope, known, tok, xt, lead);
  GT* grow = G + r * VOCAB;
  for (int ck = 0; ck < CHUNKS; ++ck) {
#if STATS_IN || CHUNKS > 1
    load_chunk(mine, row, lead, vectors, j0, ck, raw);
#endif
    const int j1 = j0 + ck * (VPT * TPR);
    if (row_ok && inner_chunk(j1, lead) && !grad.special()) {
      GT* to = grow + ((long long)j1 * E - lead);
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float f[E];
        grad.of<false>(raw[i], f);
        store_vector(to + i * (TPR * E), f);
        grad.token(grow, j1 + i * TPR);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int j = j1 + i * TPR, first = j * E - lead;
        if (j >= vectors || !row_ok) continue;
        float f[E];
        grad.of<true>(raw[i], f);
        if (first >= 0 && first + E <= VOCAB) store_vector(grow + first, f);
        else store_edge(grow, first, f);
        grad.token(grow, j);
      }
    }
  }
#endif
#if CLUSTERED
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
#endif
}
)CUDA";

// The same for many long rows: persistent CTAs whose rows pass through a ring of shared-memory slots,
// filled by bulk copies ahead of use.  A producer warp runs through the rows of the CTA chunk by chunk, into the
// next row while the consumers are still at this one, so reads go on while the row's threads combine
// their sums and write the gradient.  The consumers fold each chunk as it arrives (every thread its own
// running maximum and sum) and keep the last HOLD chunks of the row in their slots; the gradient is
// computed from those, and then from the row's first chunks, which the producer brings once more (out
// of L2).  Chunks enter, are released and come back in the one order of the ring.
const char* kStreamTemplate = R"CUDA(
#define CHUNK_BYTES (CHUNK * 16)
#define PER_THREAD (CHUNK / CONSUMERS)
__device__ __forceinline__ unsigned int shared_at(const void* p) { return (unsigned int)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(shared_at(bar)) : "memory");
}
__device__ __forceinline__ bool passed(unsigned int bar, unsigned int parity) {
  unsigned int done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  return done != 0u;
}
#define MOST_TRIES (1u << 22)
// false when the wait gave up, here or elsewhere in the CTA; every warp looks at `gave_up` once more before it
// leaves, after its own last wait, and raises the status word
__device__ __forceinline__ bool wait_for(unsigned long long* bar, unsigned int parity, volatile int* gave_up) {
  const unsigned int a = shared_at(bar);
  for (unsigned int i = 0; i < MOST_TRIES; ++i) {
    if (passed(a, parity)) return true;
    if (*gave_up) return false;
  }
  *gave_up = 1;
  return false;
}
struct Place {   // a position of the ring: slot and the parity of its current use
  int slot;
  unsigned int parity;
  __device__ __forceinline__ void next() { if (++slot == SLOTS) { slot = 0; parity ^= 1u; } }
};
struct RowAt {
  const XT* row;
  int lead, vectors, chunks, held;
  // whether every vector of chunk c lies in the row
  __device__ __forceinline__ bool inner(int c) const {
    return VOCAB % E == 0 ? (c + 1) * CHUNK <= vectors : c > 0 && (c + 1) * CHUNK < vectors;
  }
};
__device__ __forceinline__ RowAt row_at(const XT* X, long long r) {
  RowAt w;
  w.row = X + r * VOCAB;
  w.lead = (int)(((unsigned long long)w.row & 15ull) / sizeof(XT));
  w.vectors = (w.lead + VOCAB + E - 1) / E;
  w.chunks = (w.vectors + CHUNK - 1) / CHUNK;
  w.held = w.chunks < HOLD ? w.chunks : HOLD;
  return w;
}
// vectors of the buffer that lie inside it altogether; the elements of a last partial one are read singly
#define WHOLE_VECTORS ((ROWS * (long long)VOCAB) / E)

__device__ __forceinline__ Raw slot_vector(const unsigned char* at) {
  const uint4 b = *reinterpret_cast<const uint4*>(at);
  Raw v;
  v.w[0] = b.x; v.w[1] = b.y; v.w[2] = b.z; v.w[3] = b.w;
  return v;
}
// vector j of a row's first or last chunk: elements outside the row as -inf
__device__ __forceinline__ Raw edge_vector(const XT* __restrict__ X, const RowAt& w, const unsigned char* at, int j) {
  Raw v;
  if (j >= w.vectors) {
#pragma unroll
    for (int q = 0; q < 4; ++q) v.w[q] = NEG_INF_WORD;
    return v;
  }
  v = slot_vector(at);
  const int first = j * E - w.lead;
  if (first < 0 || first + E > VOCAB) {
    const bool whole = (w.row - w.lead - X) / E + j < WHOLE_VECTORS;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const bool in = first + e >= 0 && first + e < VOCAB;
#if IN_BITS == 32
      v.w[e] = !in ? NEG_INF_WORD : whole ? v.w[e] : __float_as_uint(w.row[first + e]);
#else
      const unsigned int had = (e & 1) ? v.w[e / 2] >> 16 : v.w[e / 2] & 0xffffu;
      const unsigned int bits = !in ? NEG_INF_WORD & 0xffffu : whole ? had : (unsigned int)w.row[first + e];
      v.w[e / 2] = (e & 1) ? (v.w[e / 2] & 0xffffu) | (bits << 16) : (v.w[e / 2] & 0xffff0000u) | bits;
#endif
    }
  }
  return v;
}

extern "C" __global__ void __launch_bounds__(CONSUMERS + 32, CTAS_PER_SM)
KERNEL(const XT* __restrict__ X, const TT* __restrict__ T, float* __restrict__ log_prob_out, float2* __restrict__ stats, GT* __restrict__ G, int* __restrict__ status LEAF_PARAMS) {
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ __align__(8) unsigned long long full[SLOTS], empty[SLOTS];
  __shared__ float2 cells[2][CONSUMERS / 32];
  __shared__ int gave_up_cell;
  volatile int* gave_up = &gave_up_cell;
  const int t = threadIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (t == 0) {
    gave_up_cell = 0;
    for (int i = 0; i < SLOTS; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(shared_at(&full[i])));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(shared_at(&empty[i])), "r"(CONSUMERS / 32));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (warp == CONSUMERS / 32) {
    if (lane == 0) {
      Place at{0, 1u};   // the first use of a slot waits for nothing
      // chunks that will be read again stay in L2 if they can; nothing reads the others again
      unsigned long long keep, drop;
      asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(keep));
      asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(drop));
      long long issued = 0;
      bool ok = true;
      for (long long r = blockIdx.x; r < ROWS && ok; r += gridDim.x) {
        const RowAt w = row_at(X, r);
        const XT* base = w.row - w.lead;
        const int again = GRADIENT ? w.chunks - w.held : 0;
        for (int q = 0; q < w.chunks + again; ++q) {
          const int c = q < w.chunks ? q : q - w.chunks;
          ok = wait_for(&empty[at.slot], at.parity, gave_up);
          if (!ok) break;
          int n = w.vectors - c * CHUNK < CHUNK ? w.vectors - c * CHUNK : CHUNK;
          if (VOCAB % E != 0 && (base - X) / E + c * CHUNK + n > WHOLE_VECTORS) --n;
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(shared_at(&full[at.slot])), "r"(n * 16) : "memory");
          if (n > 0)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                         :: "r"(shared_at(ring + at.slot * CHUNK_BYTES)), "l"(base + (long long)c * CHUNK * E), "r"(n * 16), "r"(shared_at(&full[at.slot])), "l"(q < again ? keep : drop) : "memory");
          at.next();
          ++issued;
        }
      }
      // no copy may be in flight when the CTA leaves, whether the consumers still wait for it or have given up
      for (long long q = issued < SLOTS ? 0 : issued - SLOTS; q < issued; ++q) {
        const unsigned int a = shared_at(&full[q % SLOTS]), parity = (unsigned int)((q / SLOTS) & 1);
        unsigned int i = 0;
        while (i < MOST_TRIES && !passed(a, parity)) ++i;
        if (i == MOST_TRIES) *gave_up = 1;
      }
      if (*gave_up) atomicExch(status, 1);
    }
    return;
  }
  // Consumers.  After a wait that gave up they go on without waiting (the results are marked invalid by
  // the status word), so that every warp still meets the others at the row's barrier.
  Place at{0, 0u};
  int turn = 0;
  long long next_tok = (long long)T[blockIdx.x];   // read a row ahead: the token's logit is read at its address
  for (long long r = blockIdx.x; r < ROWS; r += gridDim.x) {
    const RowAt w = row_at(X, r);
    const long long tok = next_tok;
    if (r + gridDim.x < ROWS) next_tok = (long long)T[r + gridDim.x];
    const bool known = tok >= 0 && tok < VOCAB;
    LEAVES
    const float xt = known ? value_of(w.row[tok]) : 0.0f;
    Sum sum;
    Place kept = at;
    for (int c = 0; c < w.chunks; ++c) {
      if (c == w.chunks - w.held) kept = at;
      wait_for(&full[at.slot], at.parity, gave_up);
      const unsigned char* slot = ring + at.slot * CHUNK_BYTES + t * 16;
      Raw raw[PER_THREAD];
      if (w.inner(c)) {
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) raw[i] = slot_vector(slot + i * (CONSUMERS * 16));
      } else {
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) raw[i] = edge_vector(X, w, slot + i * (CONSUMERS * 16), c * CHUNK + i * CONSUMERS + t);
      }
      if (!GRADIENT || c < w.chunks - w.held) {
        __syncwarp();
        if (lane == 0) arrive(&empty[at.slot]);
      }
      at.next();
      sum.fold(raw);
    }
    sum.across_lanes<32>();
    if (lane == 0) cells[turn][warp] = make_float2(sum.m, sum.s);
    asm volatile("barrier.sync 1, %0;" :: "n"(CONSUMERS) : "memory");
    {
      const float2 mine = cells[turn][lane < CONSUMERS / 32 ? lane : 0];
      sum.m = mine.x;
      sum.s = lane < CONSUMERS / 32 ? mine.y : 0.0f;
      sum.across_lanes<32>();
    }
    turn ^= 1;   // the other cells next time: these may still be read
    const float m = sum.m, total = sum.s;
    const float log_prob = known ? log_prob_at(xt, m, total) : 0.0f;
#if LOG_PROB_OUT
    if (t == 0) log_prob_out[r] = log_prob;
#endif
#if STATS_OUT
    if (t == 0) stats[r] = make_float2(m, total);
#endif
#if GRADIENT
    SLOPE
    const Slope grad(m, total, slope, known, tok, xt, w.lead);
    const bool special = grad.special();
    GT* grow = G + r * VOCAB;
    for (int q = 0; q < w.chunks; ++q) {
      const bool held = q < w.held;
      const int c = held ? w.chunks - w.held + q : q - w.held;
      const int slot_number = held ? kept.slot : at.slot;
      if (!held) wait_for(&full[at.slot], at.parity, gave_up);
      const unsigned char* slot = ring + slot_number * CHUNK_BYTES + t * 16;
      const int j0 = c * CHUNK + t;
      const bool inner = w.inner(c);
      Raw raw[PER_THREAD];
      if (inner) {
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) raw[i] = slot_vector(slot + i * (CONSUMERS * 16));
      } else {
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) raw[i] = edge_vector(X, w, slot + i * (CONSUMERS * 16), j0 + i * CONSUMERS);
      }
      __syncwarp();
      if (lane == 0) arrive(&empty[slot_number]);
      if (held) kept.next();
      else at.next();
      GT* to = grow + (j0 * E - w.lead);
      if (inner && !special) {
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) {
          float f[E];
          grad.of<false>(raw[i], f);
          store_vector(to + i * (CONSUMERS * E), f);
          grad.token(grow, j0 + i * CONSUMERS);
        }
      } else {
#pragma unroll
        for (int i = 0; i < PER_THREAD; ++i) {
          const int j = j0 + i * CONSUMERS, first = j * E - w.lead;
          if (j >= w.vectors) continue;
          const bool whole = first >= 0 && first + E <= VOCAB;
          float f[E];
          if (whole && !special) grad.of<false>(raw[i], f);
          else grad.of<true>(raw[i], f);
          if (whole) store_vector(to + i * (CONSUMERS * E), f);
          else store_edge(grow, first, f);
          grad.token(grow, j);
        }
      }
    }
#endif
  }
  if (lane == 0 && *gave_up) atomicExch(status, 1);
}
)CUDA";

}  // namespace

void emitTokenLogProb(const TokenOp& op, const std::string& name, Plan& plan, const ScheduleOverrides& ov) {
  // Elements of a row are counted in 32 bits, up to the end of the last chunk of the last part: 64 parts of whole chunks of
  // 4096 vectors of 8 elements reach less than 2^21 elements past the row.
  if (op.vocab > 0x7fc00000ll) throw PlanError("token log-probabilities over more than 2^31 - 2^22 entries are not supported");
  const int in_size = static_cast<int>(dtypeSize(op.logits_dtype)), e = 16 / in_size;
  // aligned vectors that cover a row, wherever it starts
  const int64_t vectors = op.vocab % e == 0 ? op.vocab / e : (op.vocab + 2 * e - 2) / e;
  const bool stats_in = op.stats_in >= 0, gradient = op.grad_slot >= 0;
  const int64_t row_bytes = vectors * 16;
  const int most_threads = 512, most_vpt = 8;   // 64 KB: the row in one CTA's registers, two CTAs per SM
  // Rows beyond that, with enough of them, pass through shared memory (see kStreamTemplate).  Measured with the
  // gradient on bf16 4096 x 65536: 203 us, a cluster of two CTAs per row 233 us, chunks read twice 254 us; with 150 rows
  // the three are equal, with 64 the cluster is the fastest.
  bool stream = gradient && !stats_in && vectors > most_threads * most_vpt && op.rows >= 2 * ov.sm_count;
  int64_t parts = 1;
  int tpr = 32;
  int64_t vpt = most_vpt;
  int min_blocks = 0;
  if (stats_in) {
    while (parts < 64 && ceilDiv(vectors, parts) > 256 * 4) parts *= 2;
  } else if (gradient) {
    while (parts < 8 && vectors > parts * most_threads * most_vpt) parts *= 2;
    while (parts < 8 && op.rows * parts * 2 <= 2 * ov.sm_count && vectors >= parts * 2 * 256) parts *= 2;
  } else {
    // without a gradient nothing has to be held: a row is split only to fill the GPU (bf16 150 x 131072: 18.5 us in four
    // parts, 24.6 in one; 600 x 131072: 45 us in four, 37 in one)
    while (parts < 8 && op.rows * parts * 2 <= 5 * ov.sm_count && vectors >= parts * 2 * 256) parts *= 2;
  }
  const int64_t per = ceilDiv(vectors, parts);
  const bool few = op.rows * parts <= 2 * ov.sm_count;
  if (!gradient && !few && per > 256 * most_vpt) {
    // long rows in chunks of 16 KB, six CTAs of 256 threads per SM (bf16 4096 x 32768: 49 us, from registers with 512
    // threads 53 us; f16 4092 x 50001: 76 us with six CTAs, 84 us with four that read 32 KB at a time)
    tpr = 256;
    vpt = 4;
    min_blocks = 6;
  } else {
    while (tpr < most_threads && per > static_cast<int64_t>(tpr) * (few ? 2 : most_vpt)) tpr *= 2;
    vpt = std::min<int64_t>(most_vpt, ceilDiv(per, tpr));
  }
  const int64_t chunks = ceilDiv(per, tpr * vpt);
  int rpc = parts == 1 ? std::max(1, 256 / tpr) : 1;
  while (rpc > 1 && rpc / 2 >= op.rows) rpc /= 2;
  const int threads = tpr * rpc;
  const int64_t groups = ceilDiv(op.rows, rpc);
  if (groups * parts > 0x7fffffffll) throw PlanError("token log-probabilities of too many rows");

  const Pointwise slope{op.slope.nodes, op.slope.leaves, op.row_extents, static_cast<int>(op.row_extents.size()), 1, op.slope.acc, "log_prob", "n"};
  std::ostringstream o, loads, body;
  if (gradient) {
    // the buffers are read at the top of the kernel, the arithmetic waits for the log-probability
    for (size_t i = 0; i < slope.nodes.size(); ++i)
      slope.emit(static_cast<int>(i), slope.nodes[i].op == ENode::Leaf ? loads : body, "  ");
    body << "  const float slope = " << slope.name(op.slope.result) << ";\n";
  }
  o << kernelPrelude();
  define(o, "KERNEL", name);
  define(o, "XT", storageTypeOf(op.logits_dtype));
  define(o, "TT", storageTypeOf(op.token_dtype));
  define(o, "GT", storageTypeOf(op.grad_dtype));
  std::ostringstream l2e, scale, grad_scale;
  l2e << std::scientific << std::setprecision(16) << 1.4426950408889634 * static_cast<double>(op.scale) << "f";
  scale << std::scientific << std::setprecision(9) << op.scale << "f";
  grad_scale << std::scientific << std::setprecision(9) << op.grad_scale << "f";
  define(o, "L2E", l2e.str());
  define(o, "SCALE", scale.str());
  define(o, "GRAD_SCALE", grad_scale.str());
  define(o, "STORE(x)", storeConv(op.grad_dtype, "x"));
  define(o, "OUT_16", op.grad_dtype == DType::f32 ? "0" : "1");
  define(o, "OUT_16_NAME", op.grad_dtype == DType::bf16 ? "\"bf16\"" : "\"f16\"");
  define(o, "IN_BITS", num(8 * in_size));
  define(o, "IN_BF16", op.logits_dtype == DType::bf16 ? "1" : "0");
  define(o, "E", num(e));
  define(o, "ROWS", num(op.rows) + "ll");
  define(o, "VOCAB", num(op.vocab));
  define(o, "TPR", num(tpr));
  define(o, "RPC", num(rpc));
  define(o, "THREADS", num(threads));
  define(o, "MIN_BLOCKS", num(min_blocks ? min_blocks : std::max(1, 1024 / threads)));
  define(o, "VPT", num(vpt));
  define(o, "CHUNKS", num(chunks));
  define(o, "PARTS", num(parts));
  const bool clustered = parts > 1 && !stats_in;
  define(o, "CLUSTERED", clustered ? "1" : "0");
  define(o, "CLUSTER", clustered ? "__cluster_dims__(" + num(parts) + ", 1, 1)" : "");
  define(o, "STATS_IN", stats_in ? "1" : "0");
  define(o, "STATS_OUT", op.stats_out >= 0 ? "1" : "0");
  define(o, "LOG_PROB_OUT", op.log_prob_slot >= 0 ? "1" : "0");
  define(o, "GRADIENT", gradient ? "1" : "0");
  define(o, "LEAF_PARAMS", gradient ? slope.params() : "");
  // One CTA of up to 27 warps per SM with a ring of 216 KB for rows of which two smaller rings hold too little, two CTAs of up
  // to 16 warps with 112 KB each for shorter ones, whose own latencies then overlap (bf16 4096 x 50001: 176 us with two, 188
  // with one; f32 8192 x 32768: 377 and 340 us; bf16 8192 x 131072: 797 and 709 us).  16-bit logits ask for twice the
  // arithmetic per byte, so two CTAs serve them up to longer rows.  Two vectors per thread make a chunk, and a
  // row is cut into equal ones: a last chunk of a few vectors would take as long as a whole one (bf16 4096 x 50001 in seven
  // equal chunks 172 us).
  const bool wide_ring = row_bytes >= (in_size == 4 ? 112 : 160) * 1024;
  const int64_t ctas = wide_ring ? 1 : 2, ring_bytes = (wide_ring ? 216 : 112) * 1024, most_chunk = wide_ring ? 1728 : 1024;
  const int64_t chunk = ceilDiv(ceilDiv(vectors, ceilDiv(vectors, most_chunk)), 64) * 64, consumers = chunk / 2;
  const int64_t slots = ring_bytes / (chunk * 16), hold = slots - 1;
  // A gradient of which more than half is computed from logits read again is written past L2, where it would take
  // their place (f32 2048 x 150000: 522 and 481 us; bf16 8192 x 32768, nothing read again: 182 and 188 us).
  define(o, "WRITE(p, v)", stream && row_bytes > 2 * hold * chunk * 16 ? "__stcs(p, v)" : "*(p) = (v)");
  if (stream) {
    define(o, "SLOTS", num(slots));
    define(o, "CHUNK", num(chunk));
    define(o, "CONSUMERS", num(consumers));
    define(o, "CTAS_PER_SM", num(ctas));
    define(o, "HOLD", num(hold));
  }
  o << kTokenCommon;
  std::string text = stream ? kStreamTemplate : kTokenTemplate;
  text.replace(text.find("LEAVES\n"), 7, loads.str());
  text.replace(text.find("SLOPE\n"), 6, body.str());
  o << text;
  Launch l;
  l.kernel = addKernel(plan, name, "token_log_prob", o.str());
  l.grid[0] = static_cast<uint32_t>(groups * parts);
  l.block[0] = static_cast<uint32_t>(threads);
  l.label = name + " rows=" + num(op.rows) + " vocab=" + num(op.vocab);
  // a buffer that the kernel does not use is passed as the logits
  auto or_logits = [&](int slot) { return slotArg(slot >= 0 ? slot : op.logits_slot); };
  l.args.push_back(slotArg(op.logits_slot));
  l.args.push_back(slotArg(op.token_slot));
  l.args.push_back(or_logits(op.log_prob_slot));
  l.args.push_back(or_logits(stats_in ? op.stats_in : op.stats_out));
  l.args.push_back(or_logits(op.grad_slot));
  if (stream) {
    l.args.push_back(slotArg(-2));   // the session's device status word
    l.grid[0] = static_cast<uint32_t>(std::min<int64_t>(op.rows, ctas * ov.sm_count));
    l.block[0] = static_cast<uint32_t>(consumers + 32);
    l.dynamic_smem = static_cast<uint32_t>(slots * chunk * 16);
  }
  if (gradient)
    for (const LeafRef& leaf : op.slope.leaves) l.args.push_back(slotArg(leaf.slot));
  plan.launches.push_back(l);
}

}  // namespace accy
