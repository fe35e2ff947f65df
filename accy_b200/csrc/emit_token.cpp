// Kernels of the token side of a language model: scatter_add (the gradient of an embedding lookup) and
// the log-probabilities of given tokens with their gradient.  The lookup itself is no kernel of its own:
// a gather is an indirect row offset in whatever row kernel consumes it (emit_row.cpp).
#include <algorithm>
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

  void leafLoad(int i, std::ostream& o, const std::string& ind) const {
    const ENode& n = nodes[i];
    const LeafRef& l = leaves[n.leaf];
    const std::string L = "L" + num(n.leaf), ty = ctypeOf(n.dtype), st = storageTypeOf(l.dtype);
    const std::string row = indexExpr(extents, l.strides, 0, split, "r");
    if (!element(i)) {
      o << ind << "const " << ty << " " << name(i) << " = " << loadConv(l.dtype, L + "[" + row + "]") << ";\n";
      return;
    }
    o << ind << ty << " " << name(i) << "[" << vec << "];\n";
    if (vec > 1 && wide(l)) {
      o << ind << "{ const Pack<" << st << ", " << vec << "> p = *reinterpret_cast<const Pack<" << st << ", " << vec << ">*>(" << L
        << " + " << row << " + c0);\n" << ind << "#pragma unroll\n" << ind << "  for (int e = 0; e < " << vec << "; ++e) " << name(i)
        << "[e] = " << loadConv(l.dtype, "p.v[e]") << "; }\n";
    } else {
      o << ind << "#pragma unroll\n" << ind << "for (int e = 0; e < " << vec << "; ++e) " << name(i) << "[e] = "
        << loadConv(l.dtype, L + "[" + row + " + " + indexExpr(extents, l.strides, split, rank(), "(c0 + e)") + "]") << ";\n";
    }
  }

  void emit(int i, std::ostream& o, const std::string& ind) const {
    const ENode& n = nodes[i];
    const std::string ty = ctypeOf(n.dtype);
    if (i == acc) return;
    if (n.op == ENode::Leaf) return leafLoad(i, o, ind);
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
//   order  one cluster of eight CTAs sorts by least significant digits, its CTAs exchanging digit counts
//          through distributed shared memory; meanwhile the other CTAs write the rows that no index
//          names, which for a large vocabulary is most of the traffic;
//   sum    one CTA per (piece of the list, block of columns): a thread holds its columns' running sum in
//          registers (f32 or wider), and writes a row when the run ends.  Runs that cross the ends of a
//          piece leave partial sums;
//   join   adds the partial sums of the runs that cross, in order.
// The floor is memory: updates once, rows once.
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
__device__ __forceinline__ unsigned int row_of(IT x) {
  const long long v = (long long)x;
  return v >= 0 && v < EXTENT ? (unsigned int)v : (unsigned int)EXTENT;
}

// Rows [lo, hi) that no index names: zeros, or the base's row.
__device__ __forceinline__ void fill_rows(const IT* __restrict__ I, OT* __restrict__ out, BASE_PARAM_ long long lo, long long hi, unsigned int* bits) {
  for (long long at = lo; at < hi; at += FILL_ROWS) {
    const long long end = at + FILL_ROWS < hi ? at + FILL_ROWS : hi;
    __syncthreads();
    for (int w = threadIdx.x; w < FILL_ROWS / 32; w += THREADS) bits[w] = 0u;
    __syncthreads();
#pragma unroll 4
    for (long long i = threadIdx.x; i < COUNT; i += THREADS) {
      const long long v = (long long)I[i];
      if (v >= at && v < end) atomicOr(&bits[(v - at) >> 5], 1u << ((v - at) & 31));
    }
    __syncthreads();
    const long long vectors = (end - at) * (POST / FVEC);
    for (long long p = 0; p < PRE; ++p) {
      for (long long q = threadIdx.x; q < vectors; q += THREADS) {
        const long long v = q / (POST / FVEC), c = (q - v * (POST / FVEC)) * FVEC;
        if (bits[v >> 5] >> (v & 31) & 1u) continue;
        const long long off = (p * EXTENT + at + v) * POST + c;
        Pack<OT, FVEC> o;
#pragma unroll
        for (int e = 0; e < FVEC; ++e) o.v[e] = FILL_VALUE(off + e);
        *reinterpret_cast<Pack<OT, FVEC>*>(out + off) = o;
      }
    }
  }
}

extern "C" __global__ void __cluster_dims__(8, 1, 1) __launch_bounds__(THREADS)
KERNEL(const IT* __restrict__ I, unsigned int* key_a, unsigned int* pos_a, unsigned int* key_b, unsigned int* pos_b, OT* __restrict__ out BASE_PARAM) {
  __shared__ unsigned int hist[WARPS][RADIX];
  __shared__ unsigned int total[RADIX], start[RADIX], wsum[WARPS], bits[FILL_ROWS / 32];
  if (blockIdx.x >= 8) {   // whole clusters take this branch
    const long long f = blockIdx.x - 8, per = (EXTENT + FILLERS - 1) / FILLERS;
    const long long lo = f * per, hi = lo + per < EXTENT ? lo + per : EXTENT;
    fill_rows(I, out, BASE_ARG_ lo, hi, bits);
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned int cta = blockIdx.x;
  // every warp owns one run of places, in order: that is what keeps the sort stable
  const long long slice = ((COUNT + 8 * WARPS * 32 - 1) / (8 * WARPS * 32)) * 32;
  const long long w0 = ((long long)cta * WARPS + warp) * slice, w1 = w0 + slice < COUNT ? w0 + slice : COUNT;
  for (int pass = 0; pass < PASSES; ++pass) {
    // the last pass writes the (a) arrays
    const bool to_a = ((PASSES - 1 - pass) & 1) == 0;
    const unsigned int *ks = to_a ? key_b : key_a, *ps = to_a ? pos_b : pos_a;
    unsigned int *kd = to_a ? key_a : key_b, *pd = to_a ? pos_a : pos_b;
    const int shift = pass * DIGIT_BITS;
    for (int d = threadIdx.x; d < WARPS * RADIX; d += THREADS) (&hist[0][0])[d] = 0u;
    __syncthreads();
    for (long long i = w0 + lane; i - lane < w1; i += 32) {
      const bool in = i < w1;
      unsigned int d = RADIX;
      if (in) d = ((pass == 0 ? row_of(I[i]) : __ldcg(ks + i)) >> shift) & (RADIX - 1);
      const unsigned int peers = __match_any_sync(0xffffffffu, d);
      if (in && lane == __ffs(peers) - 1) hist[warp][d] += __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < RADIX) {
      unsigned int sum = 0u;
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
    for (long long i = w0 + lane; i - lane < w1; i += 32) {
      const bool in = i < w1;
      unsigned int k = 0u, ps_i = 0u, d = RADIX;
      if (in) {
        k = pass == 0 ? row_of(I[i]) : __ldcg(ks + i);
        ps_i = pass == 0 ? (unsigned int)i : __ldcg(ps + i);
        d = (k >> shift) & (RADIX - 1);
      }
      const unsigned int peers = __match_any_sync(0xffffffffu, d);
      if (in) {
        const unsigned int to = start[d] + hist[warp][d] + __popc(peers & ((1u << lane) - 1u));
        kd[to] = k;
        pd[to] = ps_i;
      }
      __syncwarp();
      if (in && lane == __ffs(peers) - 1) hist[warp][d] += __popc(peers);
      __syncwarp();
    }
    cluster_sync();   // the lists are complete, and nobody reads this pass's counts any more
  }
}
)CUDA";

const char* kSumHead = R"CUDA(
__device__ __forceinline__ void write_row(OT* __restrict__ out, BASE_PARAM_ long long off, const VT (&sum)[VEC]) {
  Pack<OT, VEC> o;
#pragma unroll
  for (int e = 0; e < VEC; ++e) o.v[e] = WITH_BASE(off + e, sum[e]);
  *reinterpret_cast<Pack<OT, VEC>*>(out + off) = o;
}
)CUDA";

const char* kSumBody = R"CUDA(
  __shared__ unsigned int key[PIECE + 2], pos[PIECE];
  const long long begin = (long long)blockIdx.x * PIECE;
  const int n = COUNT - begin < PIECE ? (int)(COUNT - begin) : PIECE;
  // key[0] and key[n + 1] are the neighbours' keys; EXTENT + 1 stands for none
  for (int i = threadIdx.x; i < n + 2; i += THREADS) {
    const long long at = begin + i - 1;
    key[i] = at >= 0 && at < COUNT ? keys[at] : (unsigned int)EXTENT + 1u;
    if (i < n) pos[i] = places[begin + i];
  }
  __syncthreads();
  const long long c0 = ((long long)blockIdx.y * THREADS + threadIdx.x) * VEC;
  if (c0 >= POST) return;
  const long long p = blockIdx.z;
  VT sum[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[e] = 0;
  bool first = true;   // the run that starts this piece
  for (int i = 0; i < n; i += AHEAD) {
    VT u[AHEAD][VEC];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i + a >= n || key[i + a + 1] >= (unsigned int)EXTENT) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) u[a][e] = 0;
        continue;
      }
      const long long r = p * COUNT + pos[i + a];
      (void)r;
      UPDATE
    }
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (i + a >= n) break;
      const unsigned int k = key[i + a + 1];
      if (k >= (unsigned int)EXTENT) return;   // indices outside the axis come last
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] = sum[e] + u[a][e];
      const bool last = i + a + 1 == n;
      if (!last && key[i + a + 2] == k) continue;
      // the run ends here, or the piece does
      const bool from_before = first && key[0] == k, goes_on = last && key[n + 1] == k;
      if (from_before || goes_on) {
        Pack<VT, VEC> part;
#pragma unroll
        for (int e = 0; e < VEC; ++e) part.v[e] = sum[e];
        *reinterpret_cast<Pack<VT, VEC>*>(partial + ((p * PIECES + blockIdx.x) * 2 + (from_before ? 0 : 1)) * POST + c0) = part;
      } else {
        write_row(out, BASE_ARG_ (p * EXTENT + k) * POST + c0, sum);
      }
      first = false;
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] = 0;
    }
  }
}
)CUDA";

const char* kJoinBody = R"CUDA(
  const long long piece = blockIdx.x, begin = piece * PIECE, end = begin + PIECE;
  if (end >= COUNT) return;
  const unsigned int k = keys[end - 1];
  // the run at the end of this piece goes on, and began in it
  if (k >= (unsigned int)EXTENT || keys[end] != k) return;
  if (begin > 0 && keys[begin - 1] == k) return;
  // how many of the following pieces begin with it: they are next to each other
  long long more = 0;
  for (;;) {
    const long long at = (piece + 1 + more + threadIdx.x) * PIECE;
    const int here = __syncthreads_count(at < COUNT && keys[at] == k);
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
#pragma unroll 8
  for (long long m = 1; m <= more; ++m) {
    const Pack<VT, VEC> part = *reinterpret_cast<const Pack<VT, VEC>*>(from + m * 2 * POST);
#pragma unroll
    for (int e = 0; e < VEC; ++e) sum[e] = sum[e] + part.v[e];
  }
  write_row(out, BASE_ARG_ (p * EXTENT + k) * POST + c0, sum);
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
  const int passes = static_cast<int>(ceilDiv(bits, 8)), digit_bits = static_cast<int>(ceilDiv(bits, passes));
  const int64_t out_bytes = s.pre * s.extent * s.post * static_cast<int64_t>(dtypeSize(s.out_dtype));
  const int64_t fillers = 8 * std::max<int64_t>(1, std::min<int64_t>(ceilDiv(out_bytes, 8 * 65536), ceilDiv(2 * ov.sm_count, 8)));

  const int threads = static_cast<int>(std::min<int64_t>(256, ceilDiv(ceilDiv(s.post, vec), 32) * 32));
  const int64_t blocks = ceilDiv(s.post, static_cast<int64_t>(threads) * vec);
  if (blocks > 65535) throw PlanError("scatter_add rows are too long");
  // about eight CTAs per SM; longer pieces leave fewer partial sums
  int64_t piece = 8;
  while (piece < 128 && ceilDiv(s.count, piece * 2) * blocks * s.pre >= 8 * ov.sm_count) piece *= 2;
  const int64_t pieces = ceilDiv(s.count, piece);

  const int key_a = scratchSlot(plan, s.count * 4), pos_a = scratchSlot(plan, s.count * 4);
  const int key_b = scratchSlot(plan, s.count * 4), pos_b = scratchSlot(plan, s.count * 4);
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
    define(o, "WARPS", "16");
    define(o, "PASSES", num(passes));
    define(o, "DIGIT_BITS", num(digit_bits));
    define(o, "RADIX", num(1 << digit_bits));
    define(o, "FILLERS", num(fillers) + "ll");
    define(o, "FILL_ROWS", "32768");
    define(o, "FVEC", num(fvec));
    o << kOrderTemplate;
    Launch l;
    l.kernel = addKernel(plan, name + "_order", "scatter_add", o.str());
    l.grid[0] = static_cast<uint32_t>(8 + fillers);
    l.block[0] = 512;
    l.label = name + " order";
    for (int slot : {s.index_slot, key_a, pos_a, key_b, pos_b, s.out_slot}) l.args.push_back(slotArg(slot));
    if (s.base_slot >= 0) l.args.push_back(slotArg(s.base_slot));
    plan.launches.push_back(l);
  }
  auto sumHead = [&](std::ostream& o, const char* kernel, const std::string& more) {
    head(o);
    define(o, "THREADS", num(threads));
    define(o, "VEC", num(vec));
    define(o, "PIECE", num(piece));
    define(o, "PIECES", num(pieces) + "ll");
    define(o, "AHEAD", "4");
    o << kSumHead << "extern \"C\" __global__ void __launch_bounds__(" << threads << ") " << name << kernel
      << "(const unsigned int* __restrict__ keys, const unsigned int* __restrict__ places, " << vt << "* __restrict__ partial, " << ot
      << "* __restrict__ out BASE_PARAM" << more << ") {\n";
  };
  auto sumLaunch = [&](int kernel, const char* what) {
    Launch l;
    l.kernel = kernel;
    l.grid[0] = static_cast<uint32_t>(pieces);
    l.grid[1] = static_cast<uint32_t>(blocks);
    l.grid[2] = static_cast<uint32_t>(s.pre);
    l.block[0] = static_cast<uint32_t>(threads);
    l.label = name + what;
    for (int slot : {key_a, pos_a, partial, s.out_slot}) l.args.push_back(slotArg(slot));
    if (s.base_slot >= 0) l.args.push_back(slotArg(s.base_slot));
    return l;
  };
  {
    Pointwise g{s.updates.nodes, s.updates.leaves, s.updates.extents, s.updates.split, vec, -1, "", "n"};
    std::ostringstream o, update;
    for (size_t i = 0; i < g.nodes.size(); ++i) g.emit(static_cast<int>(i), update, "      ");
    update << "#pragma unroll\n      for (int e = 0; e < VEC; ++e) u[a][e] = " << g.at(s.result) << ";\n";
    sumHead(o, "_sum", g.params());
    std::string body = kSumBody;
    body.replace(body.find("UPDATE"), 6, update.str());
    o << body;
    Launch l = sumLaunch(addKernel(plan, name + "_sum", "scatter_add", o.str()), " sum");
    for (const LeafRef& leaf : s.updates.leaves) l.args.push_back(slotArg(leaf.slot));
    plan.launches.push_back(l);
  }
  if (pieces > 1) {
    std::ostringstream o;
    sumHead(o, "_join", "");
    o << "  (void)places;\n" << kJoinBody;
    plan.launches.push_back(sumLaunch(addKernel(plan, name + "_join", "scatter_add", o.str()), " join"));
  }
}

// ---------------------------------------------------------------------------------------------
// log-probabilities of tokens
// ---------------------------------------------------------------------------------------------
namespace {

// One row of logits per TPR threads (CL CTAs of a cluster share a long row).  A thread loads its part of
// the row once, folds its maximum m and its sum of 2^((x - m) log2 e), and the row's (m, sum) pairs are
// combined through shuffles, shared memory and, in a cluster, distributed shared memory:
//
//   log p = (x[token] - m) - log(sum)         d log p / d x[v] = 1[v = token] - 2^((x[v] - m) log2 e) / sum
//
// The gradient is written from the registers that hold the row, so logits are read once and the gradient
// written once; the slope of each row (what the recorded program does to its log-probability on the
// way to the loss) is evaluated in between.  Rows need not be aligned: a row is covered by aligned
// 16-byte vectors, and the elements of the first and last one that belong to its neighbours are left out.
const char* kTokenTemplate = R"CUDA(
#define L2E 1.4426950408889634f
__device__ __forceinline__ float2 peer_pair(const float2* p, unsigned int cta) {
  const unsigned int a = (unsigned int)__cvta_generic_to_shared(p);
  unsigned int b;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(cta));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(b) : "memory");
  return v;
}
__device__ __forceinline__ float finite_or_zero_ref(float m) { return m == __uint_as_float(0xff800000u) ? 0.0f : m; }
// the sum `s` relative to the maximum m, seen relative to `ref`
__device__ __forceinline__ float rescaled(float s, float m, float ref) { return s * ex2_ftz((m - ref) * L2E); }

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

struct Raw { unsigned int w[4]; };

__device__ __forceinline__ void unpack(const Raw& v, float (&f)[E]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#if IN_BITS == 32
    f[i] = __uint_as_float(v.w[i]);
#elif IN_BF16
    f[2 * i] = __uint_as_float(v.w[i] << 16);
    f[2 * i + 1] = __uint_as_float(v.w[i] & 0xffff0000u);
#else
    f[2 * i] = f16_to_f32((unsigned short)(v.w[i] & 0xffffu));
    f[2 * i + 1] = f16_to_f32((unsigned short)(v.w[i] >> 16));
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
// vector j of a row whose first element is element `lead` of its first aligned vector; elements outside
// the row read as -inf
__device__ __forceinline__ Raw load_vector(const XT* __restrict__ row, int lead, int j) {
  Raw v;
  const int first = j * E - lead;
  if (first >= 0 && first + E <= VOCAB) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]) : "l"(row + first));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v.w[i] = NEG_INF_WORD;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (first + e < 0 || first + e >= VOCAB) continue;
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
  const float xt = known ? value_of(row[tok]) : 0.0f;
  Raw raw[VPT];
#if STATS_IN
  const float2 kept = stats[r];
  const float ref = kept.x, total = kept.y;
#else
  float m = __uint_as_float(0xff800000u), s = 0.0f;
  for (int ck = 0; ck < CHUNKS; ++ck) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = j0 + (ck * VPT + i) * TPR;
      if (j < vectors) raw[i] = load_vector(row, lead, j);
      else {
#pragma unroll
        for (int w = 0; w < 4; ++w) raw[i].w[w] = NEG_INF_WORD;
      }
    }
    unsigned int top = NEG_INF_WORD;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) top = packed_max(top, raw[i].w[w]);
#if IN_BITS == 32
    const float m2 = fmaxf(m, __uint_as_float(top));
#else
    const float m2 = fmaxf(m, fmaxf(value_of((XT)(top & 0xffffu)), value_of((XT)(top >> 16))));
#endif
    const float ref2 = finite_or_zero_ref(m2);
    if (CHUNKS > 1) s = rescaled(s, m, ref2);
    m = m2;
    unsigned long long acc = pk2(s, 0.0f);
    const unsigned long long minus = pk2(-ref2, -ref2), scale = pk2(L2E, L2E);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float f[E];
      unpack(raw[i], f);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float a, b;
        upk2(mul2(add2(pk2(f[e], f[e + 1]), minus), scale), a, b);
        acc = add2(acc, pk2(ex2_ftz(a), ex2_ftz(b)));
      }
    }
    float lo, hi;
    upk2(acc, lo, hi);
    s = lo + hi;
  }
  // the row's threads: lanes, then warps, then CTAs
  constexpr int W = TPR < 32 ? TPR : 32;
  {
    float top = m;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off, W));
    const float ref2 = finite_or_zero_ref(top);
    s = rescaled(s, m, ref2);
    m = top;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off, W);
  }
#if TPR > 32
  __shared__ float2 cells[RPC * (TPR / 32)];
  if ((t & 31) == 0) cells[sub * (TPR / 32) + (t >> 5)] = make_float2(m, s);
  __syncthreads();
  {
    float top = __uint_as_float(0xff800000u);
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) top = fmaxf(top, cells[sub * (TPR / 32) + w].x);
    const float ref2 = finite_or_zero_ref(top);
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) {
      const float2 c = cells[sub * (TPR / 32) + w];
      sum += rescaled(c.y, c.x, ref2);
    }
    m = top;
    s = sum;
  }
#endif
#if CLUSTERED
  __shared__ float2 mine;
  if (threadIdx.x == 0) mine = make_float2(m, s);
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
  {
    float2 c[PARTS];
    float top = __uint_as_float(0xff800000u);
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      c[q] = peer_pair(&mine, q);
      top = fmaxf(top, c[q].x);
    }
    const float ref2 = finite_or_zero_ref(top);
    float sum = 0.0f;
#pragma unroll
    for (int q = 0; q < PARTS; ++q) sum += rescaled(c[q].y, c[q].x, ref2);
    m = top;
    s = sum;
  }
  // nobody leaves while another CTA may still read its pair; waited for at the end
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
#endif
  const float ref = finite_or_zero_ref(m), total = s;
#endif
  const float log_prob = known ? (xt - ref) - logf(total) : 0.0f;
#if LOG_PROB_OUT
  if (row_ok && part == 0 && t == 0) log_prob_out[r] = log_prob;
#endif
#if STATS_OUT
  if (row_ok && part == 0 && t == 0) stats[r] = make_float2(ref, total);
#endif
#if GRADIENT
  SLOPE
  const float g = known ? slope : 0.0f;
  // a row that the loss does not depend on is zero whatever its logits hold
  const bool none = g == 0.0f;
  const float k = -g / total;
  const int at = known ? (int)tok : -1;
  GT* grow = G + r * VOCAB;
  const unsigned long long minus_ref = pk2(-ref, -ref), log2e = pk2(L2E, L2E), kk = pk2(k, k);
  for (int ck = 0; ck < CHUNKS; ++ck) {
#if STATS_IN || CHUNKS > 1
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = j0 + (ck * VPT + i) * TPR;
      if (j < vectors) raw[i] = load_vector(row, lead, j);
    }
#endif
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int j = j0 + (ck * VPT + i) * TPR;
      if (j >= vectors || !row_ok) continue;
      const int first = j * E - lead;
      float f[E];
      unpack(raw[i], f);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float a, b;
        upk2(mul2(add2(pk2(f[e], f[e + 1]), minus_ref), log2e), a, b);
        upk2(mul2(pk2(ex2_ftz(a), ex2_ftz(b)), kk), f[e], f[e + 1]);
      }
      if (none) {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = 0.0f;
      } else if (at >= first && at < first + E) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (first + e == at) f[e] += g;
      }
      Pack<GT, E> out;
#pragma unroll
      for (int e = 0; e < E; ++e) out.v[e] = STORE(f[e]);
      if (first >= 0 && first + E <= VOCAB) {
        *reinterpret_cast<Pack<GT, E>*>(grow + first) = out;
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (first + e >= 0 && first + e < VOCAB) grow[first + e] = out.v[e];
      }
    }
  }
#endif
#if CLUSTERED
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
#endif
}
)CUDA";

}  // namespace

void emitTokenLogProb(const TokenOp& op, const std::string& name, Plan& plan, const ScheduleOverrides& ov) {
  if (op.vocab > 0x7fff0000ll) throw PlanError("token log-probabilities over more than 2^31 - 65536 entries are not supported");
  const int in_size = static_cast<int>(dtypeSize(op.logits_dtype)), e = 16 / in_size;
  // aligned vectors that cover a row, wherever it starts
  const int64_t vectors = op.vocab % e == 0 ? op.vocab / e : (op.vocab + 2 * e - 2) / e;
  const bool stats_in = op.stats_in >= 0, gradient = op.grad_slot >= 0;
  const int most_threads = 512, most_vpt = 8;
  int64_t parts = 1;
  if (stats_in) {
    while (parts < 64 && ceilDiv(vectors, parts) > 256 * 4) parts *= 2;
  } else {
    // a row that one CTA's registers cannot hold is shared by the CTAs of a cluster; so is any row of more than a few
    // KB while there are too few rows to fill the GPU
    while (parts < 8 && vectors > parts * most_threads * most_vpt) parts *= 2;
    while (parts < 8 && op.rows * parts * 2 <= 2 * ov.sm_count && vectors >= parts * 2 * 256) parts *= 2;
  }
  const int64_t per = ceilDiv(vectors, parts);
  int tpr = 32;
  while (tpr < most_threads && per > static_cast<int64_t>(tpr) * (op.rows * parts <= 2 * ov.sm_count ? 2 : most_vpt)) tpr *= 2;
  int64_t vpt = std::min<int64_t>(most_vpt, ceilDiv(per, tpr));
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
  define(o, "STORE(x)", storeConv(op.grad_dtype, "x"));
  define(o, "IN_BITS", num(8 * in_size));
  define(o, "IN_BF16", op.logits_dtype == DType::bf16 ? "1" : "0");
  define(o, "E", num(e));
  define(o, "ROWS", num(op.rows) + "ll");
  define(o, "VOCAB", num(op.vocab));
  define(o, "TPR", num(tpr));
  define(o, "RPC", num(rpc));
  define(o, "THREADS", num(threads));
  define(o, "MIN_BLOCKS", num(std::max(1, 1024 / threads)));
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
  std::string text = kTokenTemplate;
  text.replace(text.find("  LEAVES\n"), 9, loads.str());
  text.replace(text.find("  SLOPE\n"), 8, body.str());
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
  if (gradient)
    for (const LeafRef& leaf : op.slope.leaves) l.args.push_back(slotArg(leaf.slot));
  plan.launches.push_back(l);
}

}  // namespace accy
