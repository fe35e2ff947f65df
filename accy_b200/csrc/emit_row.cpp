// CUDA source emission for row kernels: fused elementwise -> named-axis reductions.
//
// One generated kernel evaluates a whole expression DAG over the space [rows | cols]:
//   * TPR threads cooperate on a row, RPC rows share a CTA; every access along the column axis is
//     a VEC-element vector (128-bit when layouts allow), VPT vectors per thread per chunk;
//   * when a row fits one chunk it is loaded once and stays in registers through every reduction
//     and the final store (the B200 form of the reference's row pipeline, row.zig:556-668);
//   * longer rows stream chunk by chunk, one pass per reduction level (the reference's fused
//     reduction prologue, reduction.zig:755-879, with 128-bit loads);
//   * a reduction folds per thread, then by warp shuffle, then across warps through shared
//     memory in a fixed order; when rows are too few to fill the GPU the columns are split over
//     several CTAs whose partials a second kernel folds in index order (deterministic two-pass
//     combine; never atomics, unlike reduction.zig:939-991).
// f32 arithmetic is emitted one operation at a time and compiled with --fmad=false so that each
// op rounds separately, as the reference's CPU code does (x64/scalar.zig:310, no FMA contraction).
#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <map>
#include <set>
#include <sstream>

#include "plan.hpp"

namespace accy {

const char* ctypeOf(DType d) {
  switch (d) {
    case DType::i1: return "bool";
    case DType::i8: return "signed char";
    case DType::i16: return "short";
    case DType::i32: return "int";
    case DType::i64: return "long long";
    case DType::u8: return "unsigned char";
    case DType::u16: return "unsigned short";
    case DType::u32: return "unsigned int";
    case DType::u64: return "unsigned long long";
    case DType::f16: case DType::bf16: case DType::f32: return "float";
    case DType::f64: return "double";
    case DType::key: return "unsigned long long";
  }
  return "float";
}

const char* storageTypeOf(DType d) {
  switch (d) {
    case DType::f16: case DType::bf16: return "unsigned short";
    case DType::i1: return "unsigned char";
    default: return ctypeOf(d);
  }
}

static bool isFloatReg(DType d) { return d == DType::f16 || d == DType::bf16 || d == DType::f32; }

static std::string hex(uint64_t v) {
  std::ostringstream s;
  s << "0x" << std::hex << v;
  return s.str();
}

static float halfBitsToFloat(uint16_t h) {
  uint32_t sign = (h & 0x8000u) << 16, exp = (h >> 10) & 0x1f, man = h & 0x3ffu, out;
  if (exp == 0) {
    if (man == 0) out = sign;
    else {
      int e = -1;
      do { ++e; man <<= 1; } while (!(man & 0x400u));
      out = sign | ((127 - 15 - e) << 23) | ((man & 0x3ffu) << 13);
    }
  } else if (exp == 31) out = sign | 0x7f800000u | (man << 13);
  else out = sign | ((exp - 15 + 127) << 23) | (man << 13);
  float f;
  std::memcpy(&f, &out, 4);
  return f;
}

std::string constLiteral(const ENode& n) {
  switch (n.dtype) {
    case DType::f32: return "__uint_as_float(" + hex(n.bits & 0xffffffffu) + "u)";
    case DType::bf16: return "__uint_as_float(" + hex((n.bits & 0xffffu) << 16) + "u)";
    case DType::f16: {
      float f = halfBitsToFloat(static_cast<uint16_t>(n.bits));
      uint32_t b;
      std::memcpy(&b, &f, 4);
      return "__uint_as_float(" + hex(b) + "u)";
    }
    case DType::f64: return "__longlong_as_double(" + hex(n.bits) + "ll)";
    case DType::i1: return (n.bits & 0xff) ? "true" : "false";
    case DType::i8: return "((signed char)" + std::to_string(static_cast<int>(static_cast<int8_t>(n.bits))) + ")";
    case DType::i16: return "((short)" + std::to_string(static_cast<int>(static_cast<int16_t>(n.bits))) + ")";
    case DType::i32: return "((int)" + hex(n.bits & 0xffffffffu) + "u)";
    case DType::i64: return "((long long)" + hex(n.bits) + "ull)";
    case DType::u8: return "((unsigned char)" + std::to_string(n.bits & 0xff) + ")";
    case DType::u16: return "((unsigned short)" + std::to_string(n.bits & 0xffff) + ")";
    case DType::u32: return hex(n.bits & 0xffffffffu) + "u";
    default: return hex(n.bits) + "ull";
  }
}

// One elementwise operation on already-evaluated operands (elementwise.zig:1687-1719 lists the
// same op set).  max/min keep the x86 maxss/minss operand order of the reference's CPU code
// (x64/scalar.zig:689,696): the second operand wins when either is NaN.
std::string elementwiseExpr(const ENode& n, const std::string& a, const std::string& b,
                            const std::string& c, DType a_dtype) {
  const bool f64 = a_dtype == DType::f64;
  const bool flt = isFloatReg(a_dtype) || f64;
  const char* sfx = f64 ? "" : "f";
  switch (n.op) {
    case ENode::Un:
      switch (static_cast<Unary>(n.sub)) {
        case Unary::neg: return "(-" + a + ")";
        case Unary::abs: return flt ? std::string("fabs") + sfx + "(" + a + ")" : "(" + a + " < 0 ? -" + a + " : " + a + ")";
        case Unary::exp: return std::string("exp") + sfx + "(" + a + ")";
        case Unary::log: return std::string("log") + sfx + "(" + a + ")";
        case Unary::sqrt: return std::string("sqrt") + sfx + "(" + a + ")";
        case Unary::tanh: return std::string("tanh") + sfx + "(" + a + ")";
        case Unary::sin: return std::string("sin") + sfx + "(" + a + ")";
        case Unary::cos: return std::string("cos") + sfx + "(" + a + ")";
        case Unary::tan: return std::string("tan") + sfx + "(" + a + ")";
      }
      break;
    case ENode::Bin:
      switch (static_cast<Binary>(n.sub)) {
        case Binary::add: return "(" + a + " + " + b + ")";
        case Binary::sub: return "(" + a + " - " + b + ")";
        case Binary::mul: return "(" + a + " * " + b + ")";
        case Binary::div: return "(" + a + " / " + b + ")";
        case Binary::max: return "(" + a + " > " + b + " ? " + a + " : " + b + ")";
        case Binary::min: return "(" + a + " < " + b + " ? " + a + " : " + b + ")";
        case Binary::pow:
          if (!flt) throw PlanError("pow on integer values is not supported by the B200 target");
          return std::string("pow") + sfx + "(" + a + ", " + b + ")";
      }
      break;
    case ENode::Cmp:
      switch (static_cast<Compare>(n.sub)) {
        case Compare::lt: return "(" + a + " < " + b + ")";
        case Compare::le: return "(" + a + " <= " + b + ")";
        case Compare::gt: return "(" + a + " > " + b + ")";
        case Compare::ge: return "(" + a + " >= " + b + ")";
        case Compare::eq: return "(" + a + " == " + b + ")";
        case Compare::ne: return "(" + a + " != " + b + ")";
      }
      break;
    case ENode::Sel:
      return "(" + a + " ? " + b + " : " + c + ")";
    default:
      break;
  }
  throw PlanError("internal: not an elementwise node");
}

static const char* kRowPrelude = R"CUDA(
// ---- helpers shared by every generated row kernel ----
template <typename T, int N> struct __align__(sizeof(T) * N) Pack { T v[N]; };
__device__ __forceinline__ float bf16_to_f32(unsigned short h) { return __uint_as_float(((unsigned int)h) << 16); }
__device__ __forceinline__ unsigned short f32_to_bf16(float f) { unsigned short r; asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r) : "f"(f)); return r; }
__device__ __forceinline__ float f16_to_f32(unsigned short h) { float f; asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"(h)); return f; }
__device__ __forceinline__ unsigned short f32_to_f16(float f) { unsigned short r; asm("cvt.rn.f16.f32 %0, %1;" : "=h"(r) : "f"(f)); return r; }
// packed f32x2 arithmetic (sm_100): two IEEE f32 operations per instruction
__device__ __forceinline__ unsigned long long pk2(float lo, float hi) { unsigned long long r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ void upk2(unsigned long long v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) { unsigned long long r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ unsigned long long sub2(unsigned long long a, unsigned long long b) { unsigned long long r; asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) { unsigned long long r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// A recorded multiply keeps its own rounding.  The assembler was measured to merge mul.rn.f32x2
// with a following add.rn.f32x2 into one packed FMA (one rounding instead of two) even with FMA
// contraction off, and also when the multiply is written as fma(a, b, -0).  The product of a
// recorded multiply is therefore passed through an exclusive-or with a zero the assembler cannot
// see through (the kernel's last argument, which the host always passes as 0), which costs one
// integer instruction per pair.
__device__ __forceinline__ unsigned long long mul2_own_rounding(unsigned long long a, unsigned long long b, unsigned long long zero) { return mul2(a, b) ^ zero; }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) { unsigned long long r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ float ex2_ftz(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <int OP, typename T> __device__ __forceinline__ T fold(T a, T b) {
  if (OP == 0) return a + b;
  if (OP == 1) return a > b ? a : b;
  return a < b ? a : b;
}
// Reduction across the TPR threads of one row: butterfly shuffles inside a warp (every lane ends
// with the same bits), then one shared-memory cell per warp, folded in warp order by every thread.
template <int OP, int TPR, typename T>
__device__ __forceinline__ T group_reduce(T v, T* cells, int t, int rsub) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1) {
    T o = __shfl_xor_sync(0xffffffffu, v, off, W);
    v = fold<OP>(v, o);
  }
  if (TPR > 32) {
    constexpr int NW = TPR / 32;
    if ((t & 31) == 0) cells[rsub * NW + (t >> 5)] = v;
    __syncthreads();
    if (sizeof(T) == 4 && NW % 4 == 0) {
      // the row's cells are read four at a time (the arrays are 16-byte aligned): two loads
      // instead of eight for a 256-thread row, folded in the same warp order
      T acc;
#pragma unroll
      for (int w = 0; w < NW; w += 4) {
        const Pack<T, 4> four = *reinterpret_cast<const Pack<T, 4>*>(cells + rsub * NW + w);
        acc = w == 0 ? four.v[0] : fold<OP>(acc, four.v[0]);
        acc = fold<OP>(acc, four.v[1]);
        acc = fold<OP>(acc, four.v[2]);
        acc = fold<OP>(acc, four.v[3]);
      }
      v = acc;
    } else {
      T acc = cells[rsub * NW];
#pragma unroll
      for (int w = 1; w < NW; ++w) acc = fold<OP>(acc, cells[rsub * NW + w]);
      v = acc;
    }
  }
  return v;
}
)CUDA";

const char* kernelPrelude() { return kRowPrelude; }

// index expression for dims [lo, hi) addressed by the flat index `flat` (row-major over those
// dims): adjacent dims whose strides chain are merged so that contiguous buffers cost one multiply
std::string indexExpr(const std::vector<int64_t>& extents, const std::vector<int64_t>& strides, int lo,
                      int hi, const std::string& flat) {
  struct Run { int64_t extent, stride, suffix; };
  std::vector<Run> runs;
  int64_t suffix = 1;
  for (int d = hi - 1; d >= lo; --d) {
    int64_t e = extents[d], s = strides[d];
    if (e == 1) continue;
    if (!runs.empty() && runs.back().stride * runs.back().extent == s && runs.back().suffix * runs.back().extent == suffix) {
      runs.back().extent *= e;
    } else if (!runs.empty() && runs.back().stride == 0 && s == 0 && runs.back().suffix * runs.back().extent == suffix) {
      runs.back().extent *= e;
    } else {
      runs.push_back({e, s, suffix});
    }
    suffix *= e;
  }
  const int64_t total = suffix;
  std::ostringstream out;
  bool any = false;
  for (const Run& r : runs) {
    if (r.stride == 0) continue;
    std::string coord = flat;
    if (r.suffix != 1) coord = "(" + coord + " / " + std::to_string(r.suffix) + "ll)";
    if (r.suffix * r.extent != total) coord = "(" + coord + " % " + std::to_string(r.extent) + "ll)";
    if (any) out << " + ";
    out << coord;
    if (r.stride != 1) out << " * " << r.stride << "ll";
    any = true;
  }
  return any ? out.str() : std::string("0ll");
}

namespace {

struct RowGen {
  const Cluster& c;
  const RowSchedule& s;
  std::ostringstream o;
  std::vector<char> cls;        // 'S' scalar everywhere, 'R' per row, 'E' per element
  std::vector<bool> emitted;    // scalar nodes emitted / element nodes emitted (register mode)
  std::vector<bool> is_out_ref;
  uint32_t row_mask;
  int ept;
  int64_t chunk;
  bool always_valid;
  bool packed;                  // element pairs use the f32x2 instructions
  int min_blocks = 0;           // __launch_bounds__ second argument (0 = none)
  std::vector<int> reds;        // Red node ids in order

  RowGen(const Cluster& cc, const RowSchedule& ss) : c(cc), s(ss) {
    row_mask = c.rowMask();
    cls.resize(c.nodes.size());
    for (size_t i = 0; i < c.nodes.size(); ++i) {
      uint32_t v = c.nodes[i].vary;
      cls[i] = v == 0 ? 'S' : ((v & ~row_mask) == 0 ? 'R' : 'E');
      if (c.nodes[i].op == ENode::Red) reds.push_back(static_cast<int>(i));
    }
    emitted.assign(c.nodes.size(), false);
    is_out_ref.assign(c.leaves.size(), false);
    for (auto& out : c.outputs) is_out_ref[out.ref] = true;
    ept = s.vec * s.vpt;
    chunk = static_cast<int64_t>(s.tpr) * s.vec * s.vpt;
    int64_t per_split = chunk * ((s.chunks + s.splits - 1) / s.splits);
    always_valid = (c.cols % chunk == 0) && (s.splits == 1 || (c.cols % per_split == 0));
    packed = s.vec % 2 == 0;
    min_blocks = s.min_blocks;
  }

  // Rows per thread (s.rpt > 1): the nodes that vary along the rows exist once per row of the
  // thread's block and carry the row's number in their names; everything else is shared.
  int cur_g = -1;               // row of the block being emitted, -1 = the shared part
  bool rowVarying(int i) const { return (c.nodes[i].vary & row_mask) != 0 || c.nodes[i].op == ENode::Red; }
  std::string rowSuffix() const { return (s.rpt > 1 && cur_g >= 0) ? "_g" + std::to_string(cur_g) : std::string(); }
  std::string rowVar() const { return "r" + rowSuffix(); }
  std::string name(int i) const { return "n" + std::to_string(i) + (rowVarying(i) ? rowSuffix() : std::string()); }
  std::string elem(int i, const std::string& idx) const {
    return cls[i] == 'E' ? name(i) + "[" + idx + "]" : name(i);
  }
  std::string loadConvert(DType d, const std::string& raw) const {
    if (d == DType::bf16) return "bf16_to_f32(" + raw + ")";
    if (d == DType::f16) return "f16_to_f32(" + raw + ")";
    if (d == DType::i1) return "(" + raw + " != 0)";
    return raw;
  }
  std::string storeConvert(DType d, const std::string& v) const {
    if (d == DType::bf16) return "f32_to_bf16(" + v + ")";
    if (d == DType::f16) return "f32_to_f16(" + v + ")";
    if (d == DType::i1) return "(unsigned char)(" + v + " ? 1 : 0)";
    return v;
  }
  bool colContiguous(const LeafRef& l) const {
    // the column part is one run of stride 1 over every non-unit column dim
    int64_t expect = 1;
    for (int d = static_cast<int>(c.extents.size()) - 1; d >= c.split; --d) {
      if (c.extents[d] == 1) continue;
      if (l.strides[d] != expect) return false;
      expect *= c.extents[d];
    }
    return true;
  }

  // Declares `var`: the offset that a looked-up leaf's index adds here, or -1 where the index is outside
  // the axis.  `col` is the flat column, "" where the index does not vary along the columns.
  void emitLookup(int leaf, const std::string& var, const std::string& col, const std::string& indent) {
    const LeafRef& l = c.leaves[leaf];
    const LeafRef& ix = c.leaves[l.index_leaf];
    std::string at = indexExpr(c.extents, ix.strides, 0, c.split, rowVar());
    if (!col.empty()) at += " + " + indexExpr(c.extents, ix.strides, c.split, static_cast<int>(c.extents.size()), col);
    o << indent << "long long " << var << " = (long long)L" << l.index_leaf << "[" << at << "];\n";
    o << indent << var << " = " << var << " >= 0 && " << var << " < " << l.index_extent << "ll ? " << var << " * "
      << l.index_stride << "ll : -1ll;\n";
  }
  // whether a looked-up leaf takes a number per element instead of one per row
  bool indexedByElement(const LeafRef& l) const { return l.index_leaf >= 0 && (c.leaves[l.index_leaf].vary & ~row_mask) != 0; }

  // ---- scalar (S / R class) nodes ----
  void emitScalarNode(int i, const std::string& indent, const std::vector<std::string>* red_values) {
    const ENode& n = c.nodes[i];
    const std::string ty = ctypeOf(n.dtype);
    if (n.op == ENode::Leaf && c.leaves[n.leaf].index_leaf >= 0) emitLookup(n.leaf, "gi_" + name(i), "", indent);
    o << indent << "const " << ty << " " << name(i) << " = ";
    switch (n.op) {
      case ENode::Leaf: {
        const LeafRef& l = c.leaves[n.leaf];
        std::string off = indexExpr(c.extents, l.strides, 0, c.split, rowVar());
        if (l.index_leaf >= 0) {
          const std::string gi = "gi_" + name(i);
          o << "(" << gi << " < 0 ? (" << ty << ")0 : " << loadConvert(l.dtype, "L" + std::to_string(n.leaf) + "[" + off + " + " + gi + "]") << ")";
          break;
        }
        o << loadConvert(l.dtype, "L" + std::to_string(n.leaf) + "[" + off + "]");
        break;
      }
      case ENode::Const: o << constLiteral(n); break;
      case ENode::Iota: {
        std::vector<int64_t> st(c.extents.size(), 0);
        st[n.dim] = 1;
        o << "(" << ty << ")(" << indexExpr(c.extents, st, 0, c.split, rowVar()) << ")";
        break;
      }
      case ENode::Red:
        o << (*red_values)[i];
        break;
      default: {
        std::string a = n.args[0] >= 0 ? name(n.args[0]) : "", b = n.args[1] >= 0 ? name(n.args[1]) : "",
                    cc = n.args[2] >= 0 ? name(n.args[2]) : "";
        o << elementwiseExpr(n, a, b, cc, c.nodes[n.args[n.op == ENode::Sel ? 1 : 0]].dtype);
      }
    }
    o << ";\n";
    markEmitted(i);
  }

  std::vector<std::vector<bool>> emitted_rows;   // s.rpt > 1: per row of the block, for the row-varying nodes
  bool isEmitted(int i) const {
    if (s.rpt > 1 && rowVarying(i)) return cur_g >= 0 && emitted_rows[cur_g][i];
    return emitted[i];
  }
  void markEmitted(int i) {
    if (s.rpt > 1 && rowVarying(i)) emitted_rows[cur_g][i] = true;
    else emitted[i] = true;
  }

  void emitReadyScalars(const std::string& indent, const std::vector<std::string>* red_values,
                        const std::vector<bool>& red_ready) {
    for (size_t i = 0; i < c.nodes.size(); ++i) {
      if (cls[i] == 'E') continue;
      if (s.rpt > 1 && rowVarying(static_cast<int>(i)) != (cur_g >= 0)) continue;   // shared part or one row's part
      if (isEmitted(static_cast<int>(i))) continue;
      const ENode& n = c.nodes[i];
      if (n.op == ENode::Red) {
        if (!red_ready[i]) continue;
      } else {
        bool ready = true;
        for (int a : n.args)
          if (a >= 0 && !isEmitted(a)) ready = false;
        if (!ready) continue;
      }
      emitScalarNode(static_cast<int>(i), indent, red_values);
    }
  }

  // ---- element (E class) nodes ----
  void emitElementNode(int i, const std::string& indent) {
    const ENode& n = c.nodes[i];
    const std::string ty = ctypeOf(n.dtype);
    o << indent << ty << " " << name(i) << "[" << ept << "];\n";
    if (n.op == ENode::Leaf) {
      const LeafRef& l = c.leaves[n.leaf];
      const std::string L = "L" + std::to_string(n.leaf);
      const std::string st = storageTypeOf(l.dtype);
      std::string rowoff = indexExpr(c.extents, l.strides, 0, c.split, rowVar());
      const bool lookup = l.index_leaf >= 0, by_element = indexedByElement(l);
      o << indent << "{\n";
      if (lookup && !by_element) {
        emitLookup(n.leaf, "gi", "", indent + "  ");
        rowoff += " + gi";
      }
      o << indent << "  const long long ro = " << rowoff << ";\n";
      o << indent << "#pragma unroll\n" << indent << "  for (int j = 0; j < " << s.vpt << "; ++j) {\n";
      o << indent << "    const long long c0 = cb + (long long)(j * " << s.tpr << " + t) * " << s.vec << ";\n";
      if (by_element) {
        std::string coloff = indexExpr(c.extents, l.strides, c.split, static_cast<int>(c.extents.size()), "c0");
        o << indent << "    " << st << " raw = 0;\n" << indent << "    if (" << (always_valid ? "true" : "c0 < cend") << ") {\n";
        emitLookup(n.leaf, "gi", "c0", indent + "      ");
        o << indent << "      if (gi >= 0) raw = " << L << "[ro + gi + " << coloff << "];\n" << indent << "    }\n";
        o << indent << "    " << name(i) << "[j] = " << loadConvert(l.dtype, "raw") << ";\n";
      } else if (colContiguous(l)) {
        o << indent << "    Pack<" << st << ", " << s.vec << "> p;\n";
        const std::string valid = std::string(always_valid ? "true" : "c0 < cend") + (lookup ? " && gi >= 0" : "");
        o << indent << "    if (" << valid << ") p = *reinterpret_cast<const Pack<" << st
          << ", " << s.vec << ">*>(" << L << " + ro + c0);\n";
        o << indent << "    else {\n" << indent << "#pragma unroll\n" << indent << "      for (int e = 0; e < "
          << s.vec << "; ++e) p.v[e] = 0; }\n";
        o << indent << "#pragma unroll\n" << indent << "    for (int e = 0; e < " << s.vec << "; ++e) " << name(i)
          << "[j * " << s.vec << " + e] = " << loadConvert(l.dtype, "p.v[e]") << ";\n";
      } else {
        std::string coloff = indexExpr(c.extents, l.strides, c.split, static_cast<int>(c.extents.size()), "c0");
        const std::string valid = std::string(always_valid ? "true" : "c0 < cend") + (lookup ? " && gi >= 0" : "");
        o << indent << "    " << st << " raw = 0;\n";
        o << indent << "    if (" << valid << ") raw = " << L << "[ro + " << coloff << "];\n";
        o << indent << "    " << name(i) << "[j] = " << loadConvert(l.dtype, "raw") << ";\n";
      }
      o << indent << "  }\n" << indent << "}\n";
      return;
    }
    if (emitPackedNode(i, indent)) return;
    o << indent << "#pragma unroll\n" << indent << "for (int i = 0; i < " << ept << "; ++i) ";
    if (n.op == ENode::Iota) {
      std::vector<int64_t> st(c.extents.size(), 0);
      st[n.dim] = 1;
      std::string cexpr = "(cb + (long long)((i / " + std::to_string(s.vec) + ") * " + std::to_string(s.tpr) +
                          " + t) * " + std::to_string(s.vec) + " + (i % " + std::to_string(s.vec) + "))";
      std::string coord;
      if (n.dim >= c.split) coord = indexExpr(c.extents, st, c.split, static_cast<int>(c.extents.size()), cexpr);
      else coord = indexExpr(c.extents, st, 0, c.split, rowVar());
      o << name(i) << "[i] = (" << ty << ")(" << coord << ");\n";
      return;
    }
    std::string a = n.args[0] >= 0 ? elem(n.args[0], "i") : "", b = n.args[1] >= 0 ? elem(n.args[1], "i") : "",
                cc = n.args[2] >= 0 ? elem(n.args[2], "i") : "";
    o << name(i) << "[i] = " << elementwiseExpr(n, a, b, cc, c.nodes[n.args[n.op == ENode::Sel ? 1 : 0]].dtype) << ";\n";
  }

  // Blackwell packed f32x2 arithmetic: add/sub/mul on two neighbouring elements per instruction
  // (add/sub/mul/fma .rn.f32x2; each lane is an ordinary IEEE f32 operation, so the results are
  // bit-identical to the scalar form and only the instruction count halves).  Division of a row by
  // a per-row value uses the row's reciprocal and two FMA correction steps per pair: correctly
  // rounded like div.rn for normal operands and results.  Rows whose divisor is zero, subnormal,
  // huge, non-finite or has an all-ones significand take the ordinary division, and a quotient
  // that is not a number falls back to x * (1/d), which carries the right infinity or NaN.
  // A product needs the guard against being merged into an FMA only where an addition can
  // consume it: every use by another multiply, a sine / cosine (whose first step multiplies or
  // takes the value as the addend of an FMA of its own), a comparison or max / min cannot absorb it.
  bool productMayMeetAnAdd(int i) const {
    bool used = false;
    for (size_t j = 0; j < c.nodes.size(); ++j) {
      const ENode& u = c.nodes[j];
      if (u.args[0] != i && u.args[1] != i && u.args[2] != i) continue;
      used = true;
      const bool harmless =
          (u.op == ENode::Bin && (static_cast<Binary>(u.sub) == Binary::mul || static_cast<Binary>(u.sub) == Binary::max ||
                                  static_cast<Binary>(u.sub) == Binary::min)) ||
          (u.op == ENode::Un && (static_cast<Unary>(u.sub) == Unary::sin || static_cast<Unary>(u.sub) == Unary::cos)) ||
          u.op == ENode::Cmp;
      if (!harmless) return true;
    }
    (void)used;  // a product that is only stored has no consumer to merge with
    return false;
  }

  // Sign of a zero quotient.  The correction steps of the packed division end in q + r * rc; when
  // the quotient is an exact zero that sum is +0 in round-to-nearest whatever the operands' signs,
  // where a true division gives -0 for (-0) / positive or (+0) / negative.  Every other quotient
  // already has the sign of the first estimate q0 = x * rc, so copying q0's sign bit onto the result
  // (one logic instruction per element) is always right; it is left out where the numerator can be
  // shown never to be -0 and the divisor never negative, as in exp(..) / sum(exp(..)) and in
  // (y - mean) / sqrt(..) of values that are themselves such quotients.
  // nonNegative: the value is >= +0 (or NaN), never -0.
  bool nonNegative(int i, int depth = 0) const {
    if (depth > 64) return false;
    const ENode& n = c.nodes[i];
    auto both = [&](int a, int b) { return nonNegative(a, depth + 1) && nonNegative(b, depth + 1); };
    switch (n.op) {
      case ENode::Const: {
        if (n.dtype == DType::f32) return (n.bits & 0x80000000ull) == 0;
        if (n.dtype == DType::bf16 || n.dtype == DType::f16) return (n.bits & 0x8000ull) == 0;
        return false;
      }
      case ENode::Un:
        switch (static_cast<Unary>(n.sub)) {
          case Unary::exp: case Unary::abs: return true;
          case Unary::sqrt: return nonNegative(n.args[0], depth + 1);
          default: return false;
        }
      case ENode::Bin:
        switch (static_cast<Binary>(n.sub)) {
          case Binary::mul: return n.args[0] == n.args[1] || both(n.args[0], n.args[1]);
          case Binary::add: case Binary::div: case Binary::max: case Binary::min: return both(n.args[0], n.args[1]);
          default: return false;
        }
      case ENode::Sel: return both(n.args[1], n.args[2]);
      case ENode::Red: {
        ENode init = constOf(i);
        const bool init_ok = (init.dtype == DType::f32 && (init.bits & 0x80000000ull) == 0) ||
                             ((init.dtype == DType::bf16 || init.dtype == DType::f16) && (init.bits & 0x8000ull) == 0);
        // a sum or a maximum of non-negative values from a non-negative start; a minimum as well
        return (init_ok || static_cast<Reducer>(n.sub) == Reducer::max) && nonNegative(n.args[0], depth + 1);
      }
      default: return false;
    }
  }
  // neverNegativeZero: the value may be negative, but it is never -0
  bool neverNegativeZero(int i, int depth = 0) const {
    if (depth > 64) return false;
    if (nonNegative(i, depth + 1)) return true;
    const ENode& n = c.nodes[i];
    if (n.op != ENode::Bin) return false;
    switch (static_cast<Binary>(n.sub)) {
      case Binary::sub: return neverNegativeZero(n.args[0], depth + 1);   // a - b is -0 only for (-0) - (+0)
      case Binary::add: return neverNegativeZero(n.args[0], depth + 1) || neverNegativeZero(n.args[1], depth + 1);
      default: return false;
    }
  }

  bool emitPackedNode(int i, const std::string& indent) {
    const ENode& n = c.nodes[i];
    if (packedSinCosNode(i)) {
      auto partner = joint_partner.find(i);
      if (partner != joint_partner.end()) {
        const bool i_is_sine = static_cast<Unary>(n.sub) == Unary::sin;
        emitPackedSinCosJoint(i_is_sine ? i : partner->second, i_is_sine ? partner->second : i, partner->second, indent);
        joint_done.insert(partner->second);
      } else {
        emitPackedSinCos(i, static_cast<Unary>(n.sub) == Unary::cos, indent);
      }
      return true;
    }
    if (packedExpNode(i)) {
      emitPackedExp(i, indent);
      return true;
    }
    if (!packed || n.op != ENode::Bin || !isFloatReg(n.dtype)) return false;
    const Binary op = static_cast<Binary>(n.sub);
    const int a = n.args[0], b = n.args[1];
    auto pairOf = [&](int node) {
      if (cls[node] == 'E') return "pk2(" + name(node) + "[i], " + name(node) + "[i + 1])";
      return "pk2(" + name(node) + ", " + name(node) + ")";
    };
    const std::string out = name(i);
    if (op == Binary::add || op == Binary::sub || op == Binary::mul) {
      const bool guarded = op == Binary::mul && productMayMeetAnAdd(i);
      const char* fn = op == Binary::add ? "add2" : (op == Binary::sub ? "sub2" : (guarded ? "mul2_own_rounding" : "mul2"));
      o << indent << "#pragma unroll\n" << indent << "for (int i = 0; i < " << ept << "; i += 2) upk2(" << fn << "("
        << pairOf(a) << ", " << pairOf(b) << (guarded ? ", oz" : "") << "), " << out << "[i], " << out << "[i + 1]);\n";
      return true;
    }
    if (op == Binary::div && cls[a] == 'E' && cls[b] != 'E') {
      o << indent << "{\n";
      o << indent << "  const float dv = " << name(b) << ";\n" << indent << "  const float rc = 1.0f / dv;\n";
      o << indent << "  const unsigned int db = __float_as_uint(dv) & 0x7fffffffu;\n";
      o << indent << "  if (db >= 0x0c800000u && db <= 0x72800000u && (db & 0x7fffffu) != 0x7fffffu) {\n";
      o << indent << "    const unsigned long long r2 = pk2(rc, rc), nd2 = pk2(-dv, -dv), z2 = pk2(0.0f, 0.0f);\n";
      o << indent << "    unsigned long long bad2 = z2;\n";
      o << indent << "#pragma unroll\n" << indent << "    for (int i = 0; i < " << ept << "; i += 2) {\n";
      o << indent << "      const unsigned long long x2 = pk2(" << name(a) << "[i], " << name(a) << "[i + 1]);\n";
      o << indent << "      const unsigned long long q0 = mul2(x2, r2);\n";
      o << indent << "      const unsigned long long q1 = fma2(fma2(q0, nd2, x2), r2, q0);\n";
      o << indent << "      const unsigned long long q2 = fma2(fma2(q1, nd2, x2), r2, q1);\n";
      o << indent << "      upk2(q2, " << out << "[i], " << out << "[i + 1]);\n";
      if (!(neverNegativeZero(a) && nonNegative(b))) {
        o << indent << "      {   // a zero quotient takes the sign of x * (1/d)\n";
        o << indent << "        float s0, s1;\n" << indent << "        upk2(q0, s0, s1);\n";
        o << indent << "        " << out << "[i] = __uint_as_float(__float_as_uint(" << out << "[i]) | (__float_as_uint(s0) & 0x80000000u));\n";
        o << indent << "        " << out << "[i + 1] = __uint_as_float(__float_as_uint(" << out << "[i + 1]) | (__float_as_uint(s1) & 0x80000000u));\n";
        o << indent << "      }\n";
      }
      o << indent << "      bad2 = fma2(q2, z2, bad2);   // stays zero while every quotient is finite\n";
      o << indent << "    }\n";
      o << indent << "    float b0, b1;\n" << indent << "    upk2(bad2, b0, b1);\n";
      o << indent << "    if (!(b0 + b1 == 0.0f)) {   // an infinite or NaN quotient: redo this thread's elements exactly\n";
      o << indent << "#pragma unroll\n" << indent << "      for (int i = 0; i < " << ept << "; ++i) " << out << "[i] = " << name(a) << "[i] / dv;\n";
      o << indent << "    }\n" << indent << "  } else {\n";
      o << indent << "#pragma unroll\n" << indent << "    for (int i = 0; i < " << ept << "; ++i) " << out << "[i] = " << name(a) << "[i] / dv;\n";
      o << indent << "  }\n" << indent << "}\n";
      return true;
    }
    return false;
  }

  bool packedExpNode(int i) const {
    static const bool off = [] { const char* e = std::getenv("ACCY_B200_PACKED_EXP"); return e && e[0] == '0'; }();
    const ENode& n = c.nodes[i];
    return !off && packed && n.op == ENode::Un && n.dtype == DType::f32 && ept % 2 == 0 && cls[i] == 'E' &&
           cls[n.args[0]] == 'E' && static_cast<Unary>(n.sub) == Unary::exp;
  }

  // exp of f32 pairs around the special-function unit's 2^x.  h = x * log2(e) rounded to f32 loses up
  // to half an ulp of h (2^-18 near h = 100, i.e. 2.6e-6 of the result), so the product's rounding
  // error l = x * L2E - h is recovered exactly with one fused step, the part of log2(e) that the f32
  // constant L2E lacks is added to it, and the result is 2^h * (1 + l * ln 2): five packed
  // operations and two ex2.approx per pair of elements, against about twenty instructions for two
  // calls of expf.  The error is that of ex2.approx (2^-22 relative) plus the final rounding.
  // Results below 2^-126 are flushed to zero where expf returns subnormal numbers.  A thread whose
  // elements hold an infinity, a NaN or an overflowing value (the result is then not finite, or the
  // correction term is not) redoes them with expf.
  void emitPackedExp(int i, const std::string& indent) {
    const ENode& n = c.nodes[i];
    const int a = n.args[0];
    const std::string out = name(i);
    o << indent << "{\n";
    o << indent << "  const unsigned long long l2e2 = pk2(1.4426950216293335f, 1.4426950216293335f), nl2e2 = pk2(-1.4426950216293335f, -1.4426950216293335f);\n";
    o << indent << "  const unsigned long long lo2 = pk2(1.9259629911266175e-08f, 1.9259629911266175e-08f), ln2 = pk2(0.6931471824645996f, 0.6931471824645996f), z2 = pk2(0.0f, 0.0f);\n";
    o << indent << "  unsigned long long bad2 = z2;\n";
    o << indent << "#pragma unroll\n" << indent << "  for (int i = 0; i < " << ept << "; i += 2) {\n";
    o << indent << "    const unsigned long long x2 = pk2(" << name(a) << "[i], " << name(a) << "[i + 1]);\n";
    o << indent << "    const unsigned long long nh2 = mul2(x2, nl2e2);\n";
    o << indent << "    unsigned long long l2 = fma2(x2, l2e2, nh2);\n";
    o << indent << "    l2 = fma2(x2, lo2, l2);\n";
    o << indent << "    float nh0, nh1;\n" << indent << "    upk2(nh2, nh0, nh1);\n";
    o << indent << "    const unsigned long long e2 = pk2(ex2_ftz(-nh0), ex2_ftz(-nh1));\n";
    o << indent << "    const unsigned long long y2 = fma2(e2, mul2(l2, ln2), e2);\n";
    o << indent << "    upk2(y2, " << out << "[i], " << out << "[i + 1]);\n";
    o << indent << "    bad2 = fma2(y2, z2, bad2);   // stays zero while every result is finite\n";
    o << indent << "  }\n";
    o << indent << "  float b0, b1;\n" << indent << "  upk2(bad2, b0, b1);\n";
    o << indent << "  if (!(b0 + b1 == 0.0f)) {\n";
    o << indent << "#pragma unroll\n" << indent << "    for (int i = 0; i < " << ept << "; ++i) " << out << "[i] = expf(" << name(a) << "[i]);\n";
    o << indent << "  }\n" << indent << "}\n";
  }

  // Range check of the packed sine / cosine.  The routines are good for |x| <= 1e5; each thread
  // tracks the largest |x| of its chunk (one max per element).  When x is a product of a value that
  // is the same for the whole row and an element value that the thread's rows share (rows per
  // thread: frequency * time in the mismatch program), the largest |x| is bounded by |row value| *
  // max |shared element|, and that maximum is taken once per chunk for all the thread's rows.
  std::map<int, std::string> shared_amax;   // shared element node -> variable holding max |element| of the chunk
  std::string sharedBound(int arg) const {
    const ENode& a = c.nodes[arg];
    if (s.rpt <= 1 || cur_g < 0 || a.op != ENode::Bin || static_cast<Binary>(a.sub) != Binary::mul) return "";
    for (int side = 0; side < 2; ++side) {
      const int scalar = a.args[side], elems = a.args[1 - side];
      if (cls[scalar] == 'E' || cls[elems] != 'E' || rowVarying(elems)) continue;
      auto it = shared_amax.find(elems);
      if (it == shared_amax.end()) continue;
      // the rounded product can exceed the exact one by half an ulp
      return "fabsf(" + name(scalar) + ") * " + it->second + " * 1.000001f";
    }
    return "";
  }
  void emitSharedMaxima(const std::set<int>& need, const std::string& indent) {
    shared_amax.clear();
    for (int i : need) {
      if (!rowVarying(i) || !packedSinCosNode(i)) continue;
      const ENode& a = c.nodes[c.nodes[i].args[0]];
      if (a.op != ENode::Bin || static_cast<Binary>(a.sub) != Binary::mul) continue;
      for (int side = 0; side < 2; ++side) {
        const int scalar = a.args[side], elems = a.args[1 - side];
        if (cls[scalar] == 'E' || cls[elems] != 'E' || rowVarying(elems) || shared_amax.count(elems)) continue;
        const std::string var = "amax_n" + std::to_string(elems);
        o << indent << "float " << var << " = 0.0f;\n";
        o << indent << "#pragma unroll\n" << indent << "for (int i = 0; i < " << ept << "; ++i) " << var << " = fmaxf(" << var
          << ", fabsf(n" << elems << "[i]));\n";
        shared_amax[elems] = var;
      }
    }
  }

  bool packedSinCosNode(int i) const {
    const ENode& n = c.nodes[i];
    return packed && n.op == ENode::Un && n.dtype == DType::f32 && ept % 2 == 0 && cls[i] == 'E' &&
           (static_cast<Unary>(n.sub) == Unary::sin || static_cast<Unary>(n.sub) == Unary::cos);
  }

  std::map<int, int> joint_partner;  // sine node <-> cosine node of the same argument, for the pass being emitted
  std::set<int> joint_done;          // partners already computed by the other node's block

  // Sine and cosine of the same f32 value, together: x = k*(pi/2) + r with k = rint(x*2/pi) from the
  // low bits of x*2/pi + 1.5*2^23 and r by three fused steps against a three-part pi/2 (72 bits);
  // sin(r) = r + r*s*ps(s) and cos(r) = 1 - s/2 + s*s*pc(s) on [-pi/4, pi/4], s = r*r, ps and pc of
  // degree 2 (least-squares fits reweighted towards equal ripple, made for this file); the quadrant
  // k mod 4 picks which of the two is the sine and which the cosine, and their signs.  14 packed
  // operations per pair of elements for both results, against 28 for the two separate routines.
  // Checked against f64 over |x| <= 1e5, near multiples of pi/2 and on the mismatch phases: at most
  // 1.53 ulp (mean 0.30) for either result.  Beyond 1e5 or at an infinity the thread redoes its
  // elements with sinf / cosf; NaN stays NaN.
  void emitPackedSinCosJoint(int sine, int cosine, int declare, const std::string& indent) {
    const int a = c.nodes[sine].args[0];
    const std::string S = name(sine), C = name(cosine);
    auto at = [&](const std::string& idx) { return cls[a] == 'E' ? name(a) + "[" + idx + "]" : name(a); };
    o << indent << "float " << name(declare) << "[" << ept << "];\n";
    o << indent << "{\n";
    o << indent << "  const unsigned long long ip2 = pk2(0.6366197466850281f, 0.6366197466850281f), mg2 = pk2(12582912.0f, 12582912.0f);\n";
    o << indent << "  const unsigned long long pa2 = pk2(-1.5707963705062866f, -1.5707963705062866f), pb2 = pk2(4.371138828673793e-08f, 4.371138828673793e-08f), pc2 = pk2(1.7151245100058819e-15f, 1.7151245100058819e-15f);\n";
    const std::string bound = sharedBound(a);
    if (bound.empty()) o << indent << "  float big = 0.0f;\n";
    else o << indent << "  const float big = " << bound << ";\n";
    o << indent << "#pragma unroll\n" << indent << "  for (int i = 0; i < " << ept << "; i += 2) {\n";
    o << indent << "    const float x0 = " << at("i") << ", x1 = " << at("i + 1") << ";\n";
    if (bound.empty()) o << indent << "    big = fmaxf(big, fmaxf(fabsf(x0), fabsf(x1)));\n";
    o << indent << "    const unsigned long long x2 = pk2(x0, x1);\n";
    o << indent << "    const unsigned long long q2 = fma2(x2, ip2, mg2);\n";
    o << indent << "    const unsigned long long k2 = sub2(q2, mg2);\n";
    o << indent << "    unsigned long long r2 = fma2(k2, pa2, x2);\n";
    o << indent << "    r2 = fma2(k2, pb2, r2);\n" << indent << "    r2 = fma2(k2, pc2, r2);\n";
    o << indent << "    const unsigned long long s2 = mul2(r2, r2);\n";
    o << indent << "    unsigned long long ps2 = fma2(pk2(-0.00019514957966748625f, -0.00019514957966748625f), s2, pk2(0.00833215843886137f, 0.00833215843886137f));\n";
    o << indent << "    ps2 = fma2(ps2, s2, pk2(-0.16666655242443085f, -0.16666655242443085f));\n";
    o << indent << "    const unsigned long long sn2 = fma2(mul2(r2, s2), ps2, r2);\n";
    o << indent << "    unsigned long long pq2 = fma2(pk2(2.4432783902739175e-05f, 2.4432783902739175e-05f), s2, pk2(-0.0013887312961742282f, -0.0013887312961742282f));\n";
    o << indent << "    pq2 = fma2(pq2, s2, pk2(0.04166664555668831f, 0.04166664555668831f));\n";
    o << indent << "    pq2 = fma2(pq2, s2, pk2(-0.5f, -0.5f));\n";
    o << indent << "    const unsigned long long cs2 = fma2(pq2, s2, pk2(1.0f, 1.0f));\n";
    o << indent << "    float sn0, sn1, cs0, cs1, q0, q1;\n";
    o << indent << "    upk2(sn2, sn0, sn1);\n" << indent << "    upk2(cs2, cs0, cs1);\n" << indent << "    upk2(q2, q0, q1);\n";
    o << indent << "    const unsigned int kb0 = __float_as_uint(q0), kb1 = __float_as_uint(q1);\n";
    o << indent << "    const bool w0 = (kb0 & 1u) != 0u, w1 = (kb1 & 1u) != 0u;   // odd quadrant: the two results swap\n";
    o << indent << "    " << S << "[i] = __uint_as_float(__float_as_uint(w0 ? cs0 : sn0) ^ ((kb0 & 2u) << 30));\n";
    o << indent << "    " << S << "[i + 1] = __uint_as_float(__float_as_uint(w1 ? cs1 : sn1) ^ ((kb1 & 2u) << 30));\n";
    o << indent << "    " << C << "[i] = __uint_as_float(__float_as_uint(w0 ? sn0 : cs0) ^ (((kb0 + 1u) & 2u) << 30));\n";
    o << indent << "    " << C << "[i + 1] = __uint_as_float(__float_as_uint(w1 ? sn1 : cs1) ^ (((kb1 + 1u) & 2u) << 30));\n";
    o << indent << "  }\n";
    o << indent << "  if (!(big <= 100000.0f)) {\n";
    o << indent << "#pragma unroll\n" << indent << "    for (int i = 0; i < " << ept << "; ++i) {\n";
    o << indent << "      " << S << "[i] = sinf(" << at("i") << ");\n";
    o << indent << "      " << C << "[i] = cosf(" << at("i") << ");\n";
    o << indent << "    }\n" << indent << "  }\n" << indent << "}\n";
  }

  // sin / cos of f32 pairs on the packed FMA path.  x = j*pi + r (cos: x = (j + 1/2)*pi + r) with
  // j = rint(x/pi) taken from the low bits of x/pi + 1.5*2^23, r by three fused steps against a
  // three-part pi (72 bits), sin(r) on [-pi/2, pi/2] as r + r*s*p(s), s = r*r, p of degree 3 (a
  // least-squares fit reweighted towards equal ripple, made for this file; its own error is 0.2
  // ulp, a degree-5 fit measured no better after rounding), sign from the parity of j.  Checked
  // against f64 over |x| <= 1e5, near multiples of pi and of pi/2: at most 1.9 ulp (mean 0.34).  A thread whose chunk holds an |x| above 1e5 or an infinity redoes its
  // elements with sinf / cosf; NaN stays NaN.  Differences from sinf: sin(-0) is +0, cos(0) is
  // 1 - 2^-24.  About 9 instructions per element against roughly 20 for sinf.
  void emitPackedSinCos(int i, bool cosine, const std::string& indent) {
    const ENode& n = c.nodes[i];
    const int a = n.args[0];
    const std::string out = name(i);
    auto at = [&](const std::string& idx) { return cls[a] == 'E' ? name(a) + "[" + idx + "]" : name(a); };
    o << indent << "{\n";
    o << indent << "  const unsigned long long ip2 = pk2(0.31830987334251404f, 0.31830987334251404f), mg2 = pk2(12582912.0f, 12582912.0f);\n";
    o << indent << "  const unsigned long long pa2 = pk2(-3.1415927410125732f, -3.1415927410125732f), pb2 = pk2(8.742277657347586e-08f, 8.742277657347586e-08f), pc2 = pk2(3.4302490200117637e-15f, 3.4302490200117637e-15f);\n";
    const std::string bound = sharedBound(a);
    if (bound.empty()) o << indent << "  float big = 0.0f;\n";
    else o << indent << "  const float big = " << bound << ";\n";
    o << indent << "#pragma unroll\n" << indent << "  for (int i = 0; i < " << ept << "; i += 2) {\n";
    o << indent << "    const float x0 = " << at("i") << ", x1 = " << at("i + 1") << ";\n";
    if (bound.empty()) o << indent << "    big = fmaxf(big, fmaxf(fabsf(x0), fabsf(x1)));\n";
    o << indent << "    const unsigned long long x2 = pk2(x0, x1);\n";
    if (cosine) {
      o << indent << "    const unsigned long long q2 = add2(fma2(x2, ip2, pk2(-0.5f, -0.5f)), mg2);\n";
      o << indent << "    const unsigned long long j2 = add2(sub2(q2, mg2), pk2(0.5f, 0.5f));\n";
    } else {
      o << indent << "    const unsigned long long q2 = fma2(x2, ip2, mg2);\n";
      o << indent << "    const unsigned long long j2 = sub2(q2, mg2);\n";
    }
    o << indent << "    unsigned long long r2 = fma2(j2, pa2, x2);\n";
    o << indent << "    r2 = fma2(j2, pb2, r2);\n" << indent << "    r2 = fma2(j2, pc2, r2);\n";
    o << indent << "    const unsigned long long s2 = mul2(r2, r2);\n";
    o << indent << "    unsigned long long p2 = fma2(pk2(2.610866431496106e-06f, 2.610866431496106e-06f), s2, pk2(-0.00019811965466942638f, -0.00019811965466942638f));\n";
    o << indent << "    p2 = fma2(p2, s2, pk2(0.008333100005984306f, 0.008333100005984306f));\n";
    o << indent << "    p2 = fma2(p2, s2, pk2(-0.16666661202907562f, -0.16666661202907562f));\n";
    o << indent << "    const unsigned long long y2 = fma2(mul2(r2, s2), p2, r2);\n";
    o << indent << "    float y0, y1, q0, q1;\n" << indent << "    upk2(y2, y0, y1);\n" << indent << "    upk2(q2, q0, q1);\n";
    const char* flip = cosine ? "~" : "";
    o << indent << "    " << out << "[i] = __uint_as_float(__float_as_uint(y0) ^ ((" << flip << "__float_as_uint(q0)) << 31));\n";
    o << indent << "    " << out << "[i + 1] = __uint_as_float(__float_as_uint(y1) ^ ((" << flip << "__float_as_uint(q1)) << 31));\n";
    o << indent << "  }\n";
    o << indent << "  if (!(big <= 100000.0f)) {\n";
    o << indent << "#pragma unroll\n" << indent << "    for (int i = 0; i < " << ept << "; ++i) " << out << "[i] = "
      << (cosine ? "cosf(" : "sinf(") << at("i") << ");\n";
    o << indent << "  }\n" << indent << "}\n";
  }

  void collectElementDeps(int i, std::set<int>& need) const {
    if (cls[i] != 'E' || need.count(i)) return;
    const ENode& n = c.nodes[i];
    if (n.op == ENode::Red) return;
    need.insert(i);
    for (int a : n.args)
      if (a >= 0) collectElementDeps(a, need);
  }

  void emitStore(const ClusterOutput& out, const std::string& indent) {
    const LeafRef& ref = c.leaves[out.ref];
    const std::string O = "L" + std::to_string(out.ref);
    const std::string st = storageTypeOf(ref.dtype);
    std::string rowoff = indexExpr(c.extents, ref.strides, 0, c.split, "r");
    o << indent << "if (row_ok) {\n" << indent << "  const long long ro = " << rowoff << ";\n";
    o << indent << "#pragma unroll\n" << indent << "  for (int j = 0; j < " << s.vpt << "; ++j) {\n";
    o << indent << "    const long long c0 = cb + (long long)(j * " << s.tpr << " + t) * " << s.vec << ";\n";
    o << indent << "    if (" << (always_valid ? "true" : "c0 < cend") << ") {\n";
    if (colContiguous(ref)) {
      o << indent << "      Pack<" << st << ", " << s.vec << "> p;\n";
      o << indent << "#pragma unroll\n" << indent << "      for (int e = 0; e < " << s.vec << "; ++e) p.v[e] = "
        << storeConvert(ref.dtype, elem(out.node, "j * " + std::to_string(s.vec) + " + e")) << ";\n";
      o << indent << "      *reinterpret_cast<Pack<" << st << ", " << s.vec << ">*>(" << O << " + ro + c0) = p;\n";
    } else {
      std::string coloff = indexExpr(c.extents, ref.strides, c.split, static_cast<int>(c.extents.size()), "c0");
      o << indent << "      " << O << "[ro + " << coloff << "] = " << storeConvert(ref.dtype, elem(out.node, "j")) << ";\n";
    }
    o << indent << "    }\n" << indent << "  }\n" << indent << "}\n";
  }

  bool outputIsElement(const ClusterOutput& out) const {
    return (c.leaves[out.ref].vary & ~row_mask) != 0;
  }

  std::string params(bool with_partials, bool with_zero = false) const {
    std::ostringstream p;
    bool first = true;
    for (size_t l = 0; l < c.leaves.size(); ++l) {
      if (!first) p << ", ";
      first = false;
      if (is_out_ref[l]) p << storageTypeOf(c.leaves[l].dtype) << "* __restrict__ L" << l;
      else p << "const " << storageTypeOf(c.leaves[l].dtype) << "* __restrict__ L" << l;
    }
    if (with_partials) {
      p << (first ? "" : ", ") << "unsigned long long* __restrict__ partials";
      first = false;
    }
    if (with_zero) p << (first ? "" : ", ") << "const unsigned long long oz";
    return p.str();
  }

  int outputLevel(const ClusterOutput& out) const { return c.nodes[out.node].level; }

  std::string generateMain(const std::string& kname) {
    const int block = s.tpr * s.rpc;
    o << kRowPrelude;
    o << "extern \"C\" __global__ void __launch_bounds__(" << block;
    if (min_blocks > 0) o << ", " << min_blocks;
    o << ") " << kname << "(" << params(s.splits > 1 && !reds.empty(), packed) << ") {\n";
    o << "  const int t = threadIdx.x % " << s.tpr << ";\n  const int rsub = threadIdx.x / " << s.tpr << ";\n";
    if (packed) o << "  (void)oz;\n";
    o << "  long long r = (long long)blockIdx.x * " << s.rpc << " + rsub;\n";
    o << "  const bool row_ok = r < " << c.rows << "ll;\n  if (!row_ok) r = " << c.rows - 1 << "ll;\n";
    const int64_t chunks_per_split = (s.chunks + s.splits - 1) / s.splits;
    if (s.splits > 1) {
      o << "  const long long ck_begin = (long long)blockIdx.y * " << chunks_per_split << "ll;\n";
      o << "  const long long ck_end = ck_begin + " << chunks_per_split << "ll < " << s.chunks << "ll ? ck_begin + "
        << chunks_per_split << "ll : " << s.chunks << "ll;\n";
    } else {
      o << "  const long long ck_begin = 0, ck_end = " << s.chunks << "ll;\n";
    }
    o << "  const long long cend = " << c.cols << "ll;\n  (void)cend; (void)ck_begin; (void)ck_end; (void)t; (void)rsub;\n";
    for (int rid : reds) {
      if (s.tpr > 32)
        o << "  __shared__ __align__(16) " << ctypeOf(c.nodes[rid].dtype) << " cells_" << rid << "[" << s.rpc * (s.tpr / 32) << "];\n";
    }
    std::vector<std::string> red_values(c.nodes.size());
    std::vector<bool> red_ready(c.nodes.size(), false);
    emitReadyScalars("  ", &red_values, red_ready);
    int max_level = 0;
    for (const ENode& n : c.nodes) max_level = std::max(max_level, n.level);
    const bool registers = s.chunks == 1;
    std::vector<bool> elem_emitted(c.nodes.size(), false);
    if (registers) o << "  const long long cb = 0;\n";
    for (int pass = 0; pass <= max_level; ++pass) {
      std::vector<int> pass_reds;
      for (int rid : reds)
        if (c.nodes[c.nodes[rid].args[0]].level == pass) pass_reds.push_back(rid);
      std::vector<const ClusterOutput*> pass_outs;
      for (auto& out : c.outputs)
        if (outputIsElement(out) && outputLevel(out) == pass) pass_outs.push_back(&out);
      if (pass_reds.empty() && pass_outs.empty()) continue;
      std::set<int> need;
      for (int rid : pass_reds) collectElementDeps(c.nodes[rid].args[0], need);
      for (auto* out : pass_outs) collectElementDeps(out->node, need);
      for (int rid : pass_reds) {
        o << "  " << ctypeOf(c.nodes[rid].dtype) << " acc_" << rid << " = " << constLiteral(identityOf(rid)) << ";\n";
        if (packedSum(rid)) o << "  unsigned long long acc2_" << rid << " = pk2(acc_" << rid << ", 0.0f);\n";
      }
      std::string ind = "  ";
      if (!registers) {
        o << "  for (long long ck = ck_begin; ck < ck_end; ++ck) {\n    const long long cb = ck * " << chunk << "ll;\n";
        ind = "    ";
      }
      // a sine and a cosine of the same value are computed together (one range reduction)
      joint_partner.clear();
      joint_done.clear();
      for (int i : need) {
        if ((registers && elem_emitted[i]) || !packedSinCosNode(i) || joint_partner.count(i)) continue;
        for (int j : need) {
          if (j <= i || (registers && elem_emitted[j]) || !packedSinCosNode(j) || joint_partner.count(j)) continue;
          if (c.nodes[j].args[0] == c.nodes[i].args[0] && c.nodes[j].sub != c.nodes[i].sub) {
            joint_partner[i] = j;
            joint_partner[j] = i;
            break;
          }
        }
      }
      for (int i : need) {  // std::set iterates in increasing id = topological order
        if (registers && elem_emitted[i]) continue;
        if (!joint_done.count(i)) emitElementNode(i, ind);
        elem_emitted[i] = true;
      }
      for (int rid : pass_reds) {
        int arg = c.nodes[rid].args[0];
        if (packedSum(rid)) {
          o << ind << "#pragma unroll\n" << ind << "for (int i = 0; i < " << ept << "; i += 2) acc2_" << rid << " = add2(acc2_"
            << rid << ", pk2(" << name(arg) << "[i], " << name(arg) << "[i + 1]));\n";
          continue;
        }
        o << ind << "#pragma unroll\n" << ind << "for (int i = 0; i < " << ept << "; ++i) {\n";
        if (!always_valid)
          o << ind << "  const long long ci = cb + (long long)((i / " << s.vec << ") * " << s.tpr << " + t) * " << s.vec
            << ";\n" << ind << "  if (ci < cend) ";
        else
          o << ind << "  ";
        o << "acc_" << rid << " = fold<" << static_cast<int>(c.nodes[rid].sub) << ">(acc_" << rid << ", "
          << elem(arg, "i") << ");\n" << ind << "}\n";
      }
      for (auto* out : pass_outs) emitStore(*out, ind);
      if (!registers) o << "  }\n";
      for (int rid : pass_reds)
        if (packedSum(rid))
          o << "  { float lo, hi; upk2(acc2_" << rid << ", lo, hi); acc_" << rid << " = lo + hi; }\n";
      for (int rid : pass_reds) {
        std::string cells = s.tpr > 32 ? "cells_" + std::to_string(rid) : std::string("(") + ctypeOf(c.nodes[rid].dtype) + "*)0";
        red_values[rid] = "group_reduce<" + std::to_string(static_cast<int>(c.nodes[rid].sub)) + ", " +
                          std::to_string(s.tpr) + ">(acc_" + std::to_string(rid) + ", " + cells + ", t, rsub)";
        // the recorded initial value enters the fold once per row (with column splits: in the
        // combine kernel), never once per thread
        if (s.splits == 1) red_values[rid] = withInit(rid, red_values[rid]);
        red_ready[rid] = true;
      }
      if (s.splits > 1 && !pass_reds.empty()) {
        // column-split rows: publish this CTA's partial of every reduction and stop; the
        // combine kernel folds the partials in split order and finishes the row
        for (size_t k = 0; k < pass_reds.size(); ++k) {
          int rid = pass_reds[k];
          const std::string ty = ctypeOf(c.nodes[rid].dtype);
          o << "  {\n    const " << ty << " part = " << red_values[rid] << ";\n";
          o << "    if (row_ok && t == 0) *reinterpret_cast<" << ty << "*>(partials + ((" << redIndex(rid) << "ll * "
            << c.rows << "ll + r) * " << s.splits << "ll + blockIdx.y)) = part;\n  }\n";
        }
        o << "}\n";
        return o.str();
      }
      emitReadyScalars("  ", &red_values, red_ready);
    }
    for (auto& out : c.outputs) {
      if (outputIsElement(out)) continue;
      const LeafRef& ref = c.leaves[out.ref];
      std::string off = indexExpr(c.extents, ref.strides, 0, c.split, "r");
      o << "  if (row_ok && t == 0" << (s.splits > 1 ? " && blockIdx.y == 0" : "") << ") L" << out.ref << "[" << off
        << "] = " << storeConvert(ref.dtype, name(out.node)) << ";\n";
    }
    o << "}\n";
    return o.str();
  }

  // Rows per thread: a streaming single-pass kernel (every reduction folds element values, nothing
  // is stored per element) in which each thread works on s.rpt neighbouring rows at once.  Values
  // that do not vary along the rows (the column vectors a broadcast stretches over every row, and
  // whatever is computed from them alone) are loaded and evaluated once per chunk and shared by the
  // thread's rows: the mismatch program reads its time and sample vectors once for two guesses.
  static bool blockable(const Cluster& c, const RowSchedule& s) {
    if (s.chunks <= 1 || s.splits != 1) return false;
    const uint32_t row_mask = c.rowMask();
    bool shared_leaf = false, any_red = false;
    for (const ENode& n : c.nodes) {
      if (n.op == ENode::Red) {
        any_red = true;
        const ENode& arg = c.nodes[n.args[0]];
        if (arg.level != 0 || (arg.vary & row_mask) == 0 || (arg.vary & ~row_mask) == 0) return false;
      }
      if (n.op == ENode::Leaf && (n.vary & row_mask) == 0 && (n.vary & ~row_mask) != 0) shared_leaf = true;
    }
    for (auto& out : c.outputs)
      if ((c.leaves[out.ref].vary & ~row_mask) != 0) return false;
    return any_red && shared_leaf;
  }

  std::string generateBlocked(const std::string& kname) {
    const int block = s.tpr * s.rpc;
    const int G = s.rpt;
    emitted_rows.assign(G, std::vector<bool>(c.nodes.size(), false));
    o << kRowPrelude;
    o << "extern \"C\" __global__ void __launch_bounds__(" << block;
    if (min_blocks > 0) o << ", " << min_blocks;
    o << ") " << kname << "(" << params(false, packed) << ") {\n";
    o << "  const int t = threadIdx.x % " << s.tpr << ";\n  const int rsub = threadIdx.x / " << s.tpr << ";\n";
    if (packed) o << "  (void)oz;\n";
    for (int g = 0; g < G; ++g) {
      o << "  long long r_g" << g << " = ((long long)blockIdx.x * " << s.rpc << " + rsub) * " << G << " + " << g << ";\n";
      o << "  const bool row_ok_g" << g << " = r_g" << g << " < " << c.rows << "ll;\n  if (!row_ok_g" << g << ") r_g" << g
        << " = " << c.rows - 1 << "ll;\n";
    }
    o << "  const long long cend = " << c.cols << "ll;\n  (void)cend; (void)t; (void)rsub;\n";
    const int nw = s.tpr / 32;
    for (int rid : reds)
      if (s.tpr > 32)
        o << "  __shared__ __align__(16) " << ctypeOf(c.nodes[rid].dtype) << " cells_" << rid << "[" << G * s.rpc * nw << "];\n";
    std::vector<std::vector<std::string>> red_values(G, std::vector<std::string>(c.nodes.size()));
    std::vector<bool> red_ready(c.nodes.size(), false);
    cur_g = -1;
    emitReadyScalars("  ", &red_values[0], red_ready);
    for (int g = 0; g < G; ++g) {
      cur_g = g;
      emitReadyScalars("  ", &red_values[g], red_ready);
    }
    std::set<int> need;
    for (int rid : reds) collectElementDeps(c.nodes[rid].args[0], need);
    for (int g = 0; g < G; ++g) {
      cur_g = g;
      for (int rid : reds) {
        o << "  " << ctypeOf(c.nodes[rid].dtype) << " acc_" << rid << rowSuffix() << " = " << constLiteral(identityOf(rid)) << ";\n";
        if (packedSum(rid)) o << "  unsigned long long acc2_" << rid << rowSuffix() << " = pk2(acc_" << rid << rowSuffix() << ", 0.0f);\n";
      }
    }
    o << "  for (long long ck = 0; ck < " << s.chunks << "ll; ++ck) {\n    const long long cb = ck * " << chunk << "ll;\n";
    const std::string ind = "    ";
    // a sine and a cosine of the same value are computed together (one range reduction)
    joint_partner.clear();
    for (int i : need) {
      if (!packedSinCosNode(i) || joint_partner.count(i)) continue;
      for (int j : need) {
        if (j <= i || !packedSinCosNode(j) || joint_partner.count(j)) continue;
        if (c.nodes[j].args[0] == c.nodes[i].args[0] && c.nodes[j].sub != c.nodes[i].sub) {
          joint_partner[i] = j;
          joint_partner[j] = i;
          break;
        }
      }
    }
    cur_g = -1;
    joint_done.clear();
    for (int i : need)   // the part shared by the thread's rows
      if (!rowVarying(i) && !joint_done.count(i)) emitElementNode(i, ind);
    emitSharedMaxima(need, ind);
    for (int g = 0; g < G; ++g) {
      cur_g = g;
      joint_done.clear();
      o << ind << "{\n";
      for (int i : need)
        if (rowVarying(i) && !joint_done.count(i)) emitElementNode(i, ind + "  ");
      for (int rid : reds) {
        const int arg = c.nodes[rid].args[0];
        const std::string acc = "acc_" + std::to_string(rid) + rowSuffix(), acc2 = "acc2_" + std::to_string(rid) + rowSuffix();
        if (packedSum(rid)) {
          o << ind << "  #pragma unroll\n" << ind << "  for (int i = 0; i < " << ept << "; i += 2) " << acc2 << " = add2(" << acc2
            << ", pk2(" << name(arg) << "[i], " << name(arg) << "[i + 1]));\n";
          continue;
        }
        o << ind << "  #pragma unroll\n" << ind << "  for (int i = 0; i < " << ept << "; ++i) {\n";
        if (!always_valid)
          o << ind << "    const long long ci = cb + (long long)((i / " << s.vec << ") * " << s.tpr << " + t) * " << s.vec
            << ";\n" << ind << "    if (ci < cend) ";
        else
          o << ind << "    ";
        o << acc << " = fold<" << static_cast<int>(c.nodes[rid].sub) << ">(" << acc << ", " << elem(arg, "i") << ");\n" << ind << "  }\n";
      }
      o << ind << "}\n";
    }
    o << "  }\n";
    for (int rid : reds) red_ready[rid] = true;
    for (int g = 0; g < G; ++g) {
      cur_g = g;
      for (int rid : reds) {
        const std::string acc = "acc_" + std::to_string(rid) + rowSuffix();
        if (packedSum(rid)) o << "  { float lo, hi; upk2(acc2_" << rid << rowSuffix() << ", lo, hi); " << acc << " = lo + hi; }\n";
        std::string cells = s.tpr > 32 ? "cells_" + std::to_string(rid) + " + " + std::to_string(g * s.rpc * nw)
                                       : std::string("(") + ctypeOf(c.nodes[rid].dtype) + "*)0";
        red_values[g][rid] = withInit(rid, "group_reduce<" + std::to_string(static_cast<int>(c.nodes[rid].sub)) + ", " +
                                               std::to_string(s.tpr) + ">(" + acc + ", " + cells + ", t, rsub)");
      }
      emitReadyScalars("  ", &red_values[g], red_ready);
      emitReadyScalars("  ", &red_values[g], red_ready);
      for (auto& out : c.outputs) {
        const LeafRef& ref = c.leaves[out.ref];
        std::string off = indexExpr(c.extents, ref.strides, 0, c.split, rowVar());
        o << "  if (row_ok_g" << g << " && t == 0) L" << out.ref << "[" << off << "] = " << storeConvert(ref.dtype, name(out.node)) << ";\n";
      }
    }
    o << "}\n";
    cur_g = -1;
    return o.str();
  }

  // a sum over per-element f32 values with every element valid: two running sums in one register pair
  bool packedSum(int rid) const {
    const ENode& r = c.nodes[rid];
    return packed && always_valid && static_cast<Reducer>(r.sub) == Reducer::sum && isFloatReg(r.dtype) &&
           cls[r.args[0]] == 'E';
  }

  int redIndex(int rid) const {
    for (size_t k = 0; k < reds.size(); ++k)
      if (reds[k] == rid) return static_cast<int>(k);
    return 0;
  }

  ENode constOf(int rid) const {
    ENode k;
    k.op = ENode::Const;
    k.dtype = c.nodes[rid].dtype;
    k.bits = c.nodes[rid].bits;
    return k;
  }

  // The value every thread's accumulator starts from: the reducer's identity (0, the lowest or the
  // highest value of the type).  The reference folds serially from the recorded initial value
  // (reduction.zig:839-863), which therefore enters a row's result exactly once; a tree of
  // per-thread accumulators that all started from it would count it once per thread.
  ENode identityOf(int rid) const {
    ENode k = constOf(rid);
    const Reducer r = static_cast<Reducer>(c.nodes[rid].sub);
    if (r == Reducer::sum) {
      k.bits = 0;
      return k;
    }
    const bool lowest = r == Reducer::max;
    switch (k.dtype) {
      case DType::f32: k.bits = lowest ? 0xff800000ull : 0x7f800000ull; break;
      case DType::f64: k.bits = lowest ? 0xfff0000000000000ull : 0x7ff0000000000000ull; break;
      case DType::f16: k.bits = lowest ? 0xfc00ull : 0x7c00ull; break;
      case DType::bf16: k.bits = lowest ? 0xff80ull : 0x7f80ull; break;
      case DType::i1: k.bits = lowest ? 0ull : 1ull; break;
      case DType::i8: k.bits = lowest ? 0x80ull : 0x7full; break;
      case DType::i16: k.bits = lowest ? 0x8000ull : 0x7fffull; break;
      case DType::i32: k.bits = lowest ? 0x80000000ull : 0x7fffffffull; break;
      case DType::i64: k.bits = lowest ? 0x8000000000000000ull : 0x7fffffffffffffffull; break;
      case DType::u8: k.bits = lowest ? 0ull : 0xffull; break;
      case DType::u16: k.bits = lowest ? 0ull : 0xffffull; break;
      case DType::u32: k.bits = lowest ? 0ull : 0xffffffffull; break;
      default: k.bits = lowest ? 0ull : ~0ull; break;
    }
    return k;
  }

  // `total` folded with the recorded initial value, the initial value on the left as in the
  // reference's serial fold; nothing to do when it is the identity the accumulators started from
  std::string withInit(int rid, const std::string& total) const {
    const size_t width = dtypeSize(c.nodes[rid].dtype);
    const uint64_t mask = width >= 8 ? ~0ull : ((1ull << (8 * width)) - 1ull);
    if (((identityOf(rid).bits ^ c.nodes[rid].bits) & mask) == 0) return total;
    return "fold<" + std::to_string(static_cast<int>(c.nodes[rid].sub)) + ", " + ctypeOf(c.nodes[rid].dtype) + ">(" +
           constLiteral(constOf(rid)) + ", " + total + ")";
  }

  // second kernel of a column-split reduction: one thread per row folds the partials in order
  // Few rows with many partials each get a warp per row: lane l folds partials l, l + 32, ... in that
  // order, a butterfly of shuffles folds the lanes, lane 0 adds the recorded start value and stores.
  // (A sum over 64 Mi elements leaves one row of several hundred partials: a single thread folding
  // them one after the other took longer than the main pass needs to read a tenth of the input.)
  static bool combineByWarp(const Cluster& c, const RowSchedule& s) { return s.splits >= 64 && c.rows <= 4096; }

  std::string generateCombine(const std::string& kname) {
    const bool by_warp = combineByWarp(c, s);
    o << kRowPrelude;
    o << "extern \"C\" __global__ void __launch_bounds__(128) " << kname << "(" << params(true) << ") {\n";
    if (by_warp)
      o << "  const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);\n  const int lane = threadIdx.x & 31;\n"
        << "  if (r >= " << c.rows << "ll) return;\n";
    else
      o << "  const long long r = (long long)blockIdx.x * 128 + threadIdx.x;\n  if (r >= " << c.rows << "ll) return;\n";
    std::vector<std::string> red_values(c.nodes.size());
    std::vector<bool> red_ready(c.nodes.size(), false);
    for (int rid : reds) {
      const std::string ty = ctypeOf(c.nodes[rid].dtype);
      const std::string op = std::to_string(static_cast<int>(c.nodes[rid].sub));
      o << "  " << ty << " comb_" << rid << ";\n  {\n    const unsigned long long* p = partials + (" << redIndex(rid)
        << "ll * " << c.rows << "ll + r) * " << s.splits << "ll;\n";
      if (by_warp) {
        o << "    " << ty << " part = " << constLiteral(identityOf(rid)) << ";\n";
        o << "    for (int sp = lane; sp < " << s.splits << "; sp += 32) part = fold<" << op << ">(part, *reinterpret_cast<const "
          << ty << "*>(p + sp));\n";
        o << "    for (int off = 16; off > 0; off >>= 1) part = fold<" << op << ">(part, __shfl_xor_sync(0xffffffffu, part, off));\n";
        o << "    comb_" << rid << " = " << withInit(rid, "part") << ";\n  }\n";
      } else {
        o << "    comb_" << rid << " = " << withInit(rid, "*reinterpret_cast<const " + ty + "*>(p)") << ";\n";
        o << "    for (int sp = 1; sp < " << s.splits << "; ++sp) comb_" << rid << " = fold<" << op << ">(comb_" << rid
          << ", *reinterpret_cast<const " << ty << "*>(p + sp));\n  }\n";
      }
      red_values[rid] = "comb_" + std::to_string(rid);
      red_ready[rid] = true;
    }
    // two sweeps: leaves/constants first, then everything that depends on the reductions
    emitReadyScalars("  ", &red_values, red_ready);
    emitReadyScalars("  ", &red_values, red_ready);
    if (by_warp) o << "  if (lane != 0) return;\n";
    for (auto& out : c.outputs) {
      const LeafRef& ref = c.leaves[out.ref];
      std::string off = indexExpr(c.extents, ref.strides, 0, c.split, "r");
      o << "  L" << out.ref << "[" << off << "] = " << storeConvert(ref.dtype, name(out.node)) << ";\n";
    }
    o << "}\n";
    return o.str();
  }
};

int floorPow2(int64_t x) {
  int p = 1;
  while (static_cast<int64_t>(p) * 2 <= x) p *= 2;
  return p;
}

}  // namespace

RowSchedule chooseRowSchedule(const Cluster& c, const ScheduleOverrides& o) {
  RowSchedule s;
  const uint32_t row_mask = c.rowMask();
  // vector width: 16 bytes per access when every column-varying buffer is contiguous along the
  // columns and every row offset keeps the alignment
  int vec = 8;
  bool gather = false;
  int max_level = 0, reds = 0;
  bool elem_out_after_reduce = false, red_after_reduce = false;
  for (const ENode& n : c.nodes) {
    max_level = std::max(max_level, n.level);
    if (n.op == ENode::Red) {
      ++reds;
      if (n.level > 1) red_after_reduce = true;
    }
  }
  std::vector<bool> is_out(c.leaves.size(), false);
  for (auto& out : c.outputs) {
    is_out[out.ref] = true;
    if ((c.leaves[out.ref].vary & ~row_mask) != 0 && c.nodes[out.node].level > 0) elem_out_after_reduce = true;
  }
  for (size_t l = 0; l < c.leaves.size(); ++l) {
    const LeafRef& leaf = c.leaves[l];
    if ((leaf.vary & ~row_mask) == 0) continue;  // read once per row as a scalar
    if (leaf.index_leaf >= 0 && (c.leaves[leaf.index_leaf].vary & ~row_mask) != 0) gather = true;  // a number per element
    int es = static_cast<int>(dtypeSize(leaf.dtype));
    vec = std::min(vec, std::max(1, 16 / es));
    int64_t expect = 1;
    for (int d = static_cast<int>(c.extents.size()) - 1; d >= c.split; --d) {
      if (c.extents[d] == 1) continue;
      if (leaf.strides[d] != expect) gather = true;
      expect *= c.extents[d];
    }
  }
  if (gather) vec = 1;
  auto rowsAligned = [&](int v) {
    for (const LeafRef& leaf : c.leaves) {
      if ((leaf.vary & ~row_mask) == 0) continue;
      if (leaf.index_leaf >= 0 && leaf.index_stride % v != 0) return false;
      for (int d = 0; d < c.split; ++d)
        if (c.extents[d] != 1 && leaf.strides[d] % v != 0) return false;
    }
    return true;
  };
  while (vec > 1 && (c.cols % vec != 0 || !rowsAligned(vec))) vec /= 2;
  s.vec = vec;
  const int64_t vectors = (c.cols + vec - 1) / vec;  // vector accesses per row
  const bool multipass = max_level >= 2 || (max_level >= 1 && elem_out_after_reduce);
  // A single-pass reduction whose buffers run along the kept (row) axes, not along the reduced one: a
  // fold over a leading axis of a row-major buffer (a column sum, the gradient of a broadcast).  One
  // thread per row then makes the 256 threads of a CTA read 256 neighbouring elements per step, where
  // 256 threads on one row would each touch a line of their own (measured on a sum over the 16384 rows
  // of f32[16384, 4096]: 1.10 TB/s with 256 threads per row, 5.06 TB/s with one).
  bool rows_fast = gather && reds > 0 && !multipass;
  {
    int dr = -1, dc = -1;
    for (int d = 0; d < c.split; ++d) if (c.extents[d] != 1) dr = d;
    for (int d = c.split; d < static_cast<int>(c.extents.size()); ++d) if (c.extents[d] != 1) dc = d;
    if (dr < 0 || dc < 0) rows_fast = false;
    bool any = false;
    for (const LeafRef& leaf : c.leaves) {
      if (!rows_fast) break;
      if ((leaf.vary & ~row_mask) == 0 || (leaf.vary & row_mask) == 0) continue;   // varies along one side only
      any = true;
      if (leaf.strides[dr] != 1 || leaf.strides[dc] == 1) rows_fast = false;
    }
    if (!any) rows_fast = false;
  }
  // a multi-pass row is kept in registers whenever it fits (<= 32 elements per thread at
  // 1024 threads); single-pass rows stream with 256 threads
  int tpr;
  if (o.threads_per_row > 0) tpr = o.threads_per_row;
  else if (rows_fast) tpr = 1;
  else {
    tpr = floorPow2(std::max<int64_t>(1, vectors / 4));
    tpr = std::min(tpr, 256);
    const int64_t max_vpt = std::max(1, 32 / vec);
    if (multipass && vectors > static_cast<int64_t>(tpr) * max_vpt) {
      while (tpr < 1024 && vectors > static_cast<int64_t>(tpr) * max_vpt) tpr *= 2;
    }
  }
  s.tpr = tpr;
  const int64_t max_vpt = std::max(1, 32 / vec);
  int64_t vpt = (vectors + tpr - 1) / tpr;
  if (o.vectors_per_thread > 0) vpt = o.vectors_per_thread;
  if (vpt <= max_vpt && o.vectors_per_thread == 0) {
    s.vpt = static_cast<int>(vpt);
    s.chunks = 1;
  } else {
    s.vpt = o.vectors_per_thread > 0 ? o.vectors_per_thread : static_cast<int>(std::min<int64_t>(4, max_vpt));
    const int64_t per_chunk = static_cast<int64_t>(tpr) * s.vpt;
    s.chunks = (vectors + per_chunk - 1) / per_chunk;
  }
  s.rpc = std::max(1, 256 / tpr);
  while (s.rpc > 1 && s.rpc / 2 >= c.rows) s.rpc /= 2;
  // column splits: only when a row is a single pass (no value computed after a reduction is
  // needed per element) and the rows alone cannot fill the GPU
  const bool splittable = !elem_out_after_reduce && !red_after_reduce && s.chunks > 1;
  const int64_t ctas = (c.rows + s.rpc - 1) / s.rpc;
  if (o.column_splits > 0 && splittable) s.splits = static_cast<int>(std::min<int64_t>(o.column_splits, s.chunks));
  else if (splittable && reds == 0 && ctas < 8 * o.sm_count) {
    // nothing to combine afterwards: one chunk per CTA (measured on a + b * c over 64 Mi f32: 4.47 TB/s
    // with two CTAs per SM looping over their chunks, 7.05 TB/s with a CTA per chunk)
    s.splits = static_cast<int>(std::min<int64_t>(s.chunks, 65535));
  } else if (splittable && rows_fast && o.threads_per_row == 0 && ctas < 7 * o.sm_count) {
    // about seven CTAs per SM, at least 64 elements of the fold per thread
    int64_t want = (7 * o.sm_count + ctas - 1) / ctas;
    want = std::min<int64_t>(want, std::max<int64_t>(1, c.cols / 64));
    s.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, s.chunks, 65535})));
  } else if (splittable && ctas < 2 * o.sm_count) {
    // six CTAs per SM where the partials are then folded by a warp per row (measured on the sum of
    // 64 Mi f32: 4.6 TB/s with two CTAs per SM, 5.9 TB/s with six), two otherwise
    int64_t want = ((c.rows <= 4096 ? 6 : 2) * o.sm_count + ctas - 1) / ctas;
    s.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, s.chunks, 65535})));
  }
  if (s.splits > 1) {
    // whole chunks per split; drop splits that would be empty
    const int64_t per = (s.chunks + s.splits - 1) / s.splits;
    s.splits = static_cast<int>((s.chunks + per - 1) / per);
  }
  (void)reds;
  // Rows held in registers with at most 16 elements per thread: ask for 1536 resident threads per
  // SM (registers capped at 40 per thread).  Measured on the softmax + layer-norm row program:
  // 6 CTAs of 256 threads reach 86% of the HBM copy rate, the uncapped build (47 registers, 5
  // CTAs) 81%, and a 32-register cap spills and drops to 64%.
  if (o.row_min_blocks > 0) s.min_blocks = o.row_min_blocks;
  else if (s.chunks == 1 && s.vec * s.vpt <= 16 && s.tpr * s.rpc >= 128) s.min_blocks = 1536 / (s.tpr * s.rpc);
  // Rows per thread: two neighbouring rows share the loads (and whatever else does not vary along
  // the rows) when the kernel qualifies and enough CTAs remain to fill the GPU several times over.
  // ACCY_B200_ROWS_PER_THREAD=<n> overrides the choice (1 turns it off).
  if (RowGen::blockable(c, s)) {
    const int64_t ctas_now = (c.rows + s.rpc - 1) / s.rpc;
    s.rpt = ctas_now / 2 >= 8 * static_cast<int64_t>(o.sm_count) ? 2 : 1;
    if (const char* e = std::getenv("ACCY_B200_ROWS_PER_THREAD")) {
      const int want = std::atoi(e);
      if (want >= 1 && want <= 8) s.rpt = want;
    }
    // measured on the mismatch program (8192 x 65536): one row per thread 1631 Gpair/s, two rows
    // 1717, two rows with 768 resident threads per SM requested of the compiler 1750, four rows 1739
    if (s.rpt > 1 && o.row_min_blocks == 0 && s.tpr * s.rpc <= 768) s.min_blocks = 768 / (s.tpr * s.rpc);
  }
  return s;
}

void emitRowKernels(const Cluster& c, const RowSchedule& s, const std::string& name, Plan& plan,
                    const std::string& label) {
  if (c.rows > 0x7fffffffll) throw PlanError("more than 2^31-1 rows in one fused region");
  bool has_reds = false, f32_math = false;
  for (const ENode& n : c.nodes) {
    if (n.op == ENode::Red) has_reds = true;
    if (n.dtype == DType::f32 || n.dtype == DType::f64) f32_math = true;
  }
  RowGen gen(c, s);
  KernelSource ks;
  ks.name = name;
  ks.family = "row";
  ks.source = s.rpt > 1 ? gen.generateBlocked(name) : gen.generateMain(name);
  if (f32_math) ks.options.push_back("--fmad=false");
  plan.kernels.push_back(ks);
  Launch launch;
  launch.kernel = static_cast<int>(plan.kernels.size()) - 1;
  launch.grid[0] = static_cast<uint32_t>((c.rows + static_cast<int64_t>(s.rpc) * s.rpt - 1) / (static_cast<int64_t>(s.rpc) * s.rpt));
  launch.grid[1] = static_cast<uint32_t>(s.splits);
  launch.block[0] = static_cast<uint32_t>(s.tpr * s.rpc);
  launch.label = label;
  for (const LeafRef& leaf : c.leaves) {
    KernelArg a;
    a.slot = leaf.slot;
    launch.args.push_back(a);
  }
  const bool two_pass = s.splits > 1 && has_reds;
  int scratch = -1;
  if (two_pass) {
    int reds = 0;
    for (const ENode& n : c.nodes) if (n.op == ENode::Red) ++reds;
    Slot sc;
    sc.role = Slot::Scratch;
    sc.bytes = static_cast<size_t>(reds) * c.rows * s.splits * 8;
    plan.slots.push_back(sc);
    scratch = static_cast<int>(plan.slots.size()) - 1;
    KernelArg a;
    a.slot = scratch;
    launch.args.push_back(a);
  }
  const std::vector<KernelArg> buffers = launch.args;
  if (gen.packed) {
    // the zero behind mul2_own_rounding: a launch argument, so no compiler pass can fold it
    KernelArg zero;
    zero.is_slot = false;
    zero.scalar = 0;
    zero.scalar_bytes = 8;
    launch.args.push_back(zero);
  }
  plan.launches.push_back(launch);
  if (two_pass) {
    RowGen comb(c, s);
    KernelSource cs;
    cs.name = name + "_combine";
    cs.family = "row_combine";
    cs.source = comb.generateCombine(cs.name);
    if (f32_math) cs.options.push_back("--fmad=false");
    plan.kernels.push_back(cs);
    Launch l2;
    l2.kernel = static_cast<int>(plan.kernels.size()) - 1;
    l2.grid[0] = static_cast<uint32_t>(RowGen::combineByWarp(c, s) ? (c.rows + 3) / 4 : (c.rows + 127) / 128);
    l2.block[0] = 128;
    l2.label = label + " (combine)";
    l2.args = buffers;
    plan.launches.push_back(l2);
  }
}

}  // namespace accy
