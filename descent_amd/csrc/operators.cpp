// Sequence-model operators: what a descriptor may ask for, and the defines under which its kernel template is compiled.
#include "codegen.hpp"

#include <algorithm>
#include <cstdio>
#include <sstream>

namespace dsc {

namespace {

using std::string;
using std::to_string;

const char* const kNames[] = {"RmsNorm", "RmsNormGrad", "Rotary", "Attention", "AttentionJoin", "AttentionGradQuery", "AttentionGradKeyValue",
                              "DualMatMul", "GatedGrad", "AttentionGradSinks", "CacheAppend"};

float as_float(uint32_t bits) {
    float f;
    std::memcpy(&f, &bits, 4);
    return f;
}
bool is_finite(uint32_t bits) { return (bits & 0x7f800000u) != 0x7f800000u; }

dsc_shape shape_of(std::initializer_list<int64_t> dims) {
    dsc_shape s{};
    for (int64_t d : dims) s.dims[s.rank++] = d;
    return s;
}

// An operand as the kernels address it: offset and strides in elements.
struct Operand {
    int64_t base = 0, stride[DSC_MAX_DIM] = {0};
    explicit Operand(const dsc_view& v) { affine_form(v, &base, stride); }
    // elements of `axis` 16-byte aligned in runs of four, whatever the other coordinates
    bool quads(const dsc_view& v, int axis) const {
        if (base % 4 != 0 || stride[axis] != 1) return false;
        for (int j = 0; j < v.out_shape.rank; ++j)
            if (j != axis && v.out_shape.dims[j] > 1 && stride[j] % 4 != 0) return false;
        return true;
    }
};

string check_strided(const dsc_view& v, bool either_axis) {
    int64_t base, coef[DSC_MAX_DIM];
    if (!affine_form(v, &base, coef)) return "the view leaves its array (clamped)";
    const int r = v.out_shape.rank;
    for (int j = 0; j < r; ++j)
        if (coef[j] < 0) return "negative strides";
    auto beside = [&](int j) { return coef[j] == 1 || v.out_shape.dims[j] == 1; };
    if (beside(r - 1) || (either_axis && r >= 2 && beside(r - 2))) return "";
    return "elements of the last axis do not lie side by side";
}

bool is_shape(const dsc_shape& s, std::initializer_list<int64_t> dims) { return same_shape(s, shape_of(dims)); }

}  // namespace

string operator_label(const dsc_kernel_desc& d) {
    string name = kNames[d.kind - DSC_KERNEL_RMS_NORM];
    if (d.kind == DSC_KERNEL_DUAL_MATMUL) name += d.op_int[0] == DSC_DUAL_GATED ? " gated" : d.op_int[0] == DSC_DUAL_SUM ? " sum" : " both";
    return name + " " + shape_str(d.shape);
}

std::vector<dsc_shape> operator_results(const dsc_kernel_desc& d) {
    const dsc_view* in = d.inputs;
    switch (d.kind) {
    case DSC_KERNEL_RMS_NORM: return {in[0].out_shape, in[0].out_shape, shape_of({in[0].out_shape.dims[0]})};
    case DSC_KERNEL_RMS_NORM_GRAD: return {in[0].out_shape, shape_of({d.op_int[1], in[0].out_shape.dims[1]})};
    case DSC_KERNEL_ROTARY: return {in[0].out_shape};
    case DSC_KERNEL_ATTENTION: {
        const int64_t* q = in[0].out_shape.dims;
        if (d.op_int[3] == 1) return {in[0].out_shape, shape_of({q[0], q[1], q[2]})};
        return {shape_of({d.op_int[3], q[0], q[1], q[2], q[3]}), shape_of({d.op_int[3], q[0], q[1], q[2]})};
    }
    case DSC_KERNEL_ATTENTION_JOIN: {
        const int64_t* p = in[0].out_shape.dims;
        return {shape_of({p[1], p[2], p[3], p[4]}), shape_of({p[1], p[2], p[3]})};
    }
    case DSC_KERNEL_ATTENTION_GRAD_QUERY: {
        const int64_t* q = in[0].out_shape.dims;
        return {in[0].out_shape, shape_of({q[0], q[1], q[2]})};
    }
    case DSC_KERNEL_ATTENTION_GRAD_KEY_VALUE: return {in[1].out_shape, in[2].out_shape};
    case DSC_KERNEL_ATTENTION_GRAD_SINKS: {
        const int64_t* k = in[1].out_shape.dims;
        const dsc_shape far = shape_of({d.op_int[3], k[0], std::min<int64_t>(d.op_int[1], k[1]), k[2], k[3]});
        return {far, far};
    }
    case DSC_KERNEL_DUAL_MATMUL: {
        const int64_t m = in[0].out_shape.dims[0], n = in[d.n_inputs - 1].out_shape.dims[1];
        const dsc_shape out = d.op_int[2] > 1 ? shape_of({d.op_int[2], m, n}) : shape_of({m, n});
        if (d.op_int[0] == DSC_DUAL_GATED) return {out, out, out};
        if (d.op_int[0] == DSC_DUAL_SUM) return {out};
        return {out, out};
    }
    case DSC_KERNEL_GATED_GRAD: return {in[0].out_shape, in[0].out_shape};
    case DSC_KERNEL_CACHE_APPEND: return {shape_of({in[0].out_shape.dims[0], d.op_int[0], in[0].out_shape.dims[2]})};
    default: return {};
    }
}

string validate_operator(const dsc_kernel_desc& d) {
    const string name = string(kNames[d.kind - DSC_KERNEL_RMS_NORM]) + ": ";
    const dsc_view* in = d.inputs;
    const int32_t* op = d.op_int;
    auto dims = [&](int i) { return in[i].out_shape.dims; };
    auto rank = [&](int i) { return in[i].out_shape.rank; };
    auto ranks = [&](std::initializer_list<int> want) {
        int i = 0;
        for (int r : want)
            if (rank(i++) != r) return false;
        return true;
    };
    // operands [0, strided) may be strided, the others are dense; `places` u32 [batch] arrays come last
    auto views = [&](std::initializer_list<int> strided, bool either_axis) -> string {
        for (int i = 0; i < d.n_inputs; ++i) {
            if (std::find(strided.begin(), strided.end(), i) != strided.end()) {
                const string e = check_strided(in[i], either_axis);
                if (!e.empty()) return "operand " + to_string(i) + ": " + e;
            } else if (!is_contiguous(in[i])) {
                return "operand " + to_string(i) + " must be dense";
            }
        }
        return "";
    };
    for (int i = 0; i < d.n_inputs; ++i)
        for (int j = 0; j < rank(i); ++j)
            if (dims(i)[j] >= (int64_t(1) << 30)) return name + "extent of 2^30 or more";
    for (int i = 0; i < 2; ++i)
        if (!is_finite(d.op_float[i])) return name + "attribute is not finite";
    string e;
    switch (d.kind) {
    case DSC_KERNEL_RMS_NORM: {
        if (op[0] < 0 || op[0] > 1 || d.n_inputs != 2 + op[0]) return name + "wrong number of operands";
        if (!ranks({2, 1}) || dims(1)[0] != dims(0)[1]) return name + "weight does not fit";
        if (op[0] && !same_shape(in[2].out_shape, in[0].out_shape)) return name + "residual differs in shape";
        if (as_float(d.op_float[0]) < 0) return name + "negative epsilon";
        e = views({0, 2}, false);
        break;
    }
    case DSC_KERNEL_RMS_NORM_GRAD: {
        if (op[0] < 0 || op[0] > 1 || d.n_inputs != 4 + op[0]) return name + "wrong number of operands";
        if (!ranks({2, 1, 1, 2})) return name + "wrong ranks";
        if (dims(1)[0] != dims(0)[0] || dims(2)[0] != dims(0)[1] || !same_shape(in[3].out_shape, in[0].out_shape)) return name + "shapes differ";
        if (op[0] && !same_shape(in[4].out_shape, in[0].out_shape)) return name + "gradient of the sum differs in shape";
        if (op[1] < 1 || op[1] > dims(0)[0]) return name + "between one partial and one per row";
        e = views({0, 3, 4}, false);
        break;
    }
    case DSC_KERNEL_ROTARY: {
        if (op[2] < 0 || op[2] > 2 || d.n_inputs != 2 + (op[2] > 0)) return name + "wrong number of operands";
        if (!ranks({4, 1}) || 2 * dims(1)[0] > dims(0)[3]) return name + "more pairs than a head holds";
        if (op[0] < 0 || op[0] > 1 || op[1] < 0 || op[1] > 1) return name + "unknown layout or direction";
        if (dims(1)[0] > 4096) return name + "kernel too large: more than 4096 pairs";
        if (op[2] == 1 && !is_shape(in[2].out_shape, {dims(0)[0]})) return name + "positions must be [batch]";
        if (op[2] == 2 && !is_shape(in[2].out_shape, {dims(0)[0], dims(0)[1]})) return name + "positions must be [batch, tokens]";
        e = views({0}, false);
        break;
    }
    case DSC_KERNEL_ATTENTION:
    case DSC_KERNEL_ATTENTION_GRAD_QUERY:
    case DSC_KERNEL_ATTENTION_GRAD_SINKS:
    case DSC_KERNEL_ATTENTION_GRAD_KEY_VALUE: {
        const bool joins = d.kind == DSC_KERNEL_ATTENTION_GRAD_KEY_VALUE && op[3] != 0;
        const int arrays = d.kind == DSC_KERNEL_ATTENTION ? 3 : joins ? 8 : 6;
        if (op[2] < 0 || op[2] > 3 || d.n_inputs != arrays + (op[2] & 1) + (op[2] >> 1)) return name + "wrong number of operands";
        if (!ranks({4, 4, 4})) return name + "queries, keys and values have four axes";
        const int64_t *q = dims(0), *k = dims(1);
        if (!same_shape(in[1].out_shape, in[2].out_shape) || q[0] != k[0] || q[3] != k[3]) return name + "queries, keys and values do not fit";
        if (q[2] % k[2] != 0) return name + "query heads do not share the key heads evenly";
        if (q[3] > 256) return name + "heads of more than 256 elements";
        if (op[0] < 0 || op[1] < 0) return name + "negative window or sinks";
        if (!(op[2] & 1) && q[1] > k[1]) return name + "more queries than keys need starts";
        // (kernels count rows in 32 bits and round them up to tiles of up to 256)
        if (q[1] * (q[2] / k[2]) > (int64_t(1) << 31) - 512) return name + "kernel too large: rows of a key head";
        for (int i = arrays; i < d.n_inputs; ++i)
            if (!is_shape(in[i].out_shape, {q[0]})) return name + "starts and lengths must be [batch]";
        if (d.kind == DSC_KERNEL_ATTENTION) {
            if (op[3] < 1 || op[3] > 64) return name + "between 1 and 64 splits";
            e = views({0, 1, 2}, false);
        } else if (d.kind == DSC_KERNEL_ATTENTION_GRAD_QUERY) {
            if (!same_shape(in[3].out_shape, in[0].out_shape) || !same_shape(in[4].out_shape, in[0].out_shape) || !is_shape(in[5].out_shape, {q[0], q[1], q[2]}))
                return name + "output, its gradient or the denominators do not fit";
            e = views({0, 1, 2, 3, 4}, false);
        } else {
            if (!same_shape(in[3].out_shape, in[0].out_shape) || !is_shape(in[4].out_shape, {q[0], q[1], q[2]}) || !is_shape(in[5].out_shape, {q[0], q[1], q[2]}))
                return name + "the output's gradient or the rows' sums do not fit";
            if (op[3] < 0 || op[3] > 64 || (d.kind == DSC_KERNEL_ATTENTION_GRAD_SINKS && op[3] == 0)) return name + "between 1 and 64 pieces";
            if (op[3] && (op[0] == 0 || op[1] == 0)) return name + "pieces without a window and sinks";
            for (int i = 6; joins && i < 8; ++i)
                if (!is_shape(in[i].out_shape, {op[3], k[0], std::min<int64_t>(op[1], k[1]), k[2], k[3]})) return name + "the sinks' pieces do not fit";
            e = views({0, 1, 2, 3}, false);
        }
        break;
    }
    case DSC_KERNEL_ATTENTION_JOIN: {
        if (d.n_inputs != 2 || !ranks({5, 4})) return name + "takes partial outputs and denominators";
        for (int j = 0; j < 4; ++j)
            if (dims(0)[j] != dims(1)[j]) return name + "partial outputs and denominators do not fit";
        e = views({}, false);
        break;
    }
    case DSC_KERNEL_DUAL_MATMUL: {
        if (op[0] < 0 || op[0] > 2 || op[1] < 0 || op[1] > 3) return name + "unknown mode or activation";
        if (op[2] < 1 || op[2] > 64 || (op[0] == DSC_DUAL_GATED && op[2] != 1)) return name + "between 1 and 64 splits, one for a gated product";
        const bool sum = op[0] == DSC_DUAL_SUM;
        if (d.n_inputs != (sum ? 4 : 3)) return name + "wrong number of operands";
        for (int i = 0; i < d.n_inputs; ++i)
            if (rank(i) != 2) return name + "operands have two axes";
        const int b = sum ? 2 : 1;
        if (sum && !same_shape(in[0].out_shape, in[1].out_shape)) return name + "left operands differ in shape";
        if (!same_shape(in[b].out_shape, in[b + 1].out_shape)) return name + "right operands differ in shape";
        if (dims(0)[1] != dims(b)[0]) return name + "inner extents differ";
        e = views({0, 1, 2, 3}, true);
        break;
    }
    case DSC_KERNEL_GATED_GRAD: {
        if (op[0] < 0 || op[0] > 3 || d.n_inputs != 3) return name + "unknown activation or wrong number of operands";
        if (!same_shape(in[0].out_shape, in[1].out_shape) || !same_shape(in[0].out_shape, in[2].out_shape)) return name + "operands differ in shape";
        e = views({}, false);
        break;
    }
    case DSC_KERNEL_CACHE_APPEND: {
        if (d.n_inputs != 2 || !ranks({3, 1}) || dims(1)[0] != dims(0)[0]) return name + "takes rows and a start per sequence";
        if (op[0] < 1) return name + "capacity must be positive";
        e = views({0}, false);
        break;
    }
    default: return "unknown kernel kind";
    }
    if (!e.empty()) return name + e;
    const std::vector<dsc_shape> results = operator_results(d);
    if (!same_shape(d.shape, results[0])) return name + "shape is not the first result's";
    if (d.n_outputs < 1 || !d.outputs || d.outputs[0] != 0) return name + "the first result is always written";
    for (int o = 1; o < d.n_outputs; ++o)
        if (d.outputs[o] <= d.outputs[o - 1] || d.outputs[o] >= (int)results.size()) return name + "results must be listed in ascending order";
    return "";
}

namespace {

string num(int64_t v) { return "(" + to_string((long long)v) + "ll)"; }

struct Defines {
    std::ostringstream text;
    void set(const string& name, int64_t v) { text << "#define " << name << " " << (v < 0 ? "(" : "") << v << (v < 0 ? ")" : "") << "\n"; }
    void set64(const string& name, int64_t v) { text << "#define " << name << " " << num(v) << "\n"; }
    void set_float(const string& name, float v) {
        char buf[64];
        std::snprintf(buf, sizeof buf, "%af", (double)v);
        text << "#define " << name << " (" << buf << ")\n";
    }
};

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }


string assemble(const FusedKernel& fk, const Defines& defs, const char* text, const string& entry, const string& function,
                const std::vector<string>& args, int64_t grid, int block, int min_waves, Generated* g) {
    if (grid >= (int64_t(1) << 31)) return "kernel too large: more than 2^31 workgroups";
    std::ostringstream k;
    k << kPreludeSource << "\n" << defs.text.str() << text << "\nextern \"C\" __global__ __launch_bounds__(" << block << ", " << min_waves << ") void "
      << entry << "(";
    for (int i = 0; i < fk.n_buffers; ++i) k << (fk.buffer_is_output[i] ? "float* b" : "const float* b") << i << ", ";
    k << "const uint* seed_cell, uint seed_value) {\n    " << function << "(";
    for (size_t i = 0; i < args.size(); ++i) k << (i ? ", " : "") << args[i];
    k << ");\n}\n";
    g->source = k.str();
    g->entry = entry;
    g->grid = (unsigned)grid;
    g->block = (unsigned)block;
    return "";
}

// the buffer that takes result `index`, or a null pointer
string result_arg(const FusedKernel& fk, int index) {
    const dsc_kernel_desc& d = fk.main.raw();
    for (int o = 0; o < d.n_outputs; ++o)
        if (d.outputs[o] == index) return "b" + to_string(fk.outputs[o]);
    return "(float*)nullptr";
}
string input_arg(const FusedKernel& fk, int i, bool u32 = false) {
    const string b = "b" + to_string(fk.inputs[i].buffer);
    return u32 ? "(const uint*)" + b : b;
}

string gen_rms_norm(const FusedKernel& fk, Generated* g) {
    const dsc_kernel_desc& d = fk.main.raw();
    const bool grad = d.kind == DSC_KERNEL_RMS_NORM_GRAD;
    const int64_t rows = d.inputs[0].out_shape.dims[0], n = d.inputs[0].out_shape.dims[1];
    // the [rows, n] operands: x and the residual; sum, d norm and d sum
    std::vector<int> wide = grad ? std::vector<int>{0, 3} : std::vector<int>{0};
    if (d.op_int[0]) wide.push_back(grad ? 4 : 2);
    bool quads = n % 4 == 0;
    for (int i : wide) quads = quads && Operand(d.inputs[i]).quads(d.inputs[i], 1);
    const int vec = quads ? 4 : 1;
    // a thread holds at most 16 elements of a row (8 in the gradient, which keeps four arrays of them) as long as
    // 1024 threads suffice.  Up to 32 it still keeps them: 2048 x 16384 (33.6 M elements, with a residual) takes 98 us
    // forward and 124 back, 1024 x 32768 104 and 209 (the gradient spills 136 registers), and 512 x 65536 in two passes
    // 143 and 172.
    const int64_t most = grad ? 8 : 16;
    int tpr = 64;
    while (tpr < 1024 && up(n, (int64_t)tpr * vec) * vec > most) tpr *= 2;
    const int64_t each = up(n, (int64_t)tpr * vec);
    const bool keep = each * vec <= 32;
    if (!keep) tpr = 1024;
    const int block = std::max(tpr, 256);
    const int groups = block / tpr;
    Defines def;
    def.set64("RN_ROWS", rows);
    def.set("RN_N", n);
    def.set("RN_VEC", vec);
    def.set("RN_TPR", tpr);
    def.set("RN_BLOCK", block);
    def.set("RN_E", up(n, (int64_t)tpr * vec));
    def.set("RN_KEEP", keep ? 1 : 0);
    const char* prefix[] = {"RN_X", "RN_R", "RN_S"};
    for (int i = 0; i < 3; ++i) {
        const Operand o(d.inputs[i < (int)wide.size() ? wide[i] : 0]);
        def.set64(string(prefix[i]) + "_BASE", o.base);
        def.set64(string(prefix[i]) + "_STRIDE", o.stride[0]);
    }
    def.set_float("RN_EPSILON", as_float(grad ? 0u : d.op_float[0]));
    def.set("RN_PARTIALS", grad ? d.op_int[1] : 1);
    g->note = string("row in ") + (keep ? "registers" : "two passes") + " of " + to_string(tpr) + " threads x" + to_string(vec);
    const string size = "_m" + to_string((long long)rows) + "_n" + to_string((long long)n);
    const double cells = 4.0 * (double)rows * (double)n;
    if (!grad) {
        g->algo_bytes = cells * (1.0 + (double)wide.size() + (result_arg(fk, 1)[0] == 'b' ? 1.0 : 0.0)) + 4.0 * (double)n;
        return assemble(fk, def, kRmsNormSource, "dsc_rms_norm" + size, "rms_norm",
                        {input_arg(fk, 0), input_arg(fk, 1), d.op_int[0] ? input_arg(fk, 2) : "(const float*)nullptr", result_arg(fk, 0), result_arg(fk, 1),
                         result_arg(fk, 2)},
                        up(rows, groups), block, 1, g);
    }
    g->algo_bytes = cells * (1.0 + (double)wide.size()) + 4.0 * (double)n;
    return assemble(fk, def, kRmsNormSource, "dsc_rms_norm_grad" + size, "rms_norm_grad",
                    {input_arg(fk, 0), input_arg(fk, 1), input_arg(fk, 2), input_arg(fk, 3), d.op_int[0] ? input_arg(fk, 4) : "(const float*)nullptr",
                     result_arg(fk, 0), result_arg(fk, 1)},
                    d.op_int[1], block, 1, g);
}

string gen_rotary(const FusedKernel& fk, Generated* g) {
    const dsc_kernel_desc& d = fk.main.raw();
    const int64_t* x = d.inputs[0].out_shape.dims;
    const int64_t tokens = x[0] * x[1], heads = x[2], dim = x[3], pairs = d.inputs[1].out_shape.dims[0];
    const Operand o(d.inputs[0]);
    const bool half = d.op_int[0] == DSC_ROTARY_HALF;
    const int vec = o.quads(d.inputs[0], 3) && dim % 4 == 0 && (half ? pairs % 4 == 0 : pairs % 2 == 0) ? 4 : 1;
    // A workgroup's share: about 1024 units (a unit is a lane's one load and store, two of each in the half layout), so
    // that its threads do four each behind the angles; with fewer than 512 workgroups down to 256 units, first fewer
    // tokens, then fewer heads.
    const int64_t units = (half ? pairs / vec : vec == 4 ? pairs / 2 : pairs) + (dim - 2 * pairs) / vec;
    int64_t tok = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(tokens, 4096 / std::max<int64_t>(1, pairs)), 1024 / (heads * units)));
    while (tok > 1 && up(tokens, tok) < 512 && tok * heads * units > 256) tok = up(tok, 2);
    int64_t each = std::min(heads, std::max<int64_t>(1, 1024 / units));
    while (each > 1 && up(tokens, tok) * up(heads, each) < 512 && tok * each * units > 256) each = up(each, 2);
    Defines def;
    def.set("RO_ROTARY", 1);
    def.set64("RO_TOKENS", tokens);
    def.set64("RO_T", x[1]);
    def.set("RO_HEADS", heads);
    def.set("RO_DIM", dim);
    def.set("RO_PAIRS", pairs);
    def.set("RO_HALF", half ? 1 : 0);
    def.set("RO_INVERSE", d.op_int[1]);
    def.set("RO_RANK", d.op_int[2]);
    def.set_float("RO_MAGNITUDE", as_float(d.op_float[0]));
    def.set("RO_VEC", vec);
    def.set("RO_TOK", tok);
    def.set("RO_HEADS_EACH", each);
    def.set("RO_HEAD_PARTS", up(heads, each));
    def.set64("RO_BASE", o.base);
    def.set64("RO_SB", o.stride[0]);
    def.set64("RO_ST", o.stride[1]);
    def.set64("RO_SH", o.stride[2]);
    g->note = "tokens " + to_string((long long)tok) + " heads " + to_string((long long)each) + " per workgroup x" + to_string(vec);
    g->algo_bytes = 8.0 * (double)(tokens * heads) * (double)dim;
    return assemble(fk, def, kRotarySource, "dsc_rotary_n" + to_string((long long)element_count(d.shape)), "rotary",
                    {input_arg(fk, 0), input_arg(fk, 1), d.op_int[2] ? input_arg(fk, 2, true) : "(const uint*)nullptr", result_arg(fk, 0)},
                    up(tokens, tok) * up(heads, each), 256, 1, g);
}

string gen_cache_append(const FusedKernel& fk, Generated* g) {
    const dsc_kernel_desc& d = fk.main.raw();
    const int64_t* x = d.inputs[0].out_shape.dims;
    const Operand o(d.inputs[0]);
    const int vec = x[2] % 4 == 0 && o.quads(d.inputs[0], 2) ? 4 : 1;
    const int64_t units = x[0] * x[1] * (x[2] / vec);
    Defines def;
    def.set64("CA_UNITS", units);
    def.set64("CA_TOKENS", x[1]);
    def.set64("CA_CAPACITY", d.op_int[0]);
    def.set64("CA_WIDTH", x[2]);
    def.set("CA_VEC", vec);
    def.set64("CA_BASE", o.base);
    def.set64("CA_SB", o.stride[0]);
    def.set64("CA_ST", o.stride[1]);
    g->note = "x" + to_string(vec);
    g->algo_bytes = 8.0 * (double)(x[0] * x[1]) * (double)x[2];
    return assemble(fk, def, kRotarySource, "dsc_cache_append_n" + to_string((long long)(x[0] * x[1] * x[2])), "cache_append",
                    {input_arg(fk, 0), input_arg(fk, 1, true), result_arg(fk, 0)}, up(units, 256), 256, 1, g);
}

string gen_attention(const FusedKernel& fk, Generated* g) {
    const dsc_kernel_desc& d = fk.main.raw();
    Defines def;
    if (d.kind == DSC_KERNEL_ATTENTION_JOIN) {
        const int64_t* p = d.inputs[0].out_shape.dims;
        for (const char* name : {"AT_S", "AT_G", "AT_WINDOW", "AT_SINKS", "AT_START", "AT_LENGTH"}) def.set(name, 1);
        def.set("AT_SPLITS", p[0]);
        def.set("AT_B", p[1]);
        def.set("AT_T", p[2]);
        def.set("AT_H", p[3]);
        def.set("AT_D", p[4]);
        def.set("AT_DP", up(p[4], 16) * 16);
        def.set("AT_VEC", 0);
        def.set_float("AT_SCALE", 1.0f);
        def.set("AT_JOIN", 1);
        const int64_t cells = element_count(d.shape);
        g->algo_bytes = 4.0 * (double)cells * (double)(p[0] + 1);
        g->note = to_string((long long)p[0]) + " pieces";
        return assemble(fk, def, kAttentionSource, "dsc_attention_join_n" + to_string((long long)cells), "attention_join",
                        {input_arg(fk, 0), input_arg(fk, 1), result_arg(fk, 0), result_arg(fk, 1)}, up(cells, 256), 256, 1, g);
    }
    const bool forward = d.kind == DSC_KERNEL_ATTENTION, grad_q = d.kind == DSC_KERNEL_ATTENTION_GRAD_QUERY;
    const int64_t *q = d.inputs[0].out_shape.dims, *k = d.inputs[1].out_shape.dims;
    const int64_t dim = q[3], dp = up(dim, 16) * 16, rows = q[1] * (q[2] / k[2]);
    const int32_t* op = d.op_int;
    def.set("AT_B", q[0]);
    def.set("AT_T", q[1]);
    def.set("AT_S", k[1]);
    def.set("AT_H", q[2]);
    def.set("AT_G", k[2]);
    def.set("AT_D", dim);
    def.set("AT_DP", dp);
    def.set("AT_WINDOW", op[0]);
    def.set("AT_SINKS", std::min<int64_t>(op[1], k[1]));  // (kernels round it up to tiles in 32 bits)
    def.set_float("AT_SCALE", as_float(d.op_float[0]));
    def.set("AT_START", op[2] & 1);
    def.set("AT_LENGTH", op[2] >> 1);
    def.set("AT_SPLITS", forward ? op[3] : 1);
    // which operand is which
    std::vector<std::pair<const char*, int>> strided = {{"AT_Q", 0}, {"AT_K", 1}, {"AT_V", 2}};
    if (grad_q) strided.push_back({"AT_O", 3});
    if (!forward) strided.push_back({"AT_DO", grad_q ? 4 : 3});
    bool quads = dim % 4 == 0;
    for (auto& s : strided) {
        const Operand o(d.inputs[s.second]);
        quads = quads && o.quads(d.inputs[s.second], 3);
        def.set64(string(s.first) + "_BASE", o.base);
        def.set64(string(s.first) + "_B", o.stride[0]);
        def.set64(string(s.first) + "_T", o.stride[1]);
        def.set64(string(s.first) + "_H", o.stride[2]);
    }
    def.set("AT_VEC", quads ? 1 : 0);
    const bool sinks = d.kind == DSC_KERNEL_ATTENTION_GRAD_SINKS, joins = !forward && !grad_q && !sinks && op[3];
    def.set("AT_PIECES", forward || grad_q ? 0 : op[3]);
    const int arrays = forward ? 3 : joins ? 8 : 6;
    const string start = op[2] & 1 ? input_arg(fk, arrays, true) : "(const uint*)nullptr";
    const string length = op[2] & 2 ? input_arg(fk, arrays + (op[2] & 1), true) : "(const uint*)nullptr";
    const string size = "_b" + to_string((long long)q[0]) + "_t" + to_string((long long)q[1]) + "_s" + to_string((long long)k[1]) + "_h" +
                        to_string((long long)q[2]) + "_g" + to_string((long long)k[2]) + "_d" + to_string((long long)dim);
    // one wave per SIMD where the accumulators and vectors of a wide head need more than 256 registers
    const int waves = dp > 128 ? 1 : 2;
    const double each = 4.0 * (double)q[0] * (double)dim;
    g->algo_bytes = each * (double)(q[1] * q[2] * (forward ? 2 : 4) + k[1] * k[2] * (forward ? 2 : grad_q ? 2 : 4));
    if (forward) {
        // few rows: no tile of keys is read twice, so each wave streams its own
        const bool few = op[3] > 1 || rows <= 64, split = !few && dim <= 128;
        def.set(few ? "AT_FEW_ROWS" : split ? "AT_FORWARD_SPLIT" : "AT_FORWARD", 1);
        // waves that share a tile of keys: eight, if their 256 rows still leave every CU a workgroup
        const int row_waves = q[0] * k[2] * up(rows, 256) >= 256 ? 8 : 4;
        def.set("AT_WAVES", row_waves);
        g->note = few ? "rows x16, keys in " + to_string(op[3]) + " pieces" : split ? "bf16x6 tiles " + to_string(32 * row_waves) + "x32" : string("tiles 64x64");
        return assemble(fk, def, kAttentionSource, (few ? "dsc_attention_few" : "dsc_attention") + size, few ? "attention_few" : split ? "attention_split" : "attention",
                        {input_arg(fk, 0), input_arg(fk, 1), input_arg(fk, 2), start, length, result_arg(fk, 0), result_arg(fk, 1)},
                        q[0] * k[2] * (few ? up(rows, 16) * op[3] : up(rows, split ? 32 * row_waves : 64)), split ? 64 * row_waves : 256, waves, g);
    }
    g->note = "tiles 64x64";
    if (grad_q) {
        def.set("AT_GRAD_QUERY", 1);
        return assemble(fk, def, kAttentionSource, "dsc_attention_grad_query" + size, "attention_grad_query",
                        {input_arg(fk, 0), input_arg(fk, 1), input_arg(fk, 2), input_arg(fk, 3), input_arg(fk, 4), input_arg(fk, 5), start, length,
                         result_arg(fk, 0), result_arg(fk, 1)},
                        q[0] * k[2] * up(rows, 64), 256, dp <= 64 ? 3 : waves, g);
    }
    if (sinks) {
        def.set("AT_GRAD_SINKS", 1);
        return assemble(fk, def, kAttentionSource, "dsc_attention_grad_sinks" + size, "attention_grad_sinks",
                        {input_arg(fk, 0), input_arg(fk, 1), input_arg(fk, 2), input_arg(fk, 3), input_arg(fk, 4), input_arg(fk, 5), start, length,
                         result_arg(fk, 0), result_arg(fk, 1)},
                        q[0] * k[2] * up(std::min<int64_t>(op[1], k[1]), 16) * op[3], 256, waves, g);
    }
    // Key gradient: four waves, two workgroups per CU, for heads of up to 64 (2048 tokens, 4 x 16 heads of 64: 697 us against
    // 769 with eight); eight up to 128, where two of four waves hold 64 KB of tiles each (4096 tokens, 16 over 4 heads of 128,
    // window 1024: 752 against 962); four beyond, one per SIMD.  Tiles of 32 keys while all of them run at once (2 x 512
    // tokens, 8 heads of 64: 33 against 52; 4 heads of 128: 55 against 91), else of 64 (32 x 512 tokens: 201 against 234).
    const int key_waves = dp > 64 && dp <= 128 ? 8 : 4;
    const int keys = q[0] * k[2] * up(k[1], 64) <= (dp <= 64 ? 256 : 128) ? 32 : 64;
    def.set("AT_KEYS", keys);
    def.set("AT_GRAD_KEY_VALUE", 1);
    g->note = "tiles " + to_string(keys) + "x64, " + to_string(key_waves) + " waves";
    def.set("AT_SHARES", 16 * key_waves / keys);
    return assemble(fk, def, kAttentionSource, "dsc_attention_grad_key_value" + size, "attention_grad_key_value",
                    {input_arg(fk, 0), input_arg(fk, 1), input_arg(fk, 2), input_arg(fk, 3), input_arg(fk, 4), input_arg(fk, 5),
                     joins ? input_arg(fk, 6) : "(const float*)nullptr", joins ? input_arg(fk, 7) : "(const float*)nullptr", start, length,
                     result_arg(fk, 0), result_arg(fk, 1)},
                    q[0] * k[2] * up(k[1], keys), 64 * key_waves, waves, g);
}

string gen_dual_matmul(const FusedKernel& fk, Generated* g) {
    const dsc_kernel_desc& d = fk.main.raw();
    Defines def;
    def.set("DM_ACT", d.kind == DSC_KERNEL_GATED_GRAD ? d.op_int[0] : d.op_int[1]);
    if (d.kind == DSC_KERNEL_GATED_GRAD) {
        const int64_t cells = element_count(d.shape);
        const int vec = cells % 4 == 0 ? 4 : 1;
        def.set("DM_MODE", 0);
        def.set64("DM_GRAD_COUNT", cells);
        def.set("DM_GRAD_VEC", vec);
        g->algo_bytes = 4.0 * (double)cells * (3.0 + d.n_outputs);
        g->note = "x" + to_string(vec);
        return assemble(fk, def, kDualMatmulSource, "dsc_gated_grad_n" + to_string((long long)cells), "gated_grad",
                        {input_arg(fk, 0), input_arg(fk, 1), input_arg(fk, 2), result_arg(fk, 0), result_arg(fk, 1)}, up(cells, 256 * vec), 256, 1, g);
    }
    const int mode = d.op_int[0];
    const bool sum = mode == DSC_DUAL_SUM, paired = !sum;
    const int b = sum ? 2 : 1;
    const int64_t m = d.inputs[0].out_shape.dims[0], n = d.inputs[b].out_shape.dims[1], k = d.inputs[0].out_shape.dims[1];
    const int a_of[2] = {0, sum ? 1 : 0}, b_of[2] = {b, b + 1};
    const char* names[4] = {"DM_A0", "DM_A1", "DM_B0", "DM_B1"};
    bool a_kc = true, b_kc = true, a_vec = true, b_vec = true, b_rows = true;
    for (int i = 0; i < 4; ++i) {
        const int in = i < 2 ? a_of[i] : b_of[i - 2];
        const Operand o(d.inputs[in]);
        const int rows = i < 2 ? 0 : 1, along = 1 - rows;  // which axis is rows (columns), which is k
        def.set64(string(names[i]) + "_BASE", o.base);
        def.set64(string(names[i]) + "_R", o.stride[rows]);
        def.set64(string(names[i]) + "_K", o.stride[along]);
        const bool kc = o.stride[along] == 1, quads = o.quads(d.inputs[in], along);
        (i < 2 ? a_kc : b_kc) &= kc;
        (i < 2 ? a_vec : b_vec) &= quads;
        if (i >= 2) b_rows = b_rows && o.quads(d.inputs[in], 1);
    }
    def.set("DM_MODE", mode);
    def.set("DM_M", m);
    def.set("DM_N", n);
    def.set("DM_K", k);
    const string size = "_m" + to_string((long long)m) + "_n" + to_string((long long)n) + "_k" + to_string((long long)k);
    g->algo_flops = 4.0 * (double)m * (double)n * (double)k;
    g->algo_bytes = 4.0 * ((double)m * (double)k * (sum ? 2 : 1) + 2.0 * (double)k * (double)n + (double)m * (double)n * d.n_outputs * d.op_int[2]);
    const std::vector<string> operands = {input_arg(fk, 0), input_arg(fk, sum ? 1 : 0), input_arg(fk, b), input_arg(fk, b + 1)};
    std::vector<string> args = operands;
    for (int i = 0; i < 3; ++i) args.push_back(result_arg(fk, i));
    const string what = sum ? "sum" : mode == DSC_DUAL_GATED ? "gated" : "both";
    const bool columns_beside = Operand(d.inputs[b]).stride[1] == 1 && Operand(d.inputs[b + 1]).stride[1] == 1;
    if (mode == DSC_DUAL_GATED && m <= 8 && columns_beside) {
        def.set("DM_FEW_ROWS", 1);
        def.set("DM_FEW_VEC", b_rows && n % 4 == 0 ? 1 : 0);
        args.erase(args.begin() + 1);
        g->note = "columns x32, k in 128 slices";
        return assemble(fk, def, kDualMatmulSource, "dsc_dual_matmul_few" + size, "gated_few_rows", args, up(n, 32), 1024, 4, g);
    }
    // Tile.  A CU's step of 16 k costs 2.4 us with 256x256 (8 waves of 128x64), 0.73 with 128x128 (8 waves of 32x64; with 4
    // waves of 64x64 0.83) and, alone on its CU, 0.55 with 64x64: the largest tile that leaves no CU without one, and
    // the smallest where even that many do not fill the CUs (1001 x 1366 columns x 512 k of both products: 32 us with
    // 128x128, 37 with 64x64; 1001 x 500, k 2 x 1366, not split: 113 and 98).  Up to 64 rows there are too few tiles for the
    // CUs and a step's latency counts: four groups of waves share k (16 x 4096 into 8000: 162 us with one group, 120 with
    // two, 84 to 89 with four; 64 x 2048 into 1366: 83, 62, 47, and 66 with tiles of 64x64).
    struct Tile {
        int bm, bn, wm, wn, ahead, groups;
    };
    const int64_t splits = d.op_int[2];
    auto count = [&](int bm, int bn) { return up(m, bm) * up(n, paired ? bn / 2 : bn) * splits; };
    Tile t = {128, 128, 4, 2, 2, 1};
    if (m <= 64) t = {32, 128, 1, 2, 4, 4};
    else if (count(256, 256) >= 256) t = {256, 256, 2, 4, 2, 1};
    else if (count(64, 64) <= 256) t = {64, 64, 2, 1, 4, 1};
    const int64_t tiles_m = up(m, t.bm), tiles_n = up(n, paired ? t.bn / 2 : t.bn);
    if (tiles_m * tiles_n * splits >= (int64_t(1) << 30)) return "kernel too large: more than 2^30 tiles";
    def.set("DM_BM", t.bm);
    def.set("DM_BN", t.bn);
    def.set("DM_WM", t.wm);
    def.set("DM_WN", t.wn);
    def.set("DM_AHEAD", t.ahead);
    def.set("DM_SPLITS", splits);
    def.set("DM_KGROUPS", t.groups);
    def.set("DM_A_KC", a_kc ? 1 : 0);
    def.set("DM_B_KC", b_kc ? 1 : 0);
    def.set("DM_A_VEC", a_vec && k % 4 == 0 ? 1 : 0);  // (quads that are moved back to end with k keep their alignment)
    def.set("DM_B_VEC", b_vec && k % 4 == 0 ? 1 : 0);
    def.set("DM_TILES_M", tiles_m);
    def.set("DM_TILES_N", tiles_n);
    def.set("DM_GROUP", 8);
    g->note = "bf16x6 32x32x16 tile " + to_string(t.bm) + "x" + to_string(t.bn) + "x16 waves " + to_string(t.wm) + "x" + to_string(t.wn) + " A" +
              (a_kc ? a_vec ? "k4" : "k1" : "r") + " B" + (b_kc ? b_vec ? "k4" : "k1" : "r");
    return assemble(fk, def, kDualMatmulSource, "dsc_dual_matmul_" + what + size, "dual_matmul", args, up(tiles_m * tiles_n * splits, 8) * 8, 64 * t.wm * t.wn * t.groups, 2, g);
}

}  // namespace

string generate_operator(const FusedKernel& fk, Generated* out) {
    switch (fk.main.raw().kind) {
    case DSC_KERNEL_RMS_NORM:
    case DSC_KERNEL_RMS_NORM_GRAD: return gen_rms_norm(fk, out);
    case DSC_KERNEL_ROTARY: return gen_rotary(fk, out);
    case DSC_KERNEL_CACHE_APPEND: return gen_cache_append(fk, out);
    case DSC_KERNEL_DUAL_MATMUL:
    case DSC_KERNEL_GATED_GRAD: return gen_dual_matmul(fk, out);
    default: return gen_attention(fk, out);
    }
}

}  // namespace dsc
