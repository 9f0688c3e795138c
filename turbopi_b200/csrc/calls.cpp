// The calls whose kernels take a few microseconds, from tensors to launch in C++: output allocation, argument struct and the
// C ABI's entry point in one step.  The Python forms of the same calls (turbopi_b200/ops.py and the modules) stay the
// reference for what is accepted: whatever a function here does not recognise as its plain case (a CPU tensor, another
// device, a dtype or a stride that needs a conversion) returns None and takes the Python form, which converts or refuses.
// A non-zero status of the C ABI comes back as an int.  Time to issue a call (us, Python form -> here): one-token INT4 linear
// 13.1 -> 7.1, 50-token MLP 31.2 -> 17.4, attention 18.2 -> 8.2, W4A4 linear 21.7 -> 12.4, FP8 quantiser + W4A8 launcher 24.4 -> 18.1,
// attention on packed prompts or a paged cache, appends, page copies 20-50 -> 4-8.
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/extension.h>

#include <optional>

#include "turbopi_b200.h"

namespace {

struct Entries {
    decltype(&tpb200_w4_gemm) w4_gemm;
    decltype(&tpb200_w4a16_gemv) w4a16_gemv;
    decltype(&tpb200_w4a16_gemm) w4a16_gemm;
    decltype(&tpb200_attention) attention;
    decltype(&quantizeActivationToFP8) quantize_fp8;
    decltype(&tpb200_last_error) last_error;
    decltype(&tpb200_nvfp4_tiled_a_bytes) tiled_a_bytes;
    decltype(&tpb200_nvfp4_quantize_act_tiled) quantize_act_tiled;
    decltype(&tpb200_nvfp4_gemm_ex) gemm_ex;
    decltype(&tpb200_packed_attention) packed_attention;
    decltype(&tpb200_paged_attention_workspace_size) paged_workspace;
    decltype(&tpb200_paged_attention) paged_attention;
    decltype(&tpb200_paged_append) paged_append;
    decltype(&tpb200_copy_pages) copy_pages;
    decltype(&tpb200_packed_attention_window) packed_attention_window;
    decltype(&tpb200_paged_attention_window) paged_attention_window;
    decltype(&tpb200_paged_attention_nvfp4_workspace_size) paged_nvfp4_workspace;
    decltype(&tpb200_paged_attention_nvfp4) paged_attention_nvfp4;
    decltype(&tpb200_paged_append_nvfp4) paged_append_nvfp4;
    decltype(&tpb200_paged_read) paged_read;
    decltype(&tpb200_paged_read_nvfp4) paged_read_nvfp4;
} g;

using OptTensor = std::optional<at::Tensor>;

// the entry points of the library that turbopi_b200/_lib.py has loaded, in the order of Entries
void bind(const std::vector<uint64_t>& a) {
    TORCH_CHECK(a.size() * sizeof(void*) == sizeof(Entries), "calls.bind: wrong number of entry points");
    memcpy(&g, a.data(), sizeof(Entries));
}

int code_of(at::ScalarType t) {
    return t == at::kBFloat16 ? TPB200_BF16 : t == at::kHalf ? TPB200_F16 : t == at::kFloat ? TPB200_F32 : -1;
}
at::ScalarType type_of(int code) { return code == TPB200_BF16 ? at::kBFloat16 : code == TPB200_F16 ? at::kHalf : at::kFloat; }

void* ptr(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }
bool on(const at::Tensor& t, int dev) { return t.is_cuda() && t.get_device() == dev; }
bool on(const OptTensor& t, int dev) { return !t.has_value() || on(*t, dev); }

// the device of `t` if it is the current one, else -1
int here(const at::Tensor& t) {
    if (!t.is_cuda()) return -1;
    const int d = t.get_device();
    return d == c10::cuda::current_device() ? d : -1;
}
tpb200_stream_t stream_of(int dev) { return reinterpret_cast<tpb200_stream_t>(c10::cuda::getCurrentCUDAStream(dev).stream()); }

template <class F>
int launch(F&& f) {                                       // without the interpreter lock, as through ctypes
    py::gil_scoped_release nogil;
    return f();
}

py::object done(int status, const at::Tensor& out) { return status == 0 ? py::cast(out) : py::int_(status); }

int w4(const at::Tensor& x, int64_t M, int64_t K, const at::Tensor& w, int64_t N, int format, const OptTensor& w_scales,
       const OptTensor& w_zeros, double alpha, double beta, const OptTensor& bias, int activation, bool gated, const at::Tensor& out,
       int flags, int dev) {
    tpb200_w4_gemm_args a = {};
    a.x = x.data_ptr();
    a.ldx = static_cast<int>(M > 1 ? x.stride(0) : K);
    a.format = format;
    a.w = w.data_ptr();
    a.w_pitch = format == TPB200_W4_NVFP4_ROWMAJOR ? static_cast<int>(w.stride(0)) : 0;
    a.w_scales = ptr(w_scales);
    a.w_zeros = ptr(w_zeros);
    a.alpha = static_cast<float>(alpha);
    a.beta = static_cast<float>(beta);
    a.bias = ptr(bias);
    a.bias_dtype = bias.has_value() ? code_of(bias->scalar_type()) : TPB200_F32;
    a.activation = activation;
    a.gated = gated;
    a.out = out.data_ptr();
    a.out_dtype = code_of(out.scalar_type());
    a.ldo = static_cast<int>(M > 1 ? out.stride(0) : out.size(1));
    a.M = static_cast<int>(M);
    a.N = static_cast<int>(N);
    a.K = static_cast<int>(K);
    a.flags = flags;
    const tpb200_stream_t s = stream_of(dev);
    return launch([&] { return g.w4_gemm(&a, s); });
}

// ops.w4_gemm
py::object w4_gemm(const at::Tensor& x, const at::Tensor& w, int64_t N, int format, const OptTensor& w_scales, const OptTensor& w_zeros,
                   double alpha, double beta, const OptTensor& bias, int activation, bool gated, const OptTensor& out, int out_code,
                   int flags) {
    const int dev = here(x);
    if (dev < 0 || x.dim() != 2 || x.scalar_type() != at::kBFloat16 || x.stride(1) != 1 || !on(w, dev) || !on(w_scales, dev) ||
        !on(w_zeros, dev) || !on(bias, dev) || !on(out, dev) || (bias.has_value() && code_of(bias->scalar_type()) < 0) ||
        (out.has_value() ? out->dim() != 2 || code_of(out->scalar_type()) < 0 : out_code < 0)) {
        return py::none();
    }
    const int64_t M = x.size(0), K = x.size(1);
    const at::Tensor y = out.has_value() ? *out : at::empty({M, gated ? N / 2 : N}, x.options().dtype(type_of(out_code)));
    return done(w4(x, M, K, w, N, format, w_scales, w_zeros, alpha, beta, bias, activation, gated, y, flags, dev), y);
}

// NVFP4PackedMLP's two launches on tiled images: gate_up with act(gate) * up in its epilogue, down on its bf16 result
py::object mlp(const at::Tensor& x, const at::Tensor& gate_up, const at::Tensor& down, const OptTensor& bias, int64_t I, int64_t H,
               double alpha_gu, double alpha_d, int activation, int flags_first, int flags_second) {
    const int dev = here(x);
    if (dev < 0 || x.dim() != 2 || x.scalar_type() != at::kBFloat16 || !x.is_contiguous() || x.size(1) != H || !on(gate_up, dev) ||
        !on(down, dev) || !on(bias, dev)) {
        return py::none();
    }
    const int64_t M = x.size(0);
    const at::Tensor h = at::empty({M, I}, x.options()), y = at::empty({M, H}, x.options());
    const int st = w4(x, M, H, gate_up, 2 * I, TPB200_W4_NVFP4_TILED, {}, {}, alpha_gu, 0.0, {}, activation, true, h, flags_first, dev);
    if (st != 0) return py::int_(st);
    return done(w4(h, M, I, down, H, TPB200_W4_NVFP4_TILED, {}, {}, alpha_d, 0.0, bias, TPB200_ACT_NONE, false, y, flags_second, dev), y);
}

// W4A16Linear.forward on its buffers
py::object w4a16_linear(const at::Tensor& input, const at::Tensor& packed, const at::Tensor& scales, const OptTensor& bias, int64_t N,
                        int flags) {
    const int dev = here(input);
    const int code = code_of(input.scalar_type());
    if (dev < 0 || code < 0 || input.dim() < 1 || !input.is_contiguous() || !on(packed, dev) || !on(scales, dev) || !on(bias, dev) ||
        packed.dim() != 3 || packed.size(0) == 0 || input.size(-1) != packed.size(0) * 32 ||
        (bias.has_value() && (code_of(bias->scalar_type()) < 0 || !bias->is_contiguous())) || scales.scalar_type() != at::kHalf) {
        return py::none();
    }
    const int64_t K = input.size(-1), T = input.numel() / K;
    if (T < 1 || (T > 16 && (K % 128 != 0 || N % 8 != 0))) return py::none();
    std::vector<int64_t> shape(input.sizes().begin(), input.sizes().end());
    shape.back() = N;
    const at::Tensor y = at::empty(shape, input.options());
    const at::Tensor x = T <= 16 || code == TPB200_BF16 ? input : input.to(at::kBFloat16);
    const void *xp = x.data_ptr(), *wp = packed.data_ptr(), *sp = scales.data_ptr(), *bp = ptr(bias);
    void* yp = y.data_ptr();
    const int bias_code = bias.has_value() ? code_of(bias->scalar_type()) : TPB200_F32;
    const tpb200_stream_t s = stream_of(dev);
    const int m = static_cast<int>(T), n = static_cast<int>(N), k = static_cast<int>(K);
    const int st = launch([&] {
        return T <= 16 ? g.w4a16_gemv(xp, code, wp, sp, TPB200_SCALE_F16, bp, bias_code, yp, code, m, n, k, 32, TPB200_INT4_KBLOCK, 0, s)
                       : g.w4a16_gemm(xp, wp, sp, nullptr, bp, bias_code, yp, code, m, n, k, n, TPB200_INT4_KBLOCK, 1.0f, 0.0f, flags, s);
    });
    return done(st, y);
}

// ops.attention without a fused quantiser
py::object attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& out, double scale,
                     const OptTensor& key_bias, const at::Tensor& workspace, int flags) {
    const int dev = here(q);
    const int64_t nd = q.dim();
    if (dev < 0 || (nd != 2 && nd != 4) || !on(workspace, dev) || !on(key_bias, dev)) return py::none();
    for (const at::Tensor* t : {&q, &k, &v, &out}) {
        if (!on(*t, dev) || t->dim() != nd || t->scalar_type() != at::kBFloat16 || t->stride(-1) != 1) return py::none();
    }
    const int64_t A = nd == 4 ? q.size(0) : 1, B = nd == 4 ? q.size(1) : 1, R = q.size(-2), D = q.size(-1), S = k.size(-2);
    if (out.sizes() != q.sizes() || v.sizes() != k.sizes() || k.size(-1) != D || (nd == 4 && (k.size(0) != A || k.size(1) != B)) ||
        (key_bias.has_value() &&
         (key_bias->scalar_type() != at::kBFloat16 || key_bias->numel() < S || !key_bias->is_contiguous()))) {
        return py::none();
    }
    tpb200_attention_args a = {};
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.out = out.data_ptr();
    a.key_bias = ptr(key_bias);
    a.n_rows = static_cast<int>(R);
    a.n_keys = static_cast<int>(S);
    a.head_dim = static_cast<int>(D);
    a.ldq = static_cast<int>(q.stride(-2));
    a.ldk = static_cast<int>(k.stride(-2));
    a.ldv = static_cast<int>(v.stride(-2));
    a.ldo = static_cast<int>(out.stride(-2));
    a.groups_outer = static_cast<int>(A);
    a.groups_inner = static_cast<int>(B);
    if (nd == 4) {
        for (int i = 0; i < 2; ++i) {
            a.q_stride[i] = q.stride(i);
            a.k_stride[i] = k.stride(i);
            a.v_stride[i] = v.stride(i);
            a.o_stride[i] = out.stride(i);
        }
    }
    a.scale = static_cast<float>(scale);
    a.workspace = workspace.data_ptr();
    a.workspace_bytes = static_cast<size_t>(workspace.numel());
    a.flags = flags;
    a.quant_rows_per_token = 1;
    const tpb200_stream_t s = stream_of(dev);
    const int st = launch([&] { return g.attention(&a, s); });
    if (st != 0) return py::int_(st);
    return py::cast(nd == 4 ? out : out.unsqueeze(0).unsqueeze(0));
}

// ops.quantize_activation_to_fp8
py::object quantize_fp8(const at::Tensor& x) {
    const int dev = here(x);
    if (dev < 0 || x.dim() != 2 || x.scalar_type() != at::kBFloat16 || !x.is_contiguous()) return py::none();
    const int64_t M = x.size(0), K = x.size(1);
    const auto bytes = x.options().dtype(at::kByte);
    const at::Tensor out = at::empty({M, K}, bytes), scales = at::empty({M, K / 16}, bytes);
    const void* xp = x.data_ptr();
    void *op = out.data_ptr(), *sp = scales.data_ptr();
    const tpb200_stream_t s = stream_of(dev);
    const int st = launch([&] {
        g.quantize_fp8(xp, op, sp, static_cast<int>(M), static_cast<int>(K), s);
        return g.last_error();
    });
    return st == 0 ? py::object(py::make_tuple(out, scales)) : py::int_(st);
}

// ops.nvfp4_linear_tiled on row-major weights
py::object nvfp4_linear(const at::Tensor& x, const at::Tensor& w, int64_t N, double alpha, const OptTensor& bias, int activation,
                        int out_code, const at::Tensor& w_sf) {
    const int dev = here(x);
    const int code = code_of(x.scalar_type());
    if (dev < 0 || code < 0 || out_code < 0 || x.dim() != 2 || !x.is_contiguous() || !on(w, dev) || !on(w_sf, dev) || !on(bias, dev) || w.dim() != 2 ||
        (bias.has_value() && (bias->scalar_type() != at::kFloat || !bias->is_contiguous()))) {
        return py::none();
    }
    const int M = static_cast<int>(x.size(0)), K = static_cast<int>(x.size(1));
    const at::Tensor a = at::empty({static_cast<int64_t>(g.tiled_a_bytes(M, K, 1))}, x.options().dtype(at::kByte));
    const at::Tensor y = at::empty({M, N}, x.options().dtype(type_of(out_code)));
    tpb200_nvfp4_gemm_args p = {};
    p.a_packed = a.data_ptr();
    p.a_pieces = 1;
    p.b_packed = w.data_ptr();
    p.b_pitch = static_cast<int>(w.stride(0));
    p.b_sf = w_sf.data_ptr();
    p.alpha = static_cast<float>(alpha);
    p.bias = static_cast<decltype(p.bias)>(ptr(bias));
    p.activation = activation;
    p.out = y.data_ptr();
    p.out_dtype = out_code;
    p.ldo = static_cast<int>(N);
    p.M = M;
    p.N = static_cast<int>(N);
    p.K = K;
    p.layout = TPB200_OPERANDS_TILED_A;
    // the quantiser is a plain launch, so what wrote the weights is complete when it starts: their blocks travel while it runs
    p.flags = TPB200_FLAG_PDL;
    const void* xp = x.data_ptr();
    void* ap = a.data_ptr();
    const tpb200_stream_t s = stream_of(dev);
    const int st = launch([&] {
        const int q = g.quantize_act_tiled(xp, code, K, ap, M, K, s);
        return q != 0 ? q : g.gemm_ex(&p, s);
    });
    return done(st, y);
}

// ------------------------------------------------------------------------------------------------ a cache of pages
// sizes that the 32 bits of the C structures hold; others are refused by the Python forms
bool fits(at::IntArrayRef sizes) {
    for (const int64_t n : sizes) {
        if (n > 0x7fffffff) return false;
    }
    return true;
}

bool half(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

// [tokens, heads, D] of one type and device with a contiguous last dimension
bool rows(const at::Tensor& t, int dev, int64_t tokens, int64_t heads, int64_t D, at::ScalarType type) {
    return on(t, dev) && t.dim() == 3 && t.size(0) == tokens && t.size(1) == heads && t.size(2) == D && fits(t.sizes()) && t.scalar_type() == type && t.stride(2) == 1;
}
bool offsets(const at::Tensor& t, int dev, int64_t n) {
    return on(t, dev) && t.dim() == 1 && t.numel() == n && t.scalar_type() == at::kInt && t.is_contiguous();
}
void strides(const at::Tensor& t, long long (&to)[2]) {
    to[0] = t.stride(0);
    to[1] = t.stride(1);
}

bool paged(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lengths, int dev, tpb200_paged_cache& c) {
    if (!on(k, dev) || !on(v, dev) || !on(table, dev) || !on(lengths, dev) || k.dim() != 4 || !half(k) || v.scalar_type() != k.scalar_type() ||
        v.sizes() != k.sizes() || v.strides() != k.strides() || k.stride(3) != 1 || table.dim() != 2 || table.scalar_type() != at::kInt ||
        lengths.dim() != 1 || lengths.scalar_type() != at::kInt || lengths.numel() != table.size(0) || !lengths.is_contiguous() ||
        (table.size(1) > 1 && table.stride(1) != 1) || !fits(k.sizes()) || !fits(table.sizes())) {
        return false;
    }
    c.k_pages = k.data_ptr();
    c.v_pages = v.data_ptr();
    c.page_stride = k.stride(0);
    c.row_stride = k.stride(1);
    c.head_stride = k.stride(2);
    c.num_pages = static_cast<int>(k.size(0));
    c.page_size = static_cast<int>(k.size(1));
    c.kv_heads = static_cast<int>(k.size(2));
    c.head_dim = static_cast<int>(k.size(3));
    c.dtype = code_of(k.scalar_type());
    c.table = static_cast<const int*>(table.data_ptr());
    c.table_stride = table.stride(0);
    c.table_width = static_cast<int>(table.size(1));
    c.lengths = static_cast<const int*>(lengths.data_ptr());
    c.seqs = static_cast<int>(table.size(0));
    return true;
}

// ops.paged_attention; window 0: all keys
py::object paged_attention_window(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lengths,
                                  double scale, const OptTensor& out, const OptTensor& workspace, int window, int sinks, int flags) {
    const int dev = here(q);
    tpb200_paged_attention_args a = {};
    if (dev < 0 || !paged(k, v, table, lengths, dev, a.cache) || q.dim() != 3 || a.cache.seqs < 1 || a.cache.kv_heads < 1) return py::none();
    const int64_t H = q.size(1);
    if (!rows(q, dev, a.cache.seqs, H, a.cache.head_dim, k.scalar_type()) || !on(workspace, dev) || H < 1 || H % a.cache.kv_heads != 0 ||
        (workspace.has_value() && !workspace->is_contiguous()) ||
        (out.has_value() && !rows(*out, dev, a.cache.seqs, H, a.cache.head_dim, k.scalar_type()))) {
        return py::none();
    }
    at::Tensor ws;
    if (workspace.has_value()) ws = *workspace;
    else {
        const size_t n = g.paged_workspace(static_cast<int>(H), a.cache.kv_heads, a.cache.head_dim);
        if (n == 0) return py::none();
        ws = at::empty({static_cast<int64_t>(n)}, q.options().dtype(at::kByte));
    }
    const at::Tensor y = out.has_value() ? *out : at::empty(q.sizes(), q.options());
    a.q = q.data_ptr();
    a.out = y.data_ptr();
    strides(q, a.q_stride);
    strides(y, a.o_stride);
    a.q_heads = static_cast<int>(H);
    a.scale = static_cast<float>(scale);
    a.workspace = ws.data_ptr();
    a.workspace_bytes = ws.nbytes();
    a.flags = flags;
    const tpb200_stream_t s = stream_of(dev);
    return done(launch([&] { return window > 0 ? g.paged_attention_window(&a, window, sinks, s) : g.paged_attention(&a, s); }), y);
}
py::object paged_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lengths,
                           double scale, const OptTensor& out, const OptTensor& workspace, int flags) {
    return paged_attention_window(q, k, v, table, lengths, scale, out, workspace, 0, 0, flags);
}

// one layer of a cache of 4-bit pages
bool paged_nvfp4(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lengths, int64_t head_dim, double k_scale,
                 double v_scale, int dev, tpb200_paged_nvfp4_cache& c) {
    if (!on(k, dev) || !on(v, dev) || !on(table, dev) || !on(lengths, dev) || k.dim() != 4 || k.scalar_type() != at::kByte ||
        v.scalar_type() != at::kByte || v.sizes() != k.sizes() || v.strides() != k.strides() || k.stride(3) != 1 || head_dim < 8 || head_dim > 256 ||
        k.size(3) != 288 * ((head_dim + 31) / 32) || table.dim() != 2 || table.scalar_type() != at::kInt || lengths.dim() != 1 ||
        lengths.scalar_type() != at::kInt || lengths.numel() != table.size(0) || !lengths.is_contiguous() ||
        (table.size(1) > 1 && table.stride(1) != 1) || !fits({k.size(0), k.size(1), 16 * k.size(2)}) || !fits(table.sizes())) {
        return false;
    }
    c.k_pages = k.data_ptr();
    c.v_pages = v.data_ptr();
    c.page_stride = k.stride(0);
    c.head_stride = k.stride(1);
    c.tile_stride = k.stride(2);
    c.num_pages = static_cast<int>(k.size(0));
    c.page_size = static_cast<int>(16 * k.size(2));
    c.kv_heads = static_cast<int>(k.size(1));
    c.head_dim = static_cast<int>(head_dim);
    c.k_scale = static_cast<float>(k_scale);
    c.v_scale = static_cast<float>(v_scale);
    c.table = static_cast<const int*>(table.data_ptr());
    c.table_stride = table.stride(0);
    c.table_width = static_cast<int>(table.size(1));
    c.lengths = static_cast<const int*>(lengths.data_ptr());
    c.seqs = static_cast<int>(table.size(0));
    return true;
}

// ops.paged_attention_nvfp4
py::object paged_attention_nvfp4(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lengths,
                                 double scale, const OptTensor& out, const OptTensor& workspace, int window, int sinks, double k_scale,
                                 double v_scale, int flags) {
    const int dev = here(q);
    tpb200_paged_attention_nvfp4_args a = {};
    if (dev < 0 || q.dim() != 3 || !half(q) || !paged_nvfp4(k, v, table, lengths, q.size(2), k_scale, v_scale, dev, a.cache) || a.cache.seqs < 1 ||
        a.cache.kv_heads < 1) {
        return py::none();
    }
    const int64_t H = q.size(1), D = q.size(2);
    if (!rows(q, dev, a.cache.seqs, H, D, q.scalar_type()) || !on(workspace, dev) || H < 1 || H % a.cache.kv_heads != 0 ||
        (workspace.has_value() && !workspace->is_contiguous()) || (out.has_value() && !rows(*out, dev, a.cache.seqs, H, D, q.scalar_type()))) {
        return py::none();
    }
    at::Tensor ws;
    if (workspace.has_value()) ws = *workspace;
    else {
        const size_t n = g.paged_nvfp4_workspace(static_cast<int>(H), a.cache.kv_heads, a.cache.head_dim);
        if (n == 0) return py::none();
        ws = at::empty({static_cast<int64_t>(n)}, q.options().dtype(at::kByte));
    }
    const at::Tensor y = out.has_value() ? *out : at::empty(q.sizes(), q.options());
    a.q = q.data_ptr();
    a.out = y.data_ptr();
    a.dtype = code_of(q.scalar_type());
    strides(q, a.q_stride);
    strides(y, a.o_stride);
    a.q_heads = static_cast<int>(H);
    a.scale = static_cast<float>(scale);
    a.window = window;
    a.sinks = sinks;
    a.workspace = ws.data_ptr();
    a.workspace_bytes = ws.nbytes();
    a.flags = flags;
    const tpb200_stream_t s = stream_of(dev);
    return done(launch([&] { return g.paged_attention_nvfp4(&a, s); }), y);
}

// (k, v) as the rows that a read gives; false where they are not the plain case
bool read_rows(const at::Tensor& pages, int64_t heads, int64_t D, at::ScalarType type, const at::Tensor& cu, int64_t seqs, int64_t tokens,
               const OptTensor& k, const OptTensor& v, int dev, at::Tensor (&y)[2], tpb200_paged_rows& a) {
    if (!offsets(cu, dev, seqs + 1) || tokens < 0 || !fits({tokens}) || k.has_value() != v.has_value() ||
        (k.has_value() && (!rows(*k, dev, tokens, heads, D, type) || !rows(*v, dev, tokens, heads, D, type)))) {
        return false;
    }
    if (k.has_value()) {
        y[0] = *k;
        y[1] = *v;
    } else {                                              // one allocation for both
        const at::Tensor both = at::empty({2, tokens, heads, D}, pages.options().dtype(type));
        y[0] = both.select(0, 0);
        y[1] = both.select(0, 1);
    }
    a.k = y[0].data_ptr();
    a.v = y[1].data_ptr();
    a.dtype = code_of(type);
    strides(y[0], a.k_stride);
    strides(y[1], a.v_stride);
    a.cu = static_cast<const int*>(cu.data_ptr());
    a.tokens = static_cast<int>(tokens);
    return true;
}
py::object pair_of(int status, const at::Tensor (&y)[2]) { return status == 0 ? py::object(py::make_tuple(y[0], y[1])) : py::int_(status); }

// ops.paged_read
py::object paged_read(const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table, const at::Tensor& cu, const at::Tensor& lengths,
                      const py::object& tokens, const OptTensor& k, const OptTensor& v, int flags) {
    const int dev = here(k_pages);
    tpb200_paged_cache c = {};
    tpb200_paged_rows a = {};
    at::Tensor y[2];
    if (dev < 0 || !PyLong_CheckExact(tokens.ptr()) || !paged(k_pages, v_pages, table, lengths, dev, c)) return py::none();
    int overflow = 0;
    const int64_t n = PyLong_AsLongAndOverflow(tokens.ptr(), &overflow);
    if (overflow != 0 || !read_rows(k_pages, c.kv_heads, c.head_dim, k_pages.scalar_type(), cu, c.seqs, n, k, v, dev, y, a)) return py::none();
    a.flags = flags;
    const tpb200_stream_t s = stream_of(dev);
    return pair_of(launch([&] { return g.paged_read(&c, &a, s); }), y);
}

// ops.paged_read_nvfp4
py::object paged_read_nvfp4(const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table, const at::Tensor& cu, const at::Tensor& lengths,
                            const py::object& head_dim, const py::object& tokens, const py::object& dtype, const OptTensor& k, const OptTensor& v,
                            double k_scale, double v_scale, int flags) {
    const int dev = here(k_pages);
    tpb200_paged_nvfp4_cache c = {};
    tpb200_paged_rows a = {};
    at::Tensor y[2];
    if (dev < 0 || !PyLong_CheckExact(tokens.ptr()) || !PyLong_CheckExact(head_dim.ptr()) || !THPDtype_Check(dtype.ptr())) return py::none();
    const auto type = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
    int overflow = 0, too_wide = 0;
    const int64_t n = PyLong_AsLongAndOverflow(tokens.ptr(), &overflow), D = PyLong_AsLongAndOverflow(head_dim.ptr(), &too_wide);
    if (overflow != 0 || too_wide != 0 || (type != at::kBFloat16 && type != at::kHalf) ||
        !paged_nvfp4(k_pages, v_pages, table, lengths, D, k_scale, v_scale, dev, c) ||
        !read_rows(k_pages, c.kv_heads, D, type, cu, c.seqs, n, k, v, dev, y, a)) {
        return py::none();
    }
    a.flags = flags;
    const tpb200_stream_t s = stream_of(dev);
    return pair_of(launch([&] { return g.paged_read_nvfp4(&c, &a, s); }), y);
}

// the rows, offsets and tables of an append; false where they are not the plain case
template <class Args>
bool append_rows(const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu, const OptTensor& q, const OptTensor& cos, const OptTensor& sin,
                 const OptTensor& q_out, at::ScalarType type, int heads, int64_t D, int seqs, int dev, at::Tensor& y, Args& a) {
    const int64_t T = k.size(0);
    if (!rows(k, dev, T, heads, D, type) || !rows(v, dev, T, heads, D, type) || !offsets(cu, dev, seqs + 1ll) ||
        cos.has_value() != sin.has_value() || (q.has_value() && !cos.has_value()) || (!q.has_value() && q_out.has_value())) {
        return false;
    }
    if (cos.has_value()) {
        if (!on(*cos, dev) || !on(*sin, dev) || cos->dim() != 2 || cos->sizes() != sin->sizes() || cos->size(1) != D / 2 ||
            cos->scalar_type() != sin->scalar_type() || code_of(cos->scalar_type()) < 0 || !cos->is_contiguous() || !sin->is_contiguous() || !fits(cos->sizes())) {
            return false;
        }
        a.cos = cos->data_ptr();
        a.sin = sin->data_ptr();
        a.rope_dtype = code_of(cos->scalar_type());
        a.rope_positions = static_cast<int>(cos->size(0));
    }
    if (q.has_value()) {
        if (q->dim() != 3 || !rows(*q, dev, T, q->size(1), D, type) || (q_out.has_value() && !rows(*q_out, dev, T, q->size(1), D, type))) {
            return false;
        }
        y = q_out.has_value() ? *q_out : at::empty(q->sizes(), q->options());
        a.q = q->data_ptr();
        a.q_out = y.data_ptr();
        a.q_heads = static_cast<int>(q->size(1));
        strides(*q, a.q_stride);
        strides(y, a.o_stride);
    }
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    strides(k, a.k_stride);
    strides(v, a.v_stride);
    a.cu = static_cast<const int*>(cu.data_ptr());
    a.tokens = static_cast<int>(T);
    return true;
}

// ops.paged_append; True where there are no queries to give back
py::object paged_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
                        const at::Tensor& cu, const at::Tensor& lengths, const OptTensor& q, const OptTensor& cos, const OptTensor& sin,
                        const OptTensor& q_out, int flags) {
    const int dev = here(k);
    tpb200_paged_append_args a = {};
    if (dev < 0 || !paged(k_pages, v_pages, table, lengths, dev, a.cache) || k.dim() != 3) return py::none();
    at::Tensor y;
    if (!append_rows(k, v, cu, q, cos, sin, q_out, k_pages.scalar_type(), a.cache.kv_heads, a.cache.head_dim, a.cache.seqs, dev, y, a)) return py::none();
    a.flags = flags;
    const tpb200_stream_t s = stream_of(dev);
    const int st = launch([&] { return g.paged_append(&a, s); });
    if (st != 0) return py::int_(st);
    return q.has_value() ? py::cast(y) : py::object(py::bool_(true));
}

// ops.paged_append_nvfp4; True where there are no queries to give back
py::object paged_append_nvfp4(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
                              const at::Tensor& cu, const at::Tensor& lengths, const OptTensor& q, const OptTensor& cos, const OptTensor& sin,
                              const OptTensor& q_out, double k_scale, double v_scale, int flags) {
    const int dev = here(k);
    tpb200_paged_append_nvfp4_args a = {};
    if (dev < 0 || k.dim() != 3 || !half(k) || !paged_nvfp4(k_pages, v_pages, table, lengths, k.size(2), k_scale, v_scale, dev, a.cache)) {
        return py::none();
    }
    at::Tensor y;
    if (!append_rows(k, v, cu, q, cos, sin, q_out, k.scalar_type(), a.cache.kv_heads, a.cache.head_dim, a.cache.seqs, dev, y, a)) return py::none();
    a.dtype = code_of(k.scalar_type());
    a.flags = flags;
    const tpb200_stream_t s = stream_of(dev);
    const int st = launch([&] { return g.paged_append_nvfp4(&a, s); });
    if (st != 0) return py::int_(st);
    return q.has_value() ? py::cast(y) : py::object(py::bool_(true));
}

// ops.packed_attention; window 0: all keys
py::object packed(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu, double scale,
                  const OptTensor& out, bool causal, const OptTensor& cu_keys, int window, int sinks, int flags) {
    const int dev = here(q);
    if (dev < 0 || q.dim() != 3 || k.dim() != 3 || !half(q)) return py::none();
    const int64_t T = q.size(0), H = q.size(1), D = q.size(2), Tk = k.size(0), Hk = k.size(1);
    const auto type = q.scalar_type();
    if (!rows(q, dev, T, H, D, type) || !rows(k, dev, Tk, Hk, D, type) || !rows(v, dev, Tk, Hk, D, type) || cu.numel() < 1 ||
        !offsets(cu, dev, cu.numel()) || !fits(cu.sizes()) || (cu_keys.has_value() ? !offsets(*cu_keys, dev, cu.numel()) : Tk != T) ||
        (out.has_value() && !rows(*out, dev, T, H, D, type))) {
        return py::none();
    }
    const at::Tensor y = out.has_value() ? *out : at::empty({T, H, D}, q.options());
    tpb200_packed_attention_args a = {};
    a.q = q.data_ptr();
    a.k = k.data_ptr();
    a.v = v.data_ptr();
    a.out = y.data_ptr();
    strides(q, a.q_stride);
    strides(k, a.k_stride);
    strides(v, a.v_stride);
    strides(y, a.o_stride);
    a.cu = static_cast<const int*>(cu.data_ptr());
    a.cu_keys = static_cast<const int*>(ptr(cu_keys));
    a.seqs = static_cast<int>(cu.numel() - 1);
    a.q_tokens = static_cast<int>(T);
    a.k_tokens = static_cast<int>(Tk);
    a.q_heads = static_cast<int>(H);
    a.kv_heads = static_cast<int>(Hk);
    a.head_dim = static_cast<int>(D);
    a.dtype = code_of(type);
    a.scale = static_cast<float>(scale);
    a.causal = causal;
    a.flags = flags;
    const tpb200_stream_t s = stream_of(dev);
    return done(launch([&] { return window > 0 ? g.packed_attention_window(&a, window, sinks, s) : g.packed_attention(&a, s); }), y);
}
py::object packed_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu, double scale,
                            const OptTensor& out, bool causal, const OptTensor& cu_keys, int flags) {
    return packed(q, k, v, cu, scale, out, causal, cu_keys, 0, 0, flags);
}
py::object packed_attention_window(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cu, double scale,
                                   const OptTensor& out, const OptTensor& cu_keys, int window, int sinks, int flags) {
    return packed(q, k, v, cu, scale, out, true, cu_keys, window, sinks, flags);
}

// ops.copy_pages on lists of ints; True when done
py::object copy_pages(const at::Tensor& pages, const py::object& src, const py::object& dst, int flags) {
    const int dev = here(pages);
    if (dev < 0 || pages.dim() < 4 || !pages.is_contiguous() || pages.numel() == 0 || !PyList_CheckExact(src.ptr()) ||
        !PyList_CheckExact(dst.ptr()) || PyList_GET_SIZE(src.ptr()) != PyList_GET_SIZE(dst.ptr()) || PyList_GET_SIZE(src.ptr()) > 0x7fffffff) {
        return py::none();
    }
    const Py_ssize_t n = PyList_GET_SIZE(src.ptr());
    std::vector<int> ids(2 * n);
    for (int side = 0; side < 2; ++side) {
        PyObject* list = side == 0 ? src.ptr() : dst.ptr();
        for (Py_ssize_t i = 0; i < n; ++i) {
            PyObject* x = PyList_GET_ITEM(list, i);
            int overflow = 0;
            const long id = PyLong_CheckExact(x) ? PyLong_AsLongAndOverflow(x, &overflow) : -1;
            if (overflow != 0 || id < 0 || id > 0x7fffffff) return py::none();       // refused by the Python form
            ids[side * n + i] = static_cast<int>(id);
        }
    }
    if (n == 0) return py::bool_(true);
    // not by strides: those of one page may be anything
    const int64_t P = pages.size(-4), page_bytes = pages.size(-3) * pages.size(-2) * pages.size(-1) * pages.element_size(), slab = page_bytes * P;
    const int64_t slabs = static_cast<int64_t>(pages.nbytes()) / slab;
    if (!fits({P, slabs})) return py::none();
    void* base = pages.data_ptr();
    const tpb200_stream_t s = stream_of(dev);
    const int st = launch([&] {
        return g.copy_pages(base, slab, static_cast<int>(slabs), page_bytes, static_cast<int>(P), ids.data(), ids.data() + n,
                            static_cast<int>(n), flags, s);
    });
    return st == 0 ? py::object(py::bool_(true)) : py::int_(st);
}

}  // namespace

PYBIND11_MODULE(_calls, m) {
    m.def("bind", &bind);
    m.def("w4_gemm", &w4_gemm);
    m.def("mlp", &mlp);
    m.def("w4a16_linear", &w4a16_linear);
    m.def("attention", &attention);
    m.def("quantize_fp8", &quantize_fp8);
    m.def("nvfp4_linear", &nvfp4_linear);
    m.def("packed_attention", &packed_attention);
    m.def("paged_attention", &paged_attention);
    m.def("paged_append", &paged_append);
    m.def("copy_pages", &copy_pages);
    m.def("packed_attention_window", &packed_attention_window);
    m.def("paged_attention_window", &paged_attention_window);
    m.def("paged_attention_nvfp4", &paged_attention_nvfp4);
    m.def("paged_append_nvfp4", &paged_append_nvfp4);
    m.def("paged_read", &paged_read);
    m.def("paged_read_nvfp4", &paged_read_nvfp4);
}
