// torch.ops.catccos.*: the operator-library face of the HIP library, as a C++ translation unit.
//
// Mirrors the reference's torch binding (examples/torch_binding/src/torch_bindings.cpp:84-239:
// `TORCH_LIBRARY(catccos, m)` with `init` / `<op>` / `finalize`, state in a function-local static, inputs
// checked with TORCH_CHECK and made contiguous, output allocated here, current stream taken, the extern "C"
// wrapper called; the device implementation registered for the accelerator key only) and its Meta twin
// (examples/torch_binding/src/torch_bindings_meta.cpp:18-35: output shapes only), for the compute halves
// this library holds instead of `allgather_matmul`.  There is no communication here, so `init` accepts
// rank_size == 1 only and makes no use of local_mem_size / ip_port (the symmetric heap they size is the
// part that was dropped).
//
// Behaviour kept from the reference: an operator called before `init` fails with the reference's message
// (torch_bindings.cpp:131-133); `init` checks its arguments like the reference and is a no-op the second
// time (:88-95); `finalize` on an uninitialised library returns 0 (:205-207).
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <atomic>
#include <cctype>
#include <functional>
#include <initializer_list>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>

#include "catccos_hip.h"

namespace {

struct CatccosTorchState {
    std::atomic<bool> initialized{false};   // read without the lock by every operator
    std::atomic<bool> launched{false};      // some operator of this library has put work on a stream
    int64_t rank_id = -1, rank_size = 0;
    std::mutex mu;
};

CatccosTorchState &State()
{
    static CatccosTorchState state;
    return state;
}

void NeedInit()
{
    TORCH_CHECK(State().initialized.load(std::memory_order_acquire), "catccos TORCH_LIBRARY not initialized, call torch.ops.catccos.init(...) first");
}

// Every tensor argument of a device kernel must live on the GPU of the first one.  The dispatcher picks the GPU
// kernel as soon as one argument is a GPU tensor; a host tensor among the others (group sizes often live on the
// host) would hand a host address to a kernel (the reference checks the same, torch_bindings.cpp:140-144).  Called
// before anything is allocated or launched.
struct NamedTensor {
    const char *name;
    const at::Tensor &t;
};
void SameDevice(const char *op, std::initializer_list<NamedTensor> args)
{
    const NamedTensor &first = *args.begin();
    for (const NamedTensor &a : args) {
        TORCH_CHECK(a.t.defined(), "catccos::", op, ": ", a.name, " is undefined");
        TORCH_CHECK(a.t.is_cuda(), "catccos::", op, ": ", a.name, " must be a GPU tensor, got one on ", a.t.device());
        TORCH_CHECK(a.t.device() == first.t.device(), "catccos::", op, ": ", a.name, " is on ", a.t.device(), " but ", first.name, " is on ",
                    first.t.device());
    }
}

int FormatCode(const std::string &name)
{
    std::string s = name;
    std::transform(s.begin(), s.end(), s.begin(), [](unsigned char c) { return std::tolower(c); });
    if (s == "e4m3" || s == "fp8") return CCH_FMT_E4M3;
    if (s == "e5m2") return CCH_FMT_E5M2;
    if (s == "e2m1" || s == "fp4") return CCH_FMT_E2M1;
    if (s == "e1m2") return CCH_FMT_E1M2;
    TORCH_CHECK(false, "unknown MX payload format '", name, "'");
    return -1;
}

bool IsFp4(int fmt) { return fmt == CCH_FMT_E2M1 || fmt == CCH_FMT_E1M2; }
int64_t ScaleCols(int64_t k) { return 2 * ((k + 63) / 64); }   // E8M0 bytes per row: block count padded to even

// (a ROCm build of PyTorch presents its HIP devices and streams under the names of the GPU key: the stream of a
// tensor's device is asked for through that front)
void *StreamOf(const at::Tensor &t)
{
    State().launched.store(true, std::memory_order_release);
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

void Check(int rc, const char *what) { TORCH_CHECK(rc == CCH_OK, "catccos::", what, ": ", cch_last_error()); }

at::Tensor Bytes(const at::Tensor &like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kByte)); }

// ---------------------------------------------------------------------------------------------
// init / finalize (reference torch_bindings.cpp:85-121, :203-229)

int64_t Init(int64_t rank_id, int64_t rank_size, int64_t local_mem_size, std::string ip_port)
{
    auto &st = State();
    std::lock_guard<std::mutex> lock(st.mu);
    if (st.initialized.load()) return 0;
    TORCH_CHECK(rank_id >= 0, "invalid rank_id: ", rank_id);
    TORCH_CHECK(rank_size > 0, "invalid rank_size: ", rank_size);
    TORCH_CHECK(local_mem_size > 0, "invalid local_mem_size: ", local_mem_size);
    TORCH_CHECK(!ip_port.empty(), "ip_port is empty");
    TORCH_CHECK(rank_size == 1 && rank_id == 0, "catccos on one GPU has no peers: rank_size must be 1 and rank_id 0, got ", rank_id, " of ",
                rank_size);
    st.rank_id = rank_id;
    st.rank_size = rank_size;
    st.initialized.store(true, std::memory_order_release);
    return 0;
}

int64_t Finalize()
{
    auto &st = State();
    std::lock_guard<std::mutex> lock(st.mu);
    if (!st.initialized.load()) return 0;
    // the reference drains its stream before it lets go of its buffers; a process in which no operator of this
    // library ever launched (only init / finalize or Meta-shape calls) has nothing to drain and must not create a
    // GPU context here
    if (st.launched.load(std::memory_order_acquire)) (void)hipStreamSynchronize(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream());
    st.initialized.store(false, std::memory_order_release);
    st.rank_id = -1;
    st.rank_size = 0;
    return 0;
}

// ---------------------------------------------------------------------------------------------
// shape helpers shared by the device and the Meta kernels

struct MxShape {
    int fmt;
    int64_t t, n, k, e;
};

// a [T, K(/2)] payload with sa [T, ScaleCols(K)]; b [(E,) K, N(/2)] or [(E,) N, K(/2)] with sb of E * ScaleCols(K) * N bytes
MxShape MxShapes(const at::Tensor &a, const at::Tensor &sa, const at::Tensor &b, const at::Tensor &sb, const std::string &fmt_name, int64_t trans_b,
                 bool grouped)
{
    MxShape s;
    s.fmt = FormatCode(fmt_name);
    TORCH_CHECK(s.fmt != CCH_FMT_E1M2, "E1M2 is a quantiser format only: the matrix instructions have no such operand type");
    const int64_t pack = s.fmt == CCH_FMT_E2M1 ? 2 : 1;
    TORCH_CHECK(a.dim() == 2 && a.scalar_type() == at::kByte, "a must be a 2-D uint8 tensor");
    TORCH_CHECK(sa.dim() == 2 && sa.scalar_type() == at::kByte, "sa must be a 2-D uint8 tensor");
    TORCH_CHECK(b.dim() == (grouped ? 3 : 2) && b.scalar_type() == at::kByte && sb.scalar_type() == at::kByte, "b / sb must be uint8 tensors of rank ",
                grouped ? 3 : 2);
    s.t = a.size(0);
    s.k = a.size(1) * pack;
    const int64_t d0 = b.size(grouped ? 1 : 0), d1 = b.size(grouped ? 2 : 1);
    const int64_t kb = trans_b ? d1 * pack : d0;
    s.n = trans_b ? d0 : d1 * pack;
    TORCH_CHECK(kb == s.k, "inner dimensions differ: a gives K=", s.k, ", b gives K=", kb);
    TORCH_CHECK(sa.size(0) == s.t && sa.size(1) == ScaleCols(s.k), "sa must be [", s.t, ",", ScaleCols(s.k), "]");
    s.e = grouped ? b.size(0) : 1;
    TORCH_CHECK(sb.numel() == s.e * ScaleCols(s.k) * s.n, "sb has ", sb.numel(), " entries, expected ", s.e * ScaleCols(s.k) * s.n);
    return s;
}

void CheckGroups(const at::Tensor &group_sizes, int64_t e)
{
    TORCH_CHECK(group_sizes.dim() == 1 && group_sizes.scalar_type() == at::kInt, "group_sizes must be a 1-D int32 tensor");
    TORCH_CHECK(group_sizes.numel() == e, "group_sizes must have one entry per expert");
}

struct I8Shape {
    int64_t t, n, k, e;
};

I8Shape I8GroupedShapes(const at::Tensor &x, const at::Tensor &w, const at::Tensor &group_sizes, const at::Tensor &per_tok, const at::Tensor &per_ch,
                        int64_t trans_b)
{
    TORCH_CHECK(x.dim() == 2 && x.scalar_type() == at::kChar, "x must be a 2-D int8 tensor");
    TORCH_CHECK(w.dim() == 3 && w.scalar_type() == at::kChar, "w must be a 3-D int8 tensor");
    I8Shape s{x.size(0), trans_b ? w.size(1) : w.size(2), x.size(1), w.size(0)};
    TORCH_CHECK((trans_b ? w.size(2) : w.size(1)) == s.k, "shape mismatch between x and w");
    CheckGroups(group_sizes, s.e);
    TORCH_CHECK(per_tok.numel() == s.t && per_ch.dim() == 2 && per_ch.size(0) == s.e && per_ch.size(1) == s.n, "per_tok must be [T] and per_ch [E,N]");
    return s;
}

// ---------------------------------------------------------------------------------------------
// device kernels (registered for the GPU key)

std::tuple<at::Tensor, at::Tensor> MxQuant(const at::Tensor &x_in, std::string fmt_name, int64_t rounding)
{
    NeedInit();
    const int fmt = FormatCode(fmt_name);
    TORCH_CHECK(x_in.dim() == 2 && (x_in.scalar_type() == at::kBFloat16 || x_in.scalar_type() == at::kHalf),
                "mx_quant expects a 2-D bfloat16 (or float16) tensor");
    SameDevice("mx_quant", {{"x", x_in}});
    c10::DeviceGuard guard(x_in.device());
    const at::Tensor x = x_in.contiguous();
    const int64_t m = x.size(0), k = x.size(1);
    at::Tensor payload = Bytes(x, {m, IsFp4(fmt) ? (k + 1) / 2 : k}), scales = Bytes(x, {m, ScaleCols(k)});
    const int rc = x.scalar_type() == at::kHalf
                       ? cch_mx_quant_rows_f16(x.data_ptr(), payload.data_ptr(), scales.data_ptr(), m, k, fmt, (int)rounding, StreamOf(x))
                       : cch_mx_quant_rows(x.data_ptr(), payload.data_ptr(), scales.data_ptr(), m, k, fmt, (int)rounding, StreamOf(x));
    Check(rc, "mx_quant");
    return {payload, scales};
}

at::Tensor W8A8MatmulDequant(const at::Tensor &a_in, const at::Tensor &b_in, const at::Tensor &per_tok_in, const at::Tensor &per_ch_in, int64_t trans_b)
{
    NeedInit();
    TORCH_CHECK(a_in.dim() == 2 && a_in.scalar_type() == at::kChar, "a must be a 2-D int8 tensor");
    TORCH_CHECK(b_in.dim() == 2 && b_in.scalar_type() == at::kChar, "b must be a 2-D int8 tensor");
    SameDevice("w8a8_matmul_dequant", {{"a", a_in}, {"b", b_in}, {"per_tok", per_tok_in}, {"per_ch", per_ch_in}});
    c10::DeviceGuard guard(a_in.device());
    const at::Tensor a = a_in.contiguous(), b = b_in.contiguous();
    const int64_t m = a.size(0), k = a.size(1), n = trans_b ? b.size(0) : b.size(1);
    TORCH_CHECK((trans_b ? b.size(1) : b.size(0)) == k, "inner dimensions differ");
    const at::Tensor per_tok = per_tok_in.contiguous().to(at::kFloat), per_ch = per_ch_in.contiguous().to(at::kFloat);
    TORCH_CHECK(per_tok.numel() == m && per_ch.numel() == n, "per_tok must have M entries and per_ch N entries");
    at::Tensor out = at::empty({m, n}, a.options().dtype(at::kBFloat16));
    Check(cch_gemm_i8_dequant_out(a.data_ptr(), b.data_ptr(), per_tok.data_ptr<float>(), per_ch.data_ptr<float>(), out.data_ptr(), m, n, k, (int)trans_b,
                                  CCH_OUT_BF16, StreamOf(a)),
          "w8a8_matmul_dequant");
    return out;
}

at::Tensor MxMatmul(const at::Tensor &a_in, const at::Tensor &sa_in, const at::Tensor &b_in, const at::Tensor &sb_in, std::string fmt_name, int64_t trans_b)
{
    NeedInit();
    SameDevice("mx_matmul", {{"a", a_in}, {"sa", sa_in}, {"b", b_in}, {"sb", sb_in}});
    c10::DeviceGuard guard(a_in.device());
    const at::Tensor a = a_in.contiguous(), sa = sa_in.contiguous(), b = b_in.contiguous(), sb = sb_in.contiguous();
    const MxShape s = MxShapes(a, sa, b, sb, fmt_name, trans_b, false);
    at::Tensor out = at::empty({s.t, s.n}, a.options().dtype(at::kBFloat16));
    Check(cch_mx_gemm_out(a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), out.data_ptr(), s.t, s.n, s.k, s.fmt, (int)trans_b, CCH_OUT_BF16,
                          StreamOf(a)),
          "mx_matmul");
    return out;
}

at::Tensor GmmDequantSwiglu(const at::Tensor &x_in, const at::Tensor &w_in, const at::Tensor &gs_in, const at::Tensor &per_tok_in,
                            const at::Tensor &per_ch_in, int64_t trans_b)
{
    NeedInit();
    SameDevice("gmm_dequant_swiglu", {{"x", x_in}, {"w", w_in}, {"group_sizes", gs_in}, {"per_tok", per_tok_in}, {"per_ch", per_ch_in}});
    c10::DeviceGuard guard(x_in.device());
    const at::Tensor x = x_in.contiguous(), w = w_in.contiguous(), gs = gs_in.contiguous();
    const at::Tensor per_tok = per_tok_in.contiguous().to(at::kFloat), per_ch = per_ch_in.contiguous().to(at::kFloat);
    const I8Shape s = I8GroupedShapes(x, w, gs, per_tok, per_ch, trans_b);
    at::Tensor out = at::empty({s.t, s.n / 2}, x.options().dtype(at::kBFloat16));
    Check(cch_gmm_i8_dequant_swiglu_out(x.data_ptr(), w.data_ptr(), gs.data_ptr<int32_t>(), per_tok.data_ptr<float>(), per_ch.data_ptr<float>(),
                                        out.data_ptr(), s.e, s.t, s.n, s.k, (int)trans_b, CCH_OUT_BF16, StreamOf(x)),
          "gmm_dequant_swiglu");
    return out;
}

std::tuple<at::Tensor, at::Tensor> GmmDequantSwigluMx(const at::Tensor &x_in, const at::Tensor &w_in, const at::Tensor &gs_in, const at::Tensor &per_tok_in,
                                                      const at::Tensor &per_ch_in, int64_t trans_b, std::string fmt_name)
{
    NeedInit();
    const int fmt = FormatCode(fmt_name);
    SameDevice("gmm_dequant_swiglu_mx", {{"x", x_in}, {"w", w_in}, {"group_sizes", gs_in}, {"per_tok", per_tok_in}, {"per_ch", per_ch_in}});
    c10::DeviceGuard guard(x_in.device());
    const at::Tensor x = x_in.contiguous(), w = w_in.contiguous(), gs = gs_in.contiguous();
    const at::Tensor per_tok = per_tok_in.contiguous().to(at::kFloat), per_ch = per_ch_in.contiguous().to(at::kFloat);
    const I8Shape s = I8GroupedShapes(x, w, gs, per_tok, per_ch, trans_b);
    TORCH_CHECK(s.n % 2 == 0 && (fmt != CCH_FMT_E2M1 || s.n % 4 == 0), "n must be even (a multiple of 4 for FP4 output)");
    const int64_t h = s.n / 2;
    at::Tensor payload = Bytes(x, {s.t, fmt == CCH_FMT_E2M1 ? h / 2 : h}), scales = Bytes(x, {s.t, ScaleCols(h)});
    Check(cch_gmm_i8_dequant_swiglu_mx(x.data_ptr(), w.data_ptr(), gs.data_ptr<int32_t>(), per_tok.data_ptr<float>(), per_ch.data_ptr<float>(),
                                       payload.data_ptr(), scales.data_ptr(), s.e, s.t, s.n, s.k, (int)trans_b, fmt, StreamOf(x)),
          "gmm_dequant_swiglu_mx");
    return {payload, scales};
}

at::Tensor MxGroupedMatmul(const at::Tensor &a_in, const at::Tensor &sa_in, const at::Tensor &b_in, const at::Tensor &sb_in, const at::Tensor &gs_in,
                           std::string fmt_name, int64_t trans_b)
{
    NeedInit();
    SameDevice("mx_grouped_matmul", {{"a", a_in}, {"sa", sa_in}, {"b", b_in}, {"sb", sb_in}, {"group_sizes", gs_in}});
    c10::DeviceGuard guard(a_in.device());
    const at::Tensor a = a_in.contiguous(), sa = sa_in.contiguous(), b = b_in.contiguous(), sb = sb_in.contiguous(), gs = gs_in.contiguous();
    const MxShape s = MxShapes(a, sa, b, sb, fmt_name, trans_b, true);
    CheckGroups(gs, s.e);
    at::Tensor out = at::empty({s.t, s.n}, a.options().dtype(at::kBFloat16));
    Check(cch_mx_gmm(a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), gs.data_ptr<int32_t>(), out.data_ptr(), s.e, s.t, s.n, s.k, s.fmt,
                     (int)trans_b, StreamOf(a)),
          "mx_grouped_matmul");
    return out;
}

std::tuple<at::Tensor, at::Tensor> MxGroupedMatmulSwigluMx(const at::Tensor &a_in, const at::Tensor &sa_in, const at::Tensor &b_in, const at::Tensor &sb_in,
                                                           const at::Tensor &gs_in, std::string fmt_name, int64_t trans_b, std::string out_fmt_name)
{
    NeedInit();
    const int ofmt = FormatCode(out_fmt_name);
    SameDevice("mx_grouped_matmul_swiglu_mx", {{"a", a_in}, {"sa", sa_in}, {"b", b_in}, {"sb", sb_in}, {"group_sizes", gs_in}});
    c10::DeviceGuard guard(a_in.device());
    const at::Tensor a = a_in.contiguous(), sa = sa_in.contiguous(), b = b_in.contiguous(), sb = sb_in.contiguous(), gs = gs_in.contiguous();
    const MxShape s = MxShapes(a, sa, b, sb, fmt_name, trans_b, true);
    CheckGroups(gs, s.e);
    TORCH_CHECK(s.n % 2 == 0 && (ofmt != CCH_FMT_E2M1 || s.n % 4 == 0), "n must be even (a multiple of 4 for FP4 output)");
    const int64_t h = s.n / 2;
    at::Tensor payload = Bytes(a, {s.t, ofmt == CCH_FMT_E2M1 ? h / 2 : h}), scales = Bytes(a, {s.t, ScaleCols(h)});
    Check(cch_mx_gmm_swiglu_mx(a.data_ptr(), sa.data_ptr(), b.data_ptr(), sb.data_ptr(), gs.data_ptr<int32_t>(), payload.data_ptr(), scales.data_ptr(), s.e,
                               s.t, s.n, s.k, s.fmt, (int)trans_b, ofmt, StreamOf(a)),
          "mx_grouped_matmul_swiglu_mx");
    return {payload, scales};
}

// The MXFP8 MoE FFN of one rank that holds every expert, routing to combine (the reference's
// Ascend950DispatchFFNCombine, examples/ascend950_dispatch_ffn_combine/ascend950_dispatch_ffn_combine_device.h:124-176):
// routing sort -> MXFP8 quantise-and-scatter -> GMM1 + SwiGLU + MXFP8 quantise -> GMM2 -> weighted un-permute.
at::Tensor MoeFfnMxfp8(const at::Tensor &x_in, const at::Tensor &expert_idx_in, const at::Tensor &probs_in, const at::Tensor &w1_in, const at::Tensor &sw1_in,
                       const at::Tensor &w2_in, const at::Tensor &sw2_in, int64_t trans_b)
{
    NeedInit();
    TORCH_CHECK(x_in.dim() == 2 && x_in.scalar_type() == at::kBFloat16, "x must be a 2-D bfloat16 tensor");
    TORCH_CHECK(expert_idx_in.dim() == 2 && expert_idx_in.size(0) == x_in.size(0) && expert_idx_in.scalar_type() == at::kInt,
                "expert_idx must be an int32 [m, top_k] tensor");
    TORCH_CHECK(probs_in.sizes() == expert_idx_in.sizes() && probs_in.scalar_type() == at::kFloat, "probs must be a float32 [m, top_k] tensor");
    TORCH_CHECK(w1_in.dim() == 3 && w2_in.dim() == 3 && w1_in.size(0) == w2_in.size(0), "w1 and w2 must hold one matrix per expert");
    SameDevice("moe_ffn_mxfp8", {{"x", x_in}, {"expert_idx", expert_idx_in}, {"probs", probs_in}, {"w1", w1_in}, {"sw1", sw1_in}, {"w2", w2_in}, {"sw2", sw2_in}});
    c10::DeviceGuard guard(x_in.device());
    const at::Tensor x = x_in.contiguous(), idx = expert_idx_in.contiguous(), probs = probs_in.contiguous();
    const at::Tensor w1 = w1_in.contiguous(), sw1 = sw1_in.contiguous(), w2 = w2_in.contiguous(), sw2 = sw2_in.contiguous();
    const int64_t m = x.size(0), k = x.size(1), top_k = idx.size(1), e = w1.size(0);
    const int64_t n = trans_b ? w1.size(1) : w1.size(2), h = n / 2;
    TORCH_CHECK((trans_b ? w1.size(2) : w1.size(1)) == k && n % 2 == 0, "w1 must be [E, k, n] (trans_b: [E, n, k]) with n even");
    TORCH_CHECK((trans_b ? w2.size(2) : w2.size(1)) == h && (trans_b ? w2.size(1) : w2.size(2)) == k, "w2 must be [E, n/2, k] (trans_b: [E, k, n/2])");
    TORCH_CHECK(sw1.numel() == e * ScaleCols(k) * n && sw2.numel() == e * ScaleCols(h) * k, "scale tensors do not match the weights");
    TORCH_CHECK(top_k >= 1 && top_k <= 8, "top_k must be 1..8");
    at::Tensor out = at::empty({m, k}, x.options());
    const int64_t ws_bytes = cch_moe_ffn_mxfp8_workspace_bytes(m, k, (int)top_k, e, n);
    at::Tensor ws = Bytes(x, {ws_bytes});
    Check(cch_moe_ffn_mxfp8(x.data_ptr(), idx.data_ptr<int32_t>(), probs.data_ptr<float>(), w1.data_ptr(), sw1.data_ptr(), w2.data_ptr(), sw2.data_ptr(),
                            out.data_ptr(), m, k, (int)top_k, e, n, (int)trans_b, ws.data_ptr(), ws_bytes, StreamOf(x)),
          "moe_ffn_mxfp8");
    return out;
}

// ---------------------------------------------------------------------------------------------
// The MoE gate, its balance loss (each with its gradient as a call of its own) and the products with 4-bit weights

typedef std::optional<at::Tensor> MaybeTensor;

int DtypeCode(const at::Tensor &t)
{
    if (t.scalar_type() == at::kBFloat16) return CCH_DTYPE_BF16;
    if (t.scalar_type() == at::kHalf) return CCH_DTYPE_F16;
    TORCH_CHECK(t.scalar_type() == at::kFloat, "bfloat16, float16 or float32 expected, got ", t.scalar_type());
    return CCH_DTYPE_F32;
}
int ScoringCode(const std::string &s)
{
    TORCH_CHECK(s == "softmax" || s == "sigmoid", "unknown scoring '", s, "' (softmax or sigmoid)");
    return s == "sigmoid" ? CCH_SCORING_SIGMOID : CCH_SCORING_SOFTMAX;
}
void CheckLogits(const at::Tensor &logits)
{
    TORCH_CHECK(logits.dim() == 2, "logits must be [tokens, experts]");
    DtypeCode(logits);
}

// An optional argument on `like`'s GPU, of the type and shape that the kernel takes it to be; contiguous.
at::Tensor Optional(const char *op, const char *name, const MaybeTensor &t, const at::Tensor &like, std::initializer_list<at::ScalarType> types, at::IntArrayRef shape)
{
    if (!t || !t->defined()) return at::Tensor();
    SameDevice(op, {{"the first argument", like}, {name, *t}});
    TORCH_CHECK(std::find(types.begin(), types.end(), t->scalar_type()) != types.end() && t->sizes() == shape, "catccos::", op, ": ", name, " must be a ", shape,
                " tensor of its type");
    return t->contiguous();
}
template <class T>
T *PtrOf(const at::Tensor &t)
{
    return t.defined() ? static_cast<T *>(t.data_ptr()) : nullptr;
}

std::tuple<at::Tensor, at::Tensor> MoeRouter(const at::Tensor &logits_in, int64_t top_k, std::string scoring, bool renormalize, double scale, const MaybeTensor &bias_in,
                                             const MaybeTensor &mask_in)
{
    NeedInit();
    CheckLogits(logits_in);
    SameDevice("moe_router", {{"logits", logits_in}});
    c10::DeviceGuard guard(logits_in.device());
    const at::Tensor logits = logits_in.contiguous();
    const int64_t tokens = logits.size(0), e = logits.size(1);
    TORCH_CHECK(top_k >= 1 && top_k <= 8 && top_k <= e, "top_k must be 1..8 and no more than the experts");
    const at::Tensor bias = Optional("moe_router", "bias", bias_in, logits, {at::kFloat}, e), mask = Optional("moe_router", "token_mask", mask_in, logits, {at::kBool, at::kByte}, tokens);
    at::Tensor probs = at::empty({tokens, top_k}, logits.options().dtype(at::kFloat)), idx = at::empty({tokens, top_k}, logits.options().dtype(at::kInt));
    Check(cch_moe_router(logits.data_ptr(), DtypeCode(logits), tokens, e, (int)top_k, ScoringCode(scoring), renormalize, (float)scale, PtrOf<float>(bias), PtrOf<uint8_t>(mask),
                         probs.data_ptr<float>(), idx.data_ptr<int32_t>(), StreamOf(logits)),
          "moe_router");
    return {probs, idx};
}

at::Tensor MoeRouterBackward(const at::Tensor &grad_in, const at::Tensor &logits_in, const at::Tensor &idx_in, std::string scoring, bool renormalize, double scale)
{
    NeedInit();
    CheckLogits(logits_in);
    SameDevice("moe_router_backward", {{"grad_probs", grad_in}, {"logits", logits_in}, {"expert_idx", idx_in}});
    TORCH_CHECK(idx_in.dim() == 2 && idx_in.size(0) == logits_in.size(0) && idx_in.scalar_type() == at::kInt, "expert_idx must be an int32 [tokens, top_k] tensor");
    TORCH_CHECK(grad_in.sizes() == idx_in.sizes() && grad_in.scalar_type() == at::kFloat, "grad_probs must be a float32 [tokens, top_k] tensor");
    c10::DeviceGuard guard(logits_in.device());
    const at::Tensor grad = grad_in.contiguous(), logits = logits_in.contiguous(), idx = idx_in.contiguous();
    at::Tensor out = at::empty(logits.sizes(), logits.options());
    Check(cch_moe_router_backward(grad.data_ptr<float>(), logits.data_ptr(), DtypeCode(logits), idx.data_ptr<int32_t>(), logits.size(0), logits.size(1), (int)idx.size(1),
                                  ScoringCode(scoring), renormalize, (float)scale, out.data_ptr(), StreamOf(logits)),
          "moe_router_backward");
    return out;
}

int64_t Sequences(const MaybeTensor &offsets)
{
    if (!offsets || !offsets->defined()) return 1;
    TORCH_CHECK(offsets->dim() == 1 && offsets->numel() >= 2, "seq_offsets must be an int32 [sequences + 1] tensor");
    return offsets->numel() - 1;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> MoeBalanceLoss(const at::Tensor &logits_in, const at::Tensor &idx_in, double coef, double z_coef, std::string scoring,
                                                              const MaybeTensor &mask_in, const MaybeTensor &offsets_in)
{
    NeedInit();
    CheckLogits(logits_in);
    SameDevice("moe_balance_loss", {{"logits", logits_in}, {"expert_idx", idx_in}});
    TORCH_CHECK(idx_in.dim() == 2 && idx_in.size(0) == logits_in.size(0) && idx_in.scalar_type() == at::kInt, "expert_idx must be an int32 [tokens, top_k] tensor");
    c10::DeviceGuard guard(logits_in.device());
    const at::Tensor logits = logits_in.contiguous(), idx = idx_in.contiguous();
    const int64_t tokens = logits.size(0), e = logits.size(1), s = Sequences(offsets_in);
    const at::Tensor mask = Optional("moe_balance_loss", "token_mask", mask_in, logits, {at::kBool, at::kByte}, tokens);
    const at::Tensor offsets = Optional("moe_balance_loss", "seq_offsets", offsets_in, logits, {at::kInt}, s + 1);
    at::Tensor loss = at::empty({}, logits.options().dtype(at::kFloat)), counted = at::empty({s}, logits.options().dtype(at::kInt));
    at::Tensor counts = offsets.defined() ? at::empty({s, e}, counted.options()) : at::empty({e}, counted.options());
    const int64_t ws_bytes = cch_moe_balance_loss_workspace_bytes(tokens, e, s);
    at::Tensor ws = Bytes(logits, {std::max<int64_t>(ws_bytes, 4)});
    Check(cch_moe_balance_loss(logits.data_ptr(), DtypeCode(logits), idx.data_ptr<int32_t>(), PtrOf<uint8_t>(mask), PtrOf<int32_t>(offsets), tokens, e, (int)idx.size(1), s,
                               ScoringCode(scoring), (float)coef, (float)z_coef, loss.data_ptr<float>(), counts.data_ptr<int32_t>(), counted.data_ptr<int32_t>(), ws.data_ptr(),
                               ws.numel(), StreamOf(logits)),
          "moe_balance_loss");
    return {loss, counts, counted};
}

at::Tensor MoeBalanceLossBackward(const at::Tensor &grad_in, const at::Tensor &logits_in, const at::Tensor &counts_in, const at::Tensor &counted_in, int64_t top_k, double coef,
                                  double z_coef, std::string scoring, const MaybeTensor &mask_in, const MaybeTensor &offsets_in)
{
    NeedInit();
    CheckLogits(logits_in);
    SameDevice("moe_balance_loss_backward", {{"grad_loss", grad_in}, {"logits", logits_in}, {"counts", counts_in}, {"tokens", counted_in}});
    c10::DeviceGuard guard(logits_in.device());
    const at::Tensor grad = grad_in.contiguous(), logits = logits_in.contiguous(), counts = counts_in.contiguous(), counted = counted_in.contiguous();
    const int64_t tokens = logits.size(0), e = logits.size(1), s = Sequences(offsets_in);
    TORCH_CHECK(grad.numel() == 1 && grad.scalar_type() == at::kFloat, "grad_loss must be one float32 value");
    TORCH_CHECK(counts.scalar_type() == at::kInt && counts.numel() == s * e && counted.scalar_type() == at::kInt && counted.numel() == s,
                "counts must be int32 [sequences, experts] and tokens int32 [sequences]");
    const at::Tensor mask = Optional("moe_balance_loss_backward", "token_mask", mask_in, logits, {at::kBool, at::kByte}, tokens);
    const at::Tensor offsets = Optional("moe_balance_loss_backward", "seq_offsets", offsets_in, logits, {at::kInt}, s + 1);
    at::Tensor out = at::empty(logits.sizes(), logits.options());
    Check(cch_moe_balance_loss_backward(grad.data_ptr<float>(), logits.data_ptr(), DtypeCode(logits), PtrOf<uint8_t>(mask), PtrOf<int32_t>(offsets), counts.data_ptr<int32_t>(),
                                        counted.data_ptr<int32_t>(), tokens, e, (int)top_k, s, ScoringCode(scoring), (float)coef, (float)z_coef, out.data_ptr(), StreamOf(logits)),
          "moe_balance_loss_backward");
    return out;
}

// Codes [.., rows, ceil(k/2)], scales and zero points of 4-bit weights, `lead` matrices of `rows` rows.
void CheckW4(const char *name, const at::Tensor &w, const at::Tensor &scales, const at::Tensor &zeros, int64_t lead, int64_t rows, int64_t k, int fmt, int64_t group,
             at::ScalarType type)
{
    const int64_t groups = fmt == CCH_FMT_INT4 ? (k + group - 1) / group : ScaleCols(k);
    TORCH_CHECK(w.scalar_type() == at::kByte && w.numel() == lead * rows * ((k + 1) / 2) && w.size(-1) == (k + 1) / 2 && w.size(-2) == rows, name, " must be a uint8 tensor of ",
                (k + 1) / 2, " bytes a row");
    TORCH_CHECK(scales.scalar_type() == (fmt == CCH_FMT_INT4 ? type : at::kByte) && scales.dim() == w.dim() && scales.size(-1) == groups &&
                    scales.sizes().slice(0, w.dim() - 1) == w.sizes().slice(0, w.dim() - 1),
                "scales of ", name, " must have a row of ", groups, " for each of its rows, of ", fmt == CCH_FMT_INT4 ? "the activations' type" : "E8M0 bytes");
    TORCH_CHECK(!zeros.defined() || (fmt == CCH_FMT_INT4 && zeros.scalar_type() == at::kByte && zeros.sizes() == scales.sizes()), "zeros of ", name,
                " must be uint8 of the scales' shape, with int4 weights only");
}
int W4Format(const std::string &name, int64_t group)
{
    TORCH_CHECK(name == "int4" || name == "e2m1" || name == "fp4", "unknown 4-bit weight format '", name, "' (int4 or e2m1)");
    TORCH_CHECK(name != "int4" || group == 32 || group == 64 || group == 128, "group_size must be 32, 64 or 128");
    return name == "int4" ? CCH_FMT_INT4 : CCH_FMT_E2M1;
}
at::Tensor Zeros(const char *op, const char *name, const MaybeTensor &zeros, const at::Tensor &x)
{
    return Optional(op, name, zeros, x, {at::kByte}, zeros && zeros->defined() ? zeros->sizes() : at::IntArrayRef());
}

at::Tensor W4A16Matmul(const at::Tensor &x_in, const at::Tensor &w_in, const at::Tensor &scales_in, const MaybeTensor &zeros_in, std::string fmt_name, int64_t group)
{
    NeedInit();
    const int fmt = W4Format(fmt_name, group);
    TORCH_CHECK(x_in.dim() == 2 && (x_in.scalar_type() == at::kBFloat16 || x_in.scalar_type() == at::kHalf), "x must be a 2-D bfloat16 or float16 tensor");
    TORCH_CHECK(w_in.dim() == 2 && scales_in.dim() == 2, "w and scales must be 2-D tensors");
    SameDevice("w4a16_matmul", {{"x", x_in}, {"w", w_in}, {"scales", scales_in}});
    c10::DeviceGuard guard(x_in.device());
    const at::Tensor x = x_in.contiguous(), w = w_in.contiguous(), scales = scales_in.contiguous(), zeros = Zeros("w4a16_matmul", "zeros", zeros_in, x);
    const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
    CheckW4("w", w, scales, zeros, 1, n, k, fmt, group, x.scalar_type());
    at::Tensor out = at::empty({m, n}, x.options());
    const int64_t ws_bytes = cch_w4a16_matmul_workspace_bytes(m, n, k);
    at::Tensor ws = Bytes(x, {ws_bytes});
    Check(cch_w4a16_matmul(x.data_ptr(), w.data_ptr(), scales.data_ptr(), PtrOf<void>(zeros), out.data_ptr(), m, n, k, fmt, (int)group, DtypeCode(x), ws.data_ptr(), ws_bytes,
                           StreamOf(x)),
          "w4a16_matmul");
    return out;
}

at::Tensor MoeFfnW4A16(const at::Tensor &x_in, const at::Tensor &idx_in, const at::Tensor &probs_in, const at::Tensor &w1_in, const at::Tensor &s1_in, const MaybeTensor &z1_in,
                       const at::Tensor &w2_in, const at::Tensor &s2_in, const MaybeTensor &z2_in, std::string fmt_name, int64_t group)
{
    NeedInit();
    const char *op = "moe_ffn_w4a16";
    const int fmt = W4Format(fmt_name, group);
    TORCH_CHECK(x_in.dim() == 2 && (x_in.scalar_type() == at::kBFloat16 || x_in.scalar_type() == at::kHalf), "x must be a 2-D bfloat16 or float16 tensor");
    TORCH_CHECK(idx_in.dim() == 2 && idx_in.size(0) == x_in.size(0) && idx_in.scalar_type() == at::kInt, "expert_idx must be an int32 [m, top_k] tensor");
    TORCH_CHECK(probs_in.sizes() == idx_in.sizes() && probs_in.scalar_type() == at::kFloat, "probs must be a float32 [m, top_k] tensor");
    TORCH_CHECK(w1_in.dim() == 3 && w2_in.dim() == 3 && s1_in.dim() == 3 && s2_in.dim() == 3 && w1_in.size(0) == w2_in.size(0) && w1_in.size(1) % 2 == 0,
                "w1 and w2 must hold one matrix per expert, w1 gate and up halves");
    SameDevice(op, {{"x", x_in}, {"expert_idx", idx_in}, {"probs", probs_in}, {"w1", w1_in}, {"scales1", s1_in}, {"w2", w2_in}, {"scales2", s2_in}});
    c10::DeviceGuard guard(x_in.device());
    const at::Tensor x = x_in.contiguous(), idx = idx_in.contiguous(), probs = probs_in.contiguous(), w1 = w1_in.contiguous(), s1 = s1_in.contiguous(), w2 = w2_in.contiguous(),
                     s2 = s2_in.contiguous(), z1 = Zeros(op, "zeros1", z1_in, x), z2 = Zeros(op, "zeros2", z2_in, x);
    const int64_t m = x.size(0), k = x.size(1), top_k = idx.size(1), e = w1.size(0), n = w1.size(1);
    TORCH_CHECK(top_k >= 1 && top_k <= 8, "top_k must be 1..8");
    CheckW4("w1", w1, s1, z1, e, n, k, fmt, group, x.scalar_type());
    CheckW4("w2", w2, s2, z2, e, k, n / 2, fmt, group, x.scalar_type());
    at::Tensor out = at::empty({m, k}, x.options());
    const int64_t ws_bytes = cch_moe_ffn_w4a16_workspace_bytes(m, k, (int)top_k, e, n);
    at::Tensor ws = Bytes(x, {std::max<int64_t>(ws_bytes, 1)});
    Check(cch_moe_ffn_w4a16(x.data_ptr(), idx.data_ptr<int32_t>(), probs.data_ptr<float>(), w1.data_ptr(), s1.data_ptr(), PtrOf<void>(z1), w2.data_ptr(), s2.data_ptr(),
                            PtrOf<void>(z2), out.data_ptr(), m, k, (int)top_k, e, n, fmt, (int)group, DtypeCode(x), ws.data_ptr(), ws.numel(), StreamOf(x)),
          op);
    return out;
}

// ---------------------------------------------------------------------------------------------
// Meta kernels: output shapes only (reference torch_bindings_meta.cpp:18-30 returns at::empty_symint of the result shape)

c10::SymInt SymScaleCols(const c10::SymInt &k) { return ((k + 63) / 64) * 2; }

at::Tensor MetaEmpty(const at::Tensor &like, c10::SymIntArrayRef shape, at::ScalarType dtype)
{
    return at::empty_symint(shape, like.options().dtype(dtype));
}

std::tuple<at::Tensor, at::Tensor> MxQuantMeta(const at::Tensor &x, std::string fmt_name, int64_t)
{
    const int fmt = FormatCode(fmt_name);
    const c10::SymInt m = x.sym_size(0), k = x.sym_size(1);
    return {MetaEmpty(x, {m, IsFp4(fmt) ? (k + 1) / 2 : k}, at::kByte), MetaEmpty(x, {m, SymScaleCols(k)}, at::kByte)};
}

c10::SymInt MxN(const at::Tensor &b, int first, int fmt, int64_t trans_b)
{
    return trans_b ? b.sym_size(first) : b.sym_size(first + 1) * (IsFp4(fmt) ? 2 : 1);
}

at::Tensor W8A8Meta(const at::Tensor &a, const at::Tensor &b, const at::Tensor &, const at::Tensor &, int64_t trans_b)
{
    return MetaEmpty(a, {a.sym_size(0), trans_b ? b.sym_size(0) : b.sym_size(1)}, at::kBFloat16);
}

at::Tensor MxMatmulMeta(const at::Tensor &a, const at::Tensor &, const at::Tensor &b, const at::Tensor &, std::string fmt_name, int64_t trans_b)
{
    return MetaEmpty(a, {a.sym_size(0), MxN(b, 0, FormatCode(fmt_name), trans_b)}, at::kBFloat16);
}

at::Tensor GmmSwigluMeta(const at::Tensor &x, const at::Tensor &w, const at::Tensor &, const at::Tensor &, const at::Tensor &, int64_t trans_b)
{
    return MetaEmpty(x, {x.sym_size(0), (trans_b ? w.sym_size(1) : w.sym_size(2)) / 2}, at::kBFloat16);
}

std::tuple<at::Tensor, at::Tensor> GmmSwigluMxMeta(const at::Tensor &x, const at::Tensor &w, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                                                   int64_t trans_b, std::string fmt_name)
{
    const c10::SymInt h = (trans_b ? w.sym_size(1) : w.sym_size(2)) / 2;
    return {MetaEmpty(x, {x.sym_size(0), IsFp4(FormatCode(fmt_name)) ? h / 2 : h}, at::kByte), MetaEmpty(x, {x.sym_size(0), SymScaleCols(h)}, at::kByte)};
}

at::Tensor MxGmmMeta(const at::Tensor &a, const at::Tensor &, const at::Tensor &b, const at::Tensor &, const at::Tensor &, std::string fmt_name, int64_t trans_b)
{
    return MetaEmpty(a, {a.sym_size(0), MxN(b, 1, FormatCode(fmt_name), trans_b)}, at::kBFloat16);
}

std::tuple<at::Tensor, at::Tensor> MxGmmSwigluMxMeta(const at::Tensor &a, const at::Tensor &, const at::Tensor &b, const at::Tensor &, const at::Tensor &,
                                                     std::string fmt_name, int64_t trans_b, std::string out_fmt_name)
{
    const c10::SymInt h = MxN(b, 1, FormatCode(fmt_name), trans_b) / 2;
    return {MetaEmpty(a, {a.sym_size(0), IsFp4(FormatCode(out_fmt_name)) ? h / 2 : h}, at::kByte), MetaEmpty(a, {a.sym_size(0), SymScaleCols(h)}, at::kByte)};
}

at::Tensor MoeFfnMeta(const at::Tensor &x, const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &,
                      const at::Tensor &, int64_t)
{
    return MetaEmpty(x, x.sym_sizes(), x.scalar_type());
}

std::tuple<at::Tensor, at::Tensor> MoeRouterMeta(const at::Tensor &logits, int64_t top_k, std::string, bool, double, const MaybeTensor &, const MaybeTensor &)
{
    return {MetaEmpty(logits, {logits.sym_size(0), top_k}, at::kFloat), MetaEmpty(logits, {logits.sym_size(0), top_k}, at::kInt)};
}
at::Tensor MoeRouterBackwardMeta(const at::Tensor &, const at::Tensor &logits, const at::Tensor &, std::string, bool, double)
{
    return MetaEmpty(logits, logits.sym_sizes(), logits.scalar_type());
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> MoeBalanceLossMeta(const at::Tensor &logits, const at::Tensor &, double, double, std::string, const MaybeTensor &,
                                                                  const MaybeTensor &offsets)
{
    const bool some = offsets && offsets->defined();
    const c10::SymInt e = logits.sym_size(1), s = some ? offsets->sym_size(0) - 1 : c10::SymInt(1);
    return {MetaEmpty(logits, {}, at::kFloat), some ? MetaEmpty(logits, {s, e}, at::kInt) : MetaEmpty(logits, {e}, at::kInt), MetaEmpty(logits, {s}, at::kInt)};
}
at::Tensor MoeBalanceLossBackwardMeta(const at::Tensor &, const at::Tensor &logits, const at::Tensor &, const at::Tensor &, int64_t, double, double, std::string,
                                      const MaybeTensor &, const MaybeTensor &)
{
    return MetaEmpty(logits, logits.sym_sizes(), logits.scalar_type());
}
at::Tensor W4A16Meta(const at::Tensor &x, const at::Tensor &w, const at::Tensor &, const MaybeTensor &, std::string, int64_t)
{
    return MetaEmpty(x, {x.sym_size(0), w.sym_size(0)}, x.scalar_type());
}
at::Tensor MoeFfnW4A16Meta(const at::Tensor &x, const at::Tensor &, const at::Tensor &, const at::Tensor &, const at::Tensor &, const MaybeTensor &, const at::Tensor &,
                           const at::Tensor &, const MaybeTensor &, std::string, int64_t)
{
    return MetaEmpty(x, x.sym_sizes(), x.scalar_type());
}

// ---------------------------------------------------------------------------------------------
// Autograd of the gate, the losses and the 4-bit products: the gradients that catccos_amd.ops' forms have, and an error where there are none.  A call with nothing to
// differentiate goes on to its kernel as it is.

template <auto F>
struct Below;   // the operator whose kernel is F, called below autograd
template <class R, class... A, R (*F)(A...)>
struct Below<F> {
    static R call(const char *name, A... a)
    {
        static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<R(A...)>();
        at::AutoDispatchBelowADInplaceOrView below;
        return op.call(a...);
    }
};
#define CCH_BELOW(f, name, ...) Below<&f>::call("catccos::" name, __VA_ARGS__)

// Some of the tensors are recorded.  A tangent is refused.
bool Recorded(const char *op, std::initializer_list<at::Tensor> tensors)
{
    bool some = false;
    for (const at::Tensor &t : tensors) {
        if (!t.defined()) continue;
        TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "catccos::", op, " has no forward-mode derivative");
        some = some || t.requires_grad();
    }
    return some && c10::GradMode::is_enabled();
}

typedef torch::autograd::AutogradContext Context;
typedef torch::autograd::variable_list Variables;

struct NoGradient : torch::autograd::Function<NoGradient> {
    static at::Tensor forward(Context *ctx, std::string op, std::function<at::Tensor()> call, const at::Tensor &, const MaybeTensor &)
    {
        ctx->saved_data["op"] = op;
        return call();
    }
    static Variables backward(Context *ctx, Variables)
    {
        TORCH_CHECK_NOT_IMPLEMENTED(false, "catccos::", ctx->saved_data["op"].toStringRef(), " has no gradient");
    }
};

at::Tensor MoeRouterBackwardAutograd(const at::Tensor &grad, const at::Tensor &logits, const at::Tensor &idx, std::string scoring, bool renormalize, double scale)
{
    auto call = [&] { return CCH_BELOW(MoeRouterBackward, "moe_router_backward", grad, logits, idx, scoring, renormalize, scale); };
    return Recorded("moe_router_backward", {grad, logits}) ? NoGradient::apply("moe_router_backward", call, grad, MaybeTensor(logits)) : call();
}
at::Tensor MoeBalanceLossBackwardAutograd(const at::Tensor &grad, const at::Tensor &logits, const at::Tensor &counts, const at::Tensor &counted, int64_t top_k, double coef,
                                          double z_coef, std::string scoring, const MaybeTensor &mask, const MaybeTensor &offsets)
{
    auto call = [&] { return CCH_BELOW(MoeBalanceLossBackward, "moe_balance_loss_backward", grad, logits, counts, counted, top_k, coef, z_coef, scoring, mask, offsets); };
    return Recorded("moe_balance_loss_backward", {grad, logits}) ? NoGradient::apply("moe_balance_loss_backward", call, grad, MaybeTensor(logits)) : call();
}
at::Tensor W4A16MatmulAutograd(const at::Tensor &x, const at::Tensor &w, const at::Tensor &scales, const MaybeTensor &zeros, std::string fmt, int64_t group)
{
    auto call = [&] { return CCH_BELOW(W4A16Matmul, "w4a16_matmul", x, w, scales, zeros, fmt, group); };
    return Recorded("w4a16_matmul", {x}) ? NoGradient::apply("w4a16_matmul", call, x, MaybeTensor()) : call();
}
at::Tensor MoeFfnW4A16Autograd(const at::Tensor &x, const at::Tensor &idx, const at::Tensor &probs, const at::Tensor &w1, const at::Tensor &s1, const MaybeTensor &z1,
                               const at::Tensor &w2, const at::Tensor &s2, const MaybeTensor &z2, std::string fmt, int64_t group)
{
    auto call = [&] { return CCH_BELOW(MoeFfnW4A16, "moe_ffn_w4a16", x, idx, probs, w1, s1, z1, w2, s2, z2, fmt, group); };
    return Recorded("moe_ffn_w4a16", {x, probs}) ? NoGradient::apply("moe_ffn_w4a16", call, x, MaybeTensor(probs)) : call();
}

struct RouterFunction : torch::autograd::Function<RouterFunction> {
    static Variables forward(Context *ctx, const at::Tensor &logits, int64_t top_k, std::string scoring, bool renormalize, double scale, const MaybeTensor &bias,
                             const MaybeTensor &mask)
    {
        const auto [probs, idx] = CCH_BELOW(MoeRouter, "moe_router", logits, top_k, scoring, renormalize, scale, bias, mask);
        ctx->save_for_backward({logits, idx});
        ctx->mark_non_differentiable({idx});
        ctx->saved_data["scoring"] = scoring;
        ctx->saved_data["renormalize"] = renormalize;
        ctx->saved_data["scale"] = scale;
        return {probs, idx};
    }
    static Variables backward(Context *ctx, Variables grads)
    {
        const Variables saved = ctx->get_saved_variables();
        return {MoeRouterBackwardAutograd(grads[0], saved[0], saved[1], ctx->saved_data["scoring"].toStringRef(), ctx->saved_data["renormalize"].toBool(),
                                          ctx->saved_data["scale"].toDouble()),
                {}, {}, {}, {}, {}, {}};
    }
};
std::tuple<at::Tensor, at::Tensor> MoeRouterAutograd(const at::Tensor &logits, int64_t top_k, std::string scoring, bool renormalize, double scale, const MaybeTensor &bias,
                                                     const MaybeTensor &mask)
{
    if (!Recorded("moe_router", {logits})) return CCH_BELOW(MoeRouter, "moe_router", logits, top_k, scoring, renormalize, scale, bias, mask);
    const Variables out = RouterFunction::apply(logits, top_k, scoring, renormalize, scale, bias, mask);
    return {out[0], out[1]};
}

struct BalanceLossFunction : torch::autograd::Function<BalanceLossFunction> {
    static Variables forward(Context *ctx, const at::Tensor &logits, const at::Tensor &idx, double coef, double z_coef, std::string scoring, const MaybeTensor &mask,
                             const MaybeTensor &offsets)
    {
        const auto [loss, counts, counted] = CCH_BELOW(MoeBalanceLoss, "moe_balance_loss", logits, idx, coef, z_coef, scoring, mask, offsets);
        ctx->save_for_backward({logits, counts, counted, mask.value_or(at::Tensor()), offsets.value_or(at::Tensor())});
        ctx->mark_non_differentiable({counts, counted});
        ctx->saved_data["top_k"] = idx.size(1);
        ctx->saved_data["coef"] = coef;
        ctx->saved_data["z_coef"] = z_coef;
        ctx->saved_data["scoring"] = scoring;
        return {loss, counts, counted};
    }
    static Variables backward(Context *ctx, Variables grads)
    {
        const Variables saved = ctx->get_saved_variables();
        const auto maybe = [](const at::Tensor &t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
        return {MoeBalanceLossBackwardAutograd(grads[0], saved[0], saved[1], saved[2], ctx->saved_data["top_k"].toInt(), ctx->saved_data["coef"].toDouble(),
                                               ctx->saved_data["z_coef"].toDouble(), ctx->saved_data["scoring"].toStringRef(), maybe(saved[3]), maybe(saved[4])),
                {}, {}, {}, {}, {}, {}};
    }
};
std::tuple<at::Tensor, at::Tensor, at::Tensor> MoeBalanceLossAutograd(const at::Tensor &logits, const at::Tensor &idx, double coef, double z_coef, std::string scoring,
                                                                      const MaybeTensor &mask, const MaybeTensor &offsets)
{
    if (!Recorded("moe_balance_loss", {logits})) return CCH_BELOW(MoeBalanceLoss, "moe_balance_loss", logits, idx, coef, z_coef, scoring, mask, offsets);
    const Variables out = BalanceLossFunction::apply(logits, idx, coef, z_coef, scoring, mask, offsets);
    return {out[0], out[1], out[2]};
}

}  // namespace

TORCH_LIBRARY(catccos, m)
{
    m.def("init(int rank_id, int rank_size, int local_mem_size, str ip_port) -> int");
    m.def("finalize() -> int");
    m.def("mx_quant(Tensor x, str fmt, int rounding) -> (Tensor, Tensor)");
    m.def("w8a8_matmul_dequant(Tensor a, Tensor b, Tensor per_tok, Tensor per_ch, int trans_b) -> Tensor");
    m.def("mx_matmul(Tensor a, Tensor sa, Tensor b, Tensor sb, str fmt, int trans_b) -> Tensor");
    m.def("gmm_dequant_swiglu(Tensor x, Tensor w, Tensor group_sizes, Tensor per_tok, Tensor per_ch, int trans_b) -> Tensor");
    m.def("mx_grouped_matmul(Tensor a, Tensor sa, Tensor b, Tensor sb, Tensor group_sizes, str fmt, int trans_b) -> Tensor");
    m.def("mx_grouped_matmul_swiglu_mx(Tensor a, Tensor sa, Tensor b, Tensor sb, Tensor group_sizes, str fmt, int trans_b, str out_fmt) -> (Tensor, Tensor)");
    m.def("gmm_dequant_swiglu_mx(Tensor x, Tensor w, Tensor group_sizes, Tensor per_tok, Tensor per_ch, int trans_b, str fmt) -> (Tensor, Tensor)");
    m.def("moe_ffn_mxfp8(Tensor x, Tensor expert_idx, Tensor probs, Tensor w1, Tensor sw1, Tensor w2, Tensor sw2, int trans_b) -> Tensor");
    m.def("moe_router(Tensor logits, int top_k, str scoring, bool renormalize, float scale, Tensor? bias, Tensor? token_mask) -> (Tensor, Tensor)");
    m.def("moe_router_backward(Tensor grad_probs, Tensor logits, Tensor expert_idx, str scoring, bool renormalize, float scale) -> Tensor");
    m.def("moe_balance_loss(Tensor logits, Tensor expert_idx, float coef, float z_coef, str scoring, Tensor? token_mask, Tensor? seq_offsets) -> (Tensor, Tensor, Tensor)");
    m.def("moe_balance_loss_backward(Tensor grad_loss, Tensor logits, Tensor counts, Tensor tokens, int top_k, float coef, float z_coef, str scoring, Tensor? token_mask, "
          "Tensor? seq_offsets) -> Tensor");
    m.def("w4a16_matmul(Tensor x, Tensor w, Tensor scales, Tensor? zeros, str fmt, int group_size) -> Tensor");
    m.def("moe_ffn_w4a16(Tensor x, Tensor expert_idx, Tensor probs, Tensor w1, Tensor scales1, Tensor? zeros1, Tensor w2, Tensor scales2, Tensor? zeros2, str fmt, "
          "int group_size) -> Tensor");
}

// init / finalize take no tensors: one kernel for every backend, as in the reference (torch_bindings.cpp:233-238)
TORCH_LIBRARY_IMPL(catccos, CompositeExplicitAutograd, m)
{
    m.impl("init", &Init);
    m.impl("finalize", &Finalize);
}

// the GPU key (HIP devices answer to it in a ROCm build of PyTorch); CPU tensors find no kernel
TORCH_LIBRARY_IMPL(catccos, CUDA, m)
{
    m.impl("mx_quant", &MxQuant);
    m.impl("w8a8_matmul_dequant", &W8A8MatmulDequant);
    m.impl("mx_matmul", &MxMatmul);
    m.impl("gmm_dequant_swiglu", &GmmDequantSwiglu);
    m.impl("mx_grouped_matmul", &MxGroupedMatmul);
    m.impl("mx_grouped_matmul_swiglu_mx", &MxGroupedMatmulSwigluMx);
    m.impl("gmm_dequant_swiglu_mx", &GmmDequantSwigluMx);
    m.impl("moe_ffn_mxfp8", &MoeFfnMxfp8);
    m.impl("moe_router", &MoeRouter);
    m.impl("moe_router_backward", &MoeRouterBackward);
    m.impl("moe_balance_loss", &MoeBalanceLoss);
    m.impl("moe_balance_loss_backward", &MoeBalanceLossBackward);
    m.impl("w4a16_matmul", &W4A16Matmul);
    m.impl("moe_ffn_w4a16", &MoeFfnW4A16);
}

TORCH_LIBRARY_IMPL(catccos, Meta, m)
{
    m.impl("mx_quant", &MxQuantMeta);
    m.impl("w8a8_matmul_dequant", &W8A8Meta);
    m.impl("mx_matmul", &MxMatmulMeta);
    m.impl("gmm_dequant_swiglu", &GmmSwigluMeta);
    m.impl("mx_grouped_matmul", &MxGmmMeta);
    m.impl("mx_grouped_matmul_swiglu_mx", &MxGmmSwigluMxMeta);
    m.impl("gmm_dequant_swiglu_mx", &GmmSwigluMxMeta);
    m.impl("moe_ffn_mxfp8", &MoeFfnMeta);
    m.impl("moe_router", &MoeRouterMeta);
    m.impl("moe_router_backward", &MoeRouterBackwardMeta);
    m.impl("moe_balance_loss", &MoeBalanceLossMeta);
    m.impl("moe_balance_loss_backward", &MoeBalanceLossBackwardMeta);
    m.impl("w4a16_matmul", &W4A16Meta);
    m.impl("moe_ffn_w4a16", &MoeFfnW4A16Meta);
}

TORCH_LIBRARY_IMPL(catccos, Autograd, m)
{
    m.impl("moe_router", &MoeRouterAutograd);
    m.impl("moe_router_backward", &MoeRouterBackwardAutograd);
    m.impl("moe_balance_loss", &MoeBalanceLossAutograd);
    m.impl("moe_balance_loss_backward", &MoeBalanceLossBackwardAutograd);
    m.impl("w4a16_matmul", &W4A16MatmulAutograd);
    m.impl("moe_ffn_w4a16", &MoeFfnW4A16Autograd);
}
