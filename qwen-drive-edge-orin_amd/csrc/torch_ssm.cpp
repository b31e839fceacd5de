// Torch ops of the state-space layers (registered by torch_binding.cpp's
// module): ssm_scan, ssm_step, causal_conv1d_prefill, request_blocks and
// gated_groupnorm over the C ABI of include/gdn_hip.h.  Like the other ops they
// allocate outputs and workspace through the caching allocator on the current
// stream of the inputs' device and raise RuntimeError for what they refuse.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <limits>
#include <optional>
#include <vector>

#include "gdn_hip.h"

namespace {

using OptTensor = std::optional<at::Tensor>;

hipStream_t current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

void check_hip(hipError_t err, const char* what) {
    TORCH_CHECK(err == hipSuccess, what, " failed: ", hipGetErrorString(err));
}

void on_device(const at::Tensor& t, const at::Tensor& x, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.device() == x.device(), name, " must be on x's HIP device");
}

int io_dtype(const at::Tensor& x) {
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
                "x must be bf16 or fp16");
    return x.scalar_type() == at::kBFloat16 ? GDN_DTYPE_BF16 : GDN_DTYPE_FP16;
}

// x without gaps at a 16-byte boundary, itself where it lies so
at::Tensor aligned16(const at::Tensor& x) {
    at::Tensor r = x.contiguous();
    return reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0 ? r : r.clone(at::MemoryFormat::Contiguous);
}

constexpr int64_t kMaxToken = 1 << 24;   // token strides of the kernels

// x [B, T, H, P] as the kernels read it in place: a row's heads next to each
// other, 16-byte aligned rows with strides that are multiples of 8; anything
// else is copied.
at::Tensor rows16(const at::Tensor& x) {
    const int64_t H = x.size(2), P = x.size(3);
    const bool ok = x.stride(3) == 1 && (H <= 1 || x.stride(2) == P) &&
                    (x.size(0) <= 1 || (x.stride(0) % 8 == 0 && x.stride(0) >= 0)) &&
                    (x.size(1) <= 1 || (x.stride(1) % 8 == 0 && x.stride(1) >= 0 &&
                                        x.stride(1) < kMaxToken)) &&
                    reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
    return ok ? x : aligned16(x);
}

// fp32 [H] parameters
const float* head_param(const at::Tensor& p, const at::Tensor& x, int64_t H, const char* name,
                        at::Tensor& keep) {
    on_device(p, x, name);
    TORCH_CHECK(p.scalar_type() == at::kFloat && p.dim() == 1 && p.size(0) == H, name,
                " must be fp32 [H]");
    keep = p.contiguous();
    return keep.data_ptr<float>();
}

// The checked arguments of a scan or step, and the tensors they point into
struct Inputs {
    gdn_ssm_inputs in{};
    at::Tensor x, dt, b, c, z, A_log, D, dt_bias;

    Inputs(const at::Tensor& x_, const at::Tensor& dt_, const at::Tensor& A_log_,
           const at::Tensor& b_, const at::Tensor& c_, const OptTensor& D_, const OptTensor& z_,
           const OptTensor& dt_bias_, double dt_min, double dt_max) {
        TORCH_CHECK(x_.is_cuda(), "x must be on a HIP device (the ops have no CPU path)");
        on_device(dt_, x_, "dt");
        on_device(b_, x_, "B");
        on_device(c_, x_, "C");
        in.io_dtype = io_dtype(x_);
        TORCH_CHECK(b_.scalar_type() == x_.scalar_type() && c_.scalar_type() == x_.scalar_type(),
                    "B and C must have the dtype of x");
        TORCH_CHECK(dt_.scalar_type() == x_.scalar_type() || dt_.scalar_type() == at::kFloat,
                    "dt must have the dtype of x or be fp32");
        in.dt_dtype = dt_.scalar_type() == at::kFloat ? GDN_DTYPE_FP32 : in.io_dtype;
        TORCH_CHECK(x_.dim() == 4 && b_.dim() == 4 && c_.dim() == 4 && dt_.dim() == 3, "bad ranks");
        const int64_t Bn = x_.size(0), T = x_.size(1), H = x_.size(2), P = x_.size(3);
        const int64_t G = b_.size(2), N = b_.size(3);
        TORCH_CHECK(c_.sizes() == b_.sizes(), "B/C shape mismatch");
        TORCH_CHECK(b_.size(0) == Bn && b_.size(1) == T && dt_.size(0) == Bn && dt_.size(1) == T &&
                        dt_.size(2) == H,
                    "batch/time/head mismatch");
        TORCH_CHECK(Bn >= 1 && H >= 1 && G >= 1 && H % G == 0, "H must be a multiple of G");
        TORCH_CHECK(P >= 16 && P <= 256 && P % 16 == 0,
                    "head dims are multiples of 16 up to 256 (got ", P, ")");
        TORCH_CHECK(N == 16 || N == 32 || N == 64 || N == 128 || N == 256,
                    "state dims are 16, 32, 64, 128 or 256 (got ", N, ")");
        TORCH_CHECK(Bn <= 0x7fffffff && T <= 0x40000000 && H * P < kMaxToken && G * N < kMaxToken,
                    "too many rows, or rows of 2^24 elements");
        TORCH_CHECK(dt_min >= 0 && dt_max >= dt_min, "0 <= dt_min <= dt_max");
        if (z_) {
            on_device(*z_, x_, "z");
            TORCH_CHECK(z_->scalar_type() == x_.scalar_type() && z_->sizes() == x_.sizes(),
                        "z must have the dtype and shape of x");
        }
        x = rows16(x_);
        b = rows16(b_);
        c = rows16(c_);
        if (z_) z = rows16(*z_);
        const bool dt_ok = (H <= 1 || dt_.stride(2) == 1) && dt_.stride(0) >= 0 &&
                           dt_.stride(1) >= 0 && (T <= 1 || dt_.stride(1) < kMaxToken);
        dt = dt_ok ? dt_ : dt_.contiguous();
        in.A_log = head_param(A_log_, x_, H, "A_log", A_log);
        in.D = D_ ? head_param(*D_, x_, H, "D", D) : nullptr;
        in.dt_bias = dt_bias_ ? head_param(*dt_bias_, x_, H, "dt_bias", dt_bias) : nullptr;
        auto batch = [&](const at::Tensor& t) { return Bn > 1 ? t.stride(0) : 0; };
        auto token = [&](const at::Tensor& t) { return T > 1 ? t.stride(1) : 0; };
        in.x = x.data_ptr();
        in.dt = dt.data_ptr();
        in.b = b.data_ptr();
        in.c = c.data_ptr();
        in.z = z_ ? z.data_ptr() : nullptr;
        in.x_batch = batch(x);
        in.x_token = token(x);
        in.dt_batch = batch(dt);
        in.dt_token = token(dt);
        in.b_batch = batch(b);
        in.b_token = token(b);
        in.c_batch = batch(c);
        in.c_token = token(c);
        if (z_) {
            in.z_batch = batch(z);
            in.z_token = token(z);
        }
        in.batch = (int)Bn;
        in.tokens = (int)T;
        in.heads = (int)H;
        in.head_dim = (int)P;
        in.groups = (int)G;
        in.state_dim = (int)N;
        in.dt_min = (float)dt_min;
        in.dt_max = (float)dt_max;
    }
};

at::Tensor cu_int32(const at::Tensor& cu, const at::Tensor& x) {
    on_device(cu, x, "cu_seqlens");
    TORCH_CHECK(cu.dim() == 1 && cu.numel() >= 2, "cu_seqlens must be a 1-D tensor [N+1]");
    TORCH_CHECK(cu.scalar_type() == at::kInt || cu.scalar_type() == at::kLong,
                "cu_seqlens must be int32 or int64");
    TORCH_CHECK(x.size(0) == 1, "cu_seqlens requires packed inputs with batch size 1");
    return cu.to(at::kInt).contiguous();
}

// slots int32 or int64 [n] as int32; what passes 32 bits stays outside any pool
at::Tensor slots_int32(const at::Tensor& slots, const at::Tensor& x, int64_t n) {
    on_device(slots, x, "slots");
    TORCH_CHECK((slots.scalar_type() == at::kInt || slots.scalar_type() == at::kLong) &&
                    slots.dim() == 1 && slots.size(0) == n,
                "slots must be int32 or int64, one per row");
    return slots.scalar_type() == at::kLong ? slots.clamp(-1, 0x7fffffff).to(at::kInt)
                                            : slots.contiguous();
}

// [y, final_state]
std::vector<at::Tensor> ssm_scan(const at::Tensor& x, const at::Tensor& dt, const at::Tensor& A_log,
                                 const at::Tensor& b, const at::Tensor& c, const OptTensor& D,
                                 const OptTensor& z, const OptTensor& dt_bias, const OptTensor& s0,
                                 const OptTensor& cu_seqlens, const OptTensor& blocks,
                                 int64_t block, double dt_min, double dt_max) {
    const Inputs a(x, dt, A_log, b, c, D, z, dt_bias, dt_min, dt_max);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t Bn = a.in.batch, T = a.in.tokens, H = a.in.heads, P = a.in.head_dim,
                  N = a.in.state_dim;
    int64_t seqs = Bn;
    at::Tensor cu, table;
    if (cu_seqlens) {
        cu = cu_int32(*cu_seqlens, x);
        seqs = cu.numel() - 1;
    }
    TORCH_CHECK(blocks.has_value() == (block != 0), "blocks and block go together");
    if (blocks) {
        TORCH_CHECK(cu_seqlens.has_value(), "blocks go with cu_seqlens");
        on_device(*blocks, x, "blocks");
        TORCH_CHECK(block >= 64 && block % 64 == 0 && block <= (1 << 20),
                    "block must be a multiple of 64");
        TORCH_CHECK(blocks->scalar_type() == at::kInt && blocks->dim() == 2 &&
                        blocks->size(1) == 4 && blocks->size(0) == T / block + seqs,
                    "blocks must be request_blocks' int32 [T / block + N, 4]");
        table = blocks->contiguous();
    } else {
        block = gdn_ssm_scan_block(&a.in, (int)seqs);
    }
    auto y = at::empty({Bn, T, H, P}, a.x.options());
    auto sf = at::empty({seqs, H, N, P}, a.x.options().dtype(at::kFloat));
    at::Tensor s0c;
    if (s0) {
        on_device(*s0, x, "s0");
        s0c = s0->to(at::kFloat).contiguous();
        TORCH_CHECK(s0c.sizes() == sf.sizes(), "s0 must be [N, H, state, head]");
    }
    const size_t bytes = gdn_ssm_scan_workspace_size(&a.in, (int)seqs, (int)block, cu.defined());
    TORCH_CHECK(bytes > 0, "unsupported scan configuration");
    auto ws = at::empty({(int64_t)bytes}, a.x.options().dtype(at::kByte));
    check_hip(gdn_ssm_scan(&a.in, y.data_ptr(), s0 ? s0c.data_ptr<float>() : nullptr,
                           sf.data_ptr<float>(), cu.defined() ? cu.data_ptr<int32_t>() : nullptr,
                           table.defined() ? table.data_ptr<int32_t>() : nullptr, (int)seqs,
                           (int)block, ws.data_ptr(), bytes, current_stream()),
              "gdn_ssm_scan");
    return {y, sf};
}

// The block that ssm_scan works on for these sizes (host arithmetic)
int64_t ssm_scan_block(int64_t tokens, int64_t batch, int64_t heads, int64_t head_dim,
                       int64_t groups, int64_t state_dim, int64_t num_seqs) {
    for (int64_t v : {batch, heads, head_dim, groups, state_dim, num_seqs})
        TORCH_CHECK(v >= 1 && v <= 0x40000000, "unsupported scan configuration");
    gdn_ssm_inputs in{};
    in.batch = (int)batch;
    in.heads = (int)heads;
    in.head_dim = (int)head_dim;
    in.groups = (int)groups;
    in.state_dim = (int)state_dim;
    TORCH_CHECK(tokens >= 0 && tokens <= 0x40000000, "bad token count");
    in.tokens = (int)tokens;
    const int block = gdn_ssm_scan_block(&in, (int)num_seqs);
    TORCH_CHECK(block > 0, "unsupported scan configuration");
    return block;
}

// y; the state is updated in place
at::Tensor ssm_step(const at::Tensor& x, const at::Tensor& dt, const at::Tensor& A_log,
                    const at::Tensor& b, const at::Tensor& c, at::Tensor state, const OptTensor& D,
                    const OptTensor& z, const OptTensor& dt_bias, const OptTensor& slots,
                    double dt_min, double dt_max) {
    const Inputs a(x, dt, A_log, b, c, D, z, dt_bias, dt_min, dt_max);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    on_device(state, x, "state");
    TORCH_CHECK(state.scalar_type() == at::kFloat && state.is_contiguous(),
                "state is updated in place and must be a contiguous fp32 tensor");
    TORCH_CHECK(state.dim() == 4 && state.size(1) == a.in.heads &&
                    state.size(2) == a.in.state_dim && state.size(3) == a.in.head_dim &&
                    (slots || state.size(0) == a.in.batch),
                "state must be [B (or slots), H, state, head]");
    at::Tensor sl;
    if (slots) {
        TORCH_CHECK(state.size(0) >= 1 && state.size(0) <= 0x7fffffff, "bad pool size");
        sl = slots_int32(*slots, x, a.in.batch);
    }
    auto y = at::empty({a.in.batch, a.in.tokens, a.in.heads, a.in.head_dim}, a.x.options());
    check_hip(gdn_ssm_step(&a.in, y.data_ptr(), state.data_ptr<float>(),
                           slots ? sl.data_ptr<int32_t>() : nullptr, (int)state.size(0),
                           current_stream()),
              "gdn_ssm_step");
    return y;
}

// x [B, D, T] -> [y [B, D, T] (a view of a contiguous [B, T, D]), state [N, D, L]]
std::vector<at::Tensor> causal_conv1d_prefill(const at::Tensor& x, const at::Tensor& weight,
                                              const OptTensor& bias, const OptTensor& state0,
                                              bool silu, const OptTensor& cu_seqlens,
                                              int64_t state_len) {
    TORCH_CHECK(x.is_cuda(), "x must be on a HIP device (the ops have no CPU path)");
    on_device(weight, x, "weight");
    if (bias) on_device(*bias, x, "bias");
    const int io = io_dtype(x);
    TORCH_CHECK(x.dim() == 3, "x must be [B, D, T]");
    const int64_t B = x.size(0), D = x.size(1), T = x.size(2);
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) == D, "weight must be [D, K]");
    const int64_t K = weight.size(1);
    TORCH_CHECK(K >= 2 && K <= 4, "2 to 4 taps");
    TORCH_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat,
                "weight must have the dtype of x or be fp32");
    TORCH_CHECK(!bias || (bias->scalar_type() == weight.scalar_type() && bias->dim() == 1 &&
                          bias->size(0) == D),
                "bias must be [D] in the dtype of weight");
    TORCH_CHECK(B >= 1 && D >= 8 && D % 8 == 0, "the channel count must be a multiple of 8");
    TORCH_CHECK(B <= 0x7fffffff && T <= 0x40000000 && D <= 0x7fffffff, "too many rows");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    int64_t seqs = B;
    at::Tensor cu;
    if (cu_seqlens) {
        cu = cu_int32(*cu_seqlens, x);
        seqs = cu.numel() - 1;
    }
    at::Tensor s0c;
    if (state0) {
        on_device(*state0, x, "state0");
        TORCH_CHECK(state0->scalar_type() == x.scalar_type() && state0->dim() == 3 &&
                        state0->size(0) == seqs && state0->size(1) == D,
                    "state0 must be [N, D, L] in the dtype of x");
        TORCH_CHECK(state_len == 0 || state_len == state0->size(2), "state0 must have state_len columns");
        state_len = state0->size(2);
        s0c = aligned16(*state0);
    }
    if (state_len == 0) state_len = K;
    TORCH_CHECK(state_len >= K - 1 && state_len <= 8, "state_len must be K - 1 .. 8");
    auto xt = x.transpose(1, 2);   // [B, T, D]
    const bool direct = xt.stride(2) == 1 && (B <= 1 || (xt.stride(0) % 8 == 0 && xt.stride(0) >= 0)) &&
                        (T <= 1 || (xt.stride(1) % 8 == 0 && xt.stride(1) >= 0)) &&
                        reinterpret_cast<uintptr_t>(xt.data_ptr()) % 16 == 0;
    if (!direct) xt = xt.contiguous();
    auto wc = aligned16(weight);
    at::Tensor bc;
    if (bias) bc = aligned16(*bias);
    auto yt = at::empty({B, T, D}, x.options());
    auto state = at::empty({seqs, D, state_len}, x.options());
    check_hip(gdn_causal_conv1d_prefill(
                  xt.data_ptr(), wc.data_ptr(), bias ? bc.data_ptr() : nullptr,
                  state0 ? s0c.data_ptr() : nullptr, yt.data_ptr(), state.data_ptr(), (int)B,
                  (int)T, (int)D, (int)K, (int)state_len, B <= 1 ? 0 : xt.stride(0),
                  T <= 1 ? 0 : xt.stride(1), T * D, D,
                  cu.defined() ? cu.data_ptr<int32_t>() : nullptr, (int)seqs, io,
                  weight.scalar_type() == at::kFloat ? GDN_DTYPE_FP32 : io, silu ? 1 : 0,
                  current_stream()),
              "gdn_causal_conv1d_prefill");
    return {yt.transpose(1, 2), state};
}

// [cu_seqlens [N+1], blocks [rows, 4], token_slots [total], token_pos [total]], all int32
std::vector<at::Tensor> request_blocks(const at::Tensor& lengths, int64_t total_tokens,
                                       int64_t block, const OptTensor& slots) {
    TORCH_CHECK(lengths.is_cuda(), "lengths must be on a HIP device (the ops have no CPU path)");
    TORCH_CHECK((lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong) &&
                    lengths.dim() == 1 && lengths.numel() >= 1,
                "lengths must be int32 or int64 [N]");
    const int64_t N = lengths.numel();
    TORCH_CHECK(N <= (1 << 24) && total_tokens >= 0 && total_tokens <= (1 << 30),
                "at most 2^24 requests and 2^30 tokens");
    TORCH_CHECK(block >= 64 && block % 64 == 0 && block <= (1 << 20), "block must be a multiple of 64");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(lengths.device());
    // 64-bit lengths beyond 32 bits are cut at the capacity, as any others
    at::Tensor len = lengths.scalar_type() == at::kLong ? lengths.clamp(0, total_tokens).to(at::kInt)
                                                        : lengths.contiguous();
    at::Tensor sl;
    if (slots) sl = slots_int32(*slots, lengths, N);
    const auto opt = lengths.options().dtype(at::kInt);
    const int64_t rows = gdn_request_block_rows((int)total_tokens, (int)N, (int)block);
    auto sums = at::empty({2, N + 1}, opt);
    auto cu = sums[0];
    auto table = at::empty({rows, 4}, opt);
    auto slot = at::empty({total_tokens}, opt);
    auto pos = at::empty({total_tokens}, opt);
    check_hip(gdn_request_blocks(len.data_ptr<int32_t>(), slots ? sl.data_ptr<int32_t>() : nullptr,
                                 (int)N, (int)total_tokens, (int)block, cu.data_ptr<int32_t>(),
                                 sums.data_ptr<int32_t>() + N + 1, table.data_ptr<int32_t>(),
                                 slot.data_ptr<int32_t>(), pos.data_ptr<int32_t>(),
                                 current_stream()),
              "gdn_request_blocks");
    return {cu, table, slot, pos};
}

// x and z [.., C] as rows one stride apart, in place where they lie so
at::Tensor as_rows(const at::Tensor& x, int64_t C, int64_t& stride) {
    at::Tensor r = x;
    bool ok = x.stride(-1) == 1 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
    int64_t step = -1;   // the row stride, from the innermost dimension with more than one row
    int64_t want = -1;
    for (int64_t d = x.dim() - 2; ok && d >= 0; --d) {
        if (x.size(d) == 1) continue;
        if (step < 0) {
            step = x.stride(d);
            ok = step >= 0 && step % 8 == 0;
        } else {
            ok = x.stride(d) == want;
        }
        want = x.stride(d) * x.size(d);
    }
    if (!ok) {
        r = aligned16(x);
        step = C;
    }
    stride = step < 0 ? C : step;
    return r;
}

at::Tensor gated_groupnorm(const at::Tensor& x, const at::Tensor& z, const at::Tensor& weight,
                           int64_t groups, double eps, bool gate_first) {
    TORCH_CHECK(x.is_cuda(), "x must be on a HIP device (the ops have no CPU path)");
    on_device(z, x, "z");
    on_device(weight, x, "weight");
    const int io = io_dtype(x);
    TORCH_CHECK(z.scalar_type() == x.scalar_type() && z.sizes() == x.sizes(),
                "z must have the dtype and shape of x");
    TORCH_CHECK(x.dim() >= 1, "x must be [.., C]");
    const int64_t C = x.size(-1);
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == C &&
                    (weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat),
                "weight must be [C] in the dtype of x or fp32");
    TORCH_CHECK(groups >= 1 && C >= 8 && C <= 0x7fffffff && C % groups == 0 &&
                    (C / groups) % 8 == 0 && C / groups <= 16384,
                "groups must split C into multiples of 8 channels up to 16384");
    TORCH_CHECK(eps >= 0, "eps must not be negative");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    int64_t xs = C, zs = C;
    auto xr = as_rows(x, C, xs), zr = as_rows(z, C, zs);
    auto wc = aligned16(weight);
    auto y = at::empty(x.sizes(), x.options());
    check_hip(gdn_gated_groupnorm_forward(
                  xr.data_ptr(), xs, zr.data_ptr(), zs, wc.data_ptr(), y.data_ptr(), x.numel() / C,
                  (int)C, (int)groups, (float)eps, gate_first ? 1 : 0, io,
                  weight.scalar_type() == at::kFloat ? GDN_DTYPE_FP32 : io, current_stream()),
              "gdn_gated_groupnorm_forward");
    return y;
}

}  // namespace

void register_ssm_ops(pybind11::module_& m) {
    using namespace pybind11::literals;
    const double inf = std::numeric_limits<double>::infinity();
    m.def("ssm_scan", &ssm_scan,
          "selective state-space scan over prompts; returns [y, final_state]", "x"_a, "dt"_a,
          "A_log"_a, "B"_a, "C"_a, "D"_a = std::nullopt, "z"_a = std::nullopt,
          "dt_bias"_a = std::nullopt, "s0"_a = std::nullopt, pybind11::kw_only(),
          "cu_seqlens"_a = std::nullopt, "blocks"_a = std::nullopt, "block"_a = 0,
          "dt_min"_a = 0.0, "dt_max"_a = inf);
    m.def("ssm_scan_block", &ssm_scan_block,
          "the block of tokens ssm_scan works on at a time for these sizes", "tokens"_a,
          "batch"_a, "heads"_a, "head_dim"_a, "groups"_a, "state_dim"_a, "num_seqs"_a);
    m.def("ssm_step", &ssm_step,
          "selective state-space step (decode), state updated in place; returns y", "x"_a, "dt"_a,
          "A_log"_a, "B"_a, "C"_a, "state"_a, "D"_a = std::nullopt, "z"_a = std::nullopt,
          "dt_bias"_a = std::nullopt, pybind11::kw_only(), "slots"_a = std::nullopt,
          "dt_min"_a = 0.0, "dt_max"_a = inf);
    m.def("causal_conv1d_prefill", &causal_conv1d_prefill,
          "causal depthwise conv1d over x [B, D, T] that continues from state0; returns "
          "[y, state]",
          "x"_a, "weight"_a, "bias"_a = std::nullopt, "state0"_a = std::nullopt,
          pybind11::kw_only(), "silu"_a = false, "cu_seqlens"_a = std::nullopt, "state_len"_a = 0);
    m.def("request_blocks", &request_blocks,
          "tables of a packed batch from request lengths; returns [cu_seqlens, blocks, "
          "token_slots, token_pos]",
          "lengths"_a, "total_tokens"_a, pybind11::kw_only(), "block"_a = 64,
          "slots"_a = std::nullopt);
    m.def("gated_groupnorm", &gated_groupnorm,
          "gated norm over groups of the last dimension; returns y", "x"_a, "z"_a, "weight"_a,
          "groups"_a, "eps"_a = 1e-6, pybind11::kw_only(), "gate_first"_a = true);
}
