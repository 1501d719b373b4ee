// Test infrastructure: the entry points of include/ovl_ssm.h and include/ovl_norm.h behind the (inputs, outputs) calling
// convention of main.cpp in this directory, for host emulation of the hand-written kernels.  The first input is an int64
// array of settings, its first entry names the function; a tensor without elements stands for one that is absent.  The
// sequences' strides are among the settings, so padded layouts are tried too.
#include "ovl_device.h"
#include "ovl_norm.h"
#include "ovl_ssm.h"

namespace {
template <typename T = void> T* at(const ovl_tensor& t) { return t.len == 0 ? nullptr : static_cast<T*>(t.data); }

ovl_ssm_scan scan_of(const int64_t* s, const ovl_tensor* in) {
    ovl_ssm_scan p = {};
    p.batch = (uint32_t)s[1]; p.length = (uint32_t)s[2]; p.channels = (uint32_t)s[3]; p.state = (uint32_t)s[4];
    p.groups = (uint32_t)s[5]; p.dtype = (int32_t)s[6]; p.softplus = (int32_t)s[7];
    p.u = {at(in[1]), s[8], s[9]};
    p.delta = {at(in[2]), s[8], s[9]};
    p.z = {at(in[3]), s[8], s[9]};
    p.B = {at(in[4]), s[10], s[11], s[12]};
    p.C = {at(in[5]), s[10], s[11], s[12]};
    p.A = at<float>(in[6]);
    p.D = at<float>(in[7]);
    p.delta_bias = at<float>(in[8]);
    p.entering = at<float>(in[9]);
    p.lengths = at<int32_t>(in[10]);
    return p;
}

struct scratch {
    void* data = nullptr;
    uint64_t bytes;
    explicit scratch(uint64_t n) : bytes(n) { if (n > 0 && posix_memalign(&data, 16, n) != 0) abort(); if (n > 0) memset(data, 0xFE, n); }
    ~scratch() { free(data); }
};
}  // namespace

extern "C" int emu_recurrent_layer(const ovl_tensor* in, uint32_t n_in, ovl_tensor* out, uint32_t n_out, void* stream) {
    const int64_t* s = static_cast<const int64_t*>(in[0].data);
    int rc = OVL_EARGS;
    if (s[0] == 0 && n_in == 11 && n_out == 3) {
        const ovl_ssm_scan p = scan_of(s, in);
        scratch work(ovl_ssm_scan_workspace_bytes(&p, 0));
        rc = ovl_ssm_scan_forward(&p, at(out[0]), at<float>(out[1]), at<float>(out[2]), work.data, work.bytes, stream);
    } else if (s[0] == 1 && n_in == 13 && n_out == 9) {
        const ovl_ssm_scan p = scan_of(s, in);
        scratch saved(ovl_ssm_scan_saved_bytes(&p)), first(ovl_ssm_scan_workspace_bytes(&p, 0)), work(ovl_ssm_scan_workspace_bytes(&p, 1));
        rc = ovl_ssm_scan_forward(&p, nullptr, nullptr, static_cast<float*>(saved.data), first.data, first.bytes, stream);
        if (rc != 0) return rc;
        ovl_ssm_scan_gradients g = {};
        g.d_y = {at(in[11]), s[8], s[9]};
        g.d_last = at<float>(in[12]);
        g.d_u = at(out[0]); g.d_delta = at(out[1]); g.d_A = at<float>(out[2]); g.d_B = at(out[3]); g.d_C = at(out[4]);
        g.d_D = at<float>(out[5]); g.d_z = at(out[6]); g.d_delta_bias = at<float>(out[7]); g.d_entering = at<float>(out[8]);
        rc = ovl_ssm_scan_backward(&p, static_cast<const float*>(saved.data), &g, work.data, work.bytes, stream);
    } else if (s[0] == 2 && n_in == 11 && n_out == 2) {
        const ovl_ssm_scan p = scan_of(s, in);
        memcpy(out[1].data, in[9].data, out[1].len * sizeof(float));
        rc = ovl_ssm_scan_step(&p, at<float>(out[1]), (int64_t)p.channels * p.state, at(out[0]), stream);
    } else if (s[0] >= 3 && s[0] <= 5) {
        ovl_ssm_conv p = {};
        p.batch = (uint32_t)s[1]; p.length = (uint32_t)s[2]; p.channels = (uint32_t)s[3]; p.width = (uint32_t)s[4];
        p.dtype = (int32_t)s[5]; p.silu = (int32_t)s[6];
        const int64_t rows = (int64_t)p.width - 1;
        p.x = {at(in[1]), s[7], s[8]};
        p.weight = at<float>(in[2]);
        p.bias = at<float>(in[3]);
        p.own_weights = in[0].len > 9 ? (int32_t)s[9] : 0;
        p.kept = {at(in[4]), rows * p.channels, p.channels};
        p.lengths = at<int32_t>(in[5]);
        if (s[0] == 3) {
            rc = ovl_ssm_conv_forward(&p, at(out[0]), at(out[1]), stream);
        } else if (s[0] == 4) {
            scratch work(ovl_ssm_conv_workspace_bytes(&p));
            const ovl_ssm_sequence d_y = {at(in[6]), s[7], s[8]}, d_last = {at(in[7]), rows * p.channels, p.channels};
            rc = ovl_ssm_conv_backward(&p, &d_y, d_last.data != nullptr ? &d_last : nullptr, at(out[0]), at(out[3]), at<float>(out[1]),
                                       at<float>(out[2]), work.data, work.bytes, stream);
        } else {
            memcpy(out[1].data, in[4].data, out[1].len * (p.dtype == OVL_SSM_FLOAT32 ? 4 : 2));
            p.kept.data = at(out[1]);
            rc = ovl_ssm_conv_step(&p, at(out[0]), stream);
        }
    } else if (s[0] >= 6 && s[0] <= 8) {
        ovl_norm p = {};
        p.rows = (uint32_t)s[1]; p.columns = (uint32_t)s[2]; p.dtype = (int32_t)s[3]; p.residual_dtype = (int32_t)s[4];
        p.weight_dtype = (int32_t)s[5]; p.eps = s[0] == 7 && in[0].len > 9 ? 0.0f : 1e-5f;
        p.x = at(in[1]); p.x_stride = s[6];
        p.residual = at(in[2]); p.residual_stride = s[7];
        p.weight = at(in[3]);
        if (s[0] == 6) {
            rc = ovl_norm_forward(&p, at(out[0]), at(out[1]), stream);
        } else if (s[0] == 7) {
            rc = ovl_norm_forward_quantized(&p, (uint32_t)s[8], at(out[0]), at<float>(out[1]), at(out[2]), stream);
        } else {
            // in[2]: the gradient of y, in[4]: that of the sum
            p.residual = nullptr;
            scratch work(ovl_norm_workspace_bytes(&p));
            rc = ovl_norm_backward(&p, at(in[2]), s[7], at(in[4]), p.columns, at(out[0]), at(out[1]), at(out[2]), work.data, work.bytes, stream);
        }
    }
    if (rc != 0) fprintf(stderr, "%s %s\n", ovl_ssm_last_error(), ovl_norm_last_error());
    return rc;
}
