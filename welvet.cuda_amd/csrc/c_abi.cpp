// C ABI of the quantized Dense path (declarations in include/welvet_c.h).
// Status conversion and truncation follow src/interop/c_abi.cpp:41-47; no C++
// exception crosses the boundary.
#include "welvet_c.h"

#include <cstdio>
#include <cstdlib>
#include <cmath>
#include <cstring>
#include <memory>
#include <mutex>
#include <new>
#include <string>

#include "codec.h"
#include "kvcache.h"
#include "layers.h"
#include "model.h"
#include "runtime.h"
#include "sessions.h"

using wv::Status;

namespace {

welvet_status to_c(const Status& st) {
  welvet_status out{};
  out.code = st.code;
  std::strncpy(out.message, st.message.c_str(), sizeof(out.message) - 1);
  out.message[sizeof(out.message) - 1] = '\0';
  return out;
}

welvet_status invalid(const char* msg) { return to_c(Status::err(wv::kInvalid, msg)); }

template <class F>
welvet_status guarded(F&& fn) {
  try {
    return to_c(fn());
  } catch (const std::bad_alloc&) {
    return to_c(Status::err(wv::kInternal, "out of host memory"));
  } catch (const std::exception& e) {
    return to_c(Status::err(wv::kInternal, e.what()));
  } catch (...) {
    return to_c(Status::err(wv::kInternal, "unknown native failure"));
  }
}

welvet_status gap(const char* what) {
  return to_c(Status::err(wv::kGap, std::string("gap? ") + what +
                                        " is outside the quantized Dense path of this library"));
}

hipStream_t pick(void* stream, hipStream_t own) {
  return stream ? static_cast<hipStream_t>(stream) : own;
}

}  // namespace

struct welvet_swiglu_session {
  wv::HostSession host;
  wv::Stream stream;
  wv::SwiGLULayer layer;
  wv::Workspace ws;
  int rows = 0;
  wv::DevBuf x, pre, post;
};

struct welvet_mha_session {
  wv::HostSession host;
  wv::Stream stream;
  wv::MHALayer layer;
  wv::Workspace ws;
  int batch = 0, seq = 0;
  wv::DevBuf x, pre, post;
};

struct welvet_kv_session {
  wv::Stream stream;
  wv::KvCache cache;
};

extern "C" {

const char* welvet_version(void) { return "0.79"; }

const char* welvet_runtime_identity(void) {
  static thread_local std::string id;
  id = wv::identity();
  return id.c_str();
}

welvet_status welvet_cuda_init(void) { return to_c(wv::init_device()); }

int32_t welvet_cuda_available(void) { return wv::device_available() ? 1 : 0; }

// Ledger of this library: reference C entry points served on the GPU vs those
// returning code 3.
int32_t welvet_gaps_count(void) { return 41; }
int32_t welvet_gaps_done(void) { return 18; }

// Measurement extension: one streaming read of a device buffer.
welvet_status welvet_read_probe(const void* buf, size_t bytes, uint32_t* out_words,
                                size_t out_cap, void* stream) {
  if (!buf || !out_words) return invalid("read probe: null buffer");
  if (out_cap < wv::read_probe_words(bytes)) return invalid("read probe: output too small");
  return guarded([&]() -> Status {
    return wv::launch_read_probe(static_cast<const uint8_t*>(buf), bytes, out_words,
                                 static_cast<hipStream_t>(stream));
  });
}

size_t welvet_read_probe_words(size_t bytes) { return wv::read_probe_words(bytes); }

welvet_status welvet_fetch_probe(const void* buf, size_t region_bytes, int32_t iters,
                                 int32_t workgroups, uint32_t* out_words, size_t out_cap,
                                 void* stream) {
  if (!buf || !out_words) return invalid("fetch probe: null buffer");
  if (workgroups > 0 && out_cap < (size_t)workgroups) return invalid("fetch probe: output too small");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    return wv::launch_fetch_probe(static_cast<const uint8_t*>(buf), region_bytes, iters, workgroups,
                                  out_words, static_cast<hipStream_t>(stream));
  });
}

welvet_status welvet_mfma_probe(int32_t fmt_a, int32_t fmt_b, int32_t shape, int32_t iters,
                                int32_t workgroups, float* out, size_t out_cap, void* stream) {
  if (!out) return invalid("mfma probe: null output");
  if (workgroups > 0 && out_cap < (size_t)workgroups * 256) return invalid("mfma probe: output too small");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    return wv::launch_mfma_probe(fmt_a, fmt_b, shape, iters, workgroups, out,
                                 static_cast<hipStream_t>(stream));
  });
}

welvet_status welvet_clock_stamp(uint64_t* out, void* stream) {
  if (!out) return invalid("clock stamp: null output");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    return wv::launch_clock_stamp(out, static_cast<hipStream_t>(stream));
  });
}

int64_t welvet_clock_rate_khz(void) {
  if (!wv::init_device()) return 0;
  int khz = 0;
  if (hipDeviceGetAttribute(&khz, hipDeviceAttributeWallClockRate, 0) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return khz;
}

// ---------------------------------------------------------------- Dense ----
static welvet_status dense_mount(int32_t batch, int32_t in, int32_t out, int32_t act,
                                 int32_t dtype, int32_t backend, const float* W_init,
                                 const double* bias, size_t bias_len,
                                 welvet_dense_session** sess_out) {
  if (!sess_out) return invalid("null mount args");
  *sess_out = nullptr;
  if (!W_init) return invalid("null mount args");
  if (batch <= 0 || in <= 0 || out <= 0) return invalid("bad dims");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    auto* s = new welvet_dense_session();
    auto fail = [&](Status st) {
      delete s;
      return st;
    };
    Status st = s->stream.create();
    int scheme = 0, terms = wv::kTerms;
    if (st) st = wv::decode_backend(backend, &scheme, &terms);
    if (st) st = wv::dense_build(in, out, act, dtype, scheme, W_init, bias, bias_len, &s->layer,
                                 s->stream.s);
    s->layer.terms = terms;
    if (st && terms == 1 && batch > wv::kMxvMaxBatch && batch <= 32)
      st = Status::err(wv::kUnsupported, "one activation term needs a batch above 32 rows (or 1-4)");
    if (st) st = wv::dense_prepare_rows(&s->layer, batch, s->stream.s);
    if (st) st = wv::ensure_split(&s->ws, wv::dense_workspace_bytes(s->layer, batch));
    if (st) st = s->x.alloc((size_t)batch * in * sizeof(float));
    if (st) st = s->pre.alloc((size_t)batch * out * sizeof(float));
    if (st) st = s->post.alloc((size_t)batch * out * sizeof(float));
    if (!st) return fail(st);
    s->batch = batch;
    *sess_out = s;
    return Status::ok();
  });
}

welvet_status welvet_dense_mount(int32_t batch, int32_t in, int32_t out, int32_t act,
                                 int32_t dtype, const float* W_init, const double* bias,
                                 size_t bias_len, welvet_dense_session** sess_out) {
  return dense_mount(batch, in, out, act, dtype, 0, W_init, bias, bias_len, sess_out);
}

welvet_status welvet_dense_mount_q(int32_t batch, int32_t in, int32_t out, int32_t act,
                                   int32_t dtype, int32_t backend, const float* W_init,
                                   const double* bias, size_t bias_len,
                                   welvet_dense_session** sess_out) {
  return dense_mount(batch, in, out, act, dtype, backend, W_init, bias, bias_len, sess_out);
}

welvet_status welvet_dense_mount_format(int32_t batch, int32_t in, int32_t out, int32_t act,
                                        int32_t format, const float* W_init,
                                        const uint8_t* blocks, size_t blocks_len,
                                        const double* bias, size_t bias_len,
                                        welvet_dense_session** sess_out) {
  if (!sess_out) return invalid("null mount args");
  *sess_out = nullptr;
  if (batch <= 0 || in <= 0 || out <= 0) return invalid("bad dims");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    auto* s = new welvet_dense_session();
    Status st = s->stream.create();
    if (st) st = wv::dense_build_format(in, out, act, format, W_init, blocks, blocks_len, bias,
                                        bias_len, &s->layer, s->stream.s);
    if (st) st = wv::dense_prepare_rows(&s->layer, batch, s->stream.s);
    if (st) st = wv::ensure_split(&s->ws, wv::dense_workspace_bytes(s->layer, batch));
    if (st) st = s->x.alloc((size_t)batch * in * sizeof(float));
    if (st) st = s->pre.alloc((size_t)batch * out * sizeof(float));
    if (st) st = s->post.alloc((size_t)batch * out * sizeof(float));
    if (!st) {
      delete s;
      return st;
    }
    s->batch = batch;
    *sess_out = s;
    return Status::ok();
  });
}

welvet_status welvet_dense_export_blocks(welvet_dense_session* s, uint8_t* blocks, size_t cap,
                                         size_t* len) {
  if (!s) return invalid("null session");
  if (!s->layer.format) return to_c(Status::err(wv::kUnsupported, "not a packed block format session"));
  const std::vector<uint8_t>& b = s->layer.fw.blocks;
  if (len) *len = b.size();
  if (blocks) {
    if (cap < b.size()) return invalid("block buffer too small");
    std::memcpy(blocks, b.data(), b.size());
  }
  return to_c(Status::ok());
}

welvet_status welvet_dense_export_f32(welvet_dense_session* s, float* W) {
  if (!s || !W) return invalid("null export args");
  return guarded([&]() -> Status {
    const size_t n = (size_t)s->layer.in * s->layer.out;
    wv::DevBuf w;
    WV_TRY(w.alloc(n * sizeof(float)));
    WV_TRY(wv::dense_export_f32(s->layer, w.as<float>(), s->stream.s));
    WV_TRY(wv::copy_d2h(W, w.p, n * sizeof(float), s->stream.s));
    WV_HIP(hipStreamSynchronize(s->stream.s));
    return Status::ok();
  });
}

welvet_status welvet_dense_execute(welvet_dense_session* s, const float* x, float* pre,
                                   float* post) {
  if (!s || !x || !pre || !post) return invalid("null execute args");
  return guarded([&]() -> Status {
    const size_t xb = (size_t)s->batch * s->layer.in * sizeof(float);
    const size_t yb = (size_t)s->batch * s->layer.out * sizeof(float);
    hipStream_t st = s->stream.s;
    return wv::host_call(x, s->x.p, xb, pre, s->pre.p, yb, post, s->post.p, yb, st, [&] {
      return wv::dense_forward(s->layer, s->batch, s->x.as<float>(), s->pre.as<float>(),
                               s->post.as<float>(), &s->ws, st);
    });
  });
}

welvet_status welvet_dense_execute_device(welvet_dense_session* s, const float* x, float* pre,
                                          float* post, void* stream) {
  if (!s || !x || !pre || !post) return invalid("null execute args");
  if (pre == post && s->layer.need_epi()) return invalid("pre and post must differ");
  return guarded([&]() -> Status {
    return wv::dense_forward(s->layer, s->batch, x, pre, post, &s->ws, pick(stream, s->stream.s));
  });
}

welvet_status welvet_dense_backward_device(welvet_dense_session* s, const float* x,
                                           const float* pre, const float* post, const float* g,
                                           int32_t use_target, float* dpre, float* dX, float* dW,
                                           double* loss_part, void* stream) {
  if (!s || !x || !pre || !g || !dpre || !dX || !dW || (use_target && (!post || !loss_part)))
    return invalid("null backward args");
  return guarded([&]() -> Status {
    return wv::dense_backward(s->layer, s->batch, x, pre, post, g, use_target != 0, dpre, dX, dW,
                              loss_part, &s->ws, pick(stream, s->stream.s));
  });
}

// ---- grouped Dense execution (extension) ----
struct welvet_dense_group {
  wv::Stream stream;
  std::vector<welvet_dense_session*> members;
  std::vector<const float*> x;
  std::vector<float*> pre, post;
  bool fused = false;
  wv::DenseGroup g;
};

welvet_status welvet_dense_group_mount(welvet_dense_session* const* sessions, int32_t n,
                                       const float* const* x, float* const* pre,
                                       float* const* post, welvet_dense_group** out) {
  if (!out) return invalid("null group out");
  *out = nullptr;
  if (n <= 0 || !sessions || !x || !pre || !post) return invalid("group: null or empty arguments");
  return guarded([&]() -> Status {
    auto grp = std::make_unique<welvet_dense_group>();
    for (int i = 0; i < n; ++i) {
      welvet_dense_session* s = sessions[i];
      if (!s) return wv::Status::err(wv::kInvalid, "group: null session");
      if (s->batch != sessions[0]->batch)
        return wv::Status::err(wv::kInvalid, "group: sessions differ in batch");
      if (!x[i] || !pre[i] || !post[i]) return wv::Status::err(wv::kInvalid, "group: null buffer");
      if (pre[i] == post[i] && s->layer.need_epi())
        return wv::Status::err(wv::kInvalid, "group: pre and post must differ");
      grp->members.push_back(s);
      grp->x.push_back(x[i]);
      grp->pre.push_back(pre[i]);
      grp->post.push_back(post[i]);
    }
    const int batch = sessions[0]->batch;
    WV_TRY(grp->stream.create());
    grp->fused = wv::dense_group_fused(batch);
    if (grp->fused) {
      std::vector<const wv::DenseLayer*> layers;
      for (auto* s : grp->members) layers.push_back(&s->layer);
      WV_TRY(wv::dense_group_build(layers.data(), n, batch, grp->x.data(), grp->pre.data(),
                                   grp->post.data(), &grp->g));
    }
    *out = grp.release();
    return Status::ok();
  });
}

welvet_status welvet_dense_group_execute(welvet_dense_group* g, void* stream) {
  if (!g) return invalid("null group");
  return guarded([&]() -> Status {
    hipStream_t st = pick(stream, g->stream.s);
    if (g->fused) return wv::dense_group_forward(g->g, st);
    for (size_t i = 0; i < g->members.size(); ++i) {
      welvet_dense_session* s = g->members[i];
      WV_TRY(wv::dense_forward(s->layer, s->batch, g->x[i], g->pre[i], g->post[i], &s->ws, st));
    }
    return Status::ok();
  });
}

void welvet_dense_group_release(welvet_dense_group* g) { delete g; }

// ---- chained groups (extension) ----
struct welvet_dense_chain {
  wv::Stream stream;
  std::vector<welvet_dense_group*> groups;
  bool fused = false;
  wv::DenseChain c;
};

welvet_status welvet_dense_chain_mount(welvet_dense_group* const* groups, int32_t n,
                                       welvet_dense_chain** out) {
  return welvet_dense_chain_mount_ex(groups, n, 0, out);
}

welvet_status welvet_dense_chain_mount_ex(welvet_dense_group* const* groups, int32_t n,
                                          int32_t flags, welvet_dense_chain** out) {
  if (!out) return invalid("null chain out");
  *out = nullptr;
  if (n <= 0 || !groups) return invalid("chain: null or empty arguments");
  if (flags & ~WELVET_CHAIN_INNER_NOT_KEPT) return invalid("chain: unknown flags");
  return guarded([&]() -> Status {
    auto ch = std::make_unique<welvet_dense_chain>();
    bool fused = true;
    for (int k = 0; k < n; ++k) {
      welvet_dense_group* g = groups[k];
      if (!g) return wv::Status::err(wv::kInvalid, "chain: null group");
      if (k > 0) {
        const welvet_dense_group* p = groups[k - 1];
        if (g->members.size() != p->members.size() ||
            g->members[0]->batch != p->members[0]->batch)
          return wv::Status::err(wv::kInvalid, "chain: groups differ in members or batch");
        for (size_t i = 0; i < g->members.size(); ++i)
          if (g->members[i]->layer.in != p->members[i]->layer.out ||
              (g->x[i] != p->post[i] && g->x[i] != p->pre[i]) ||
              (g->x[i] == p->pre[i] && g->x[i] != p->post[i] && p->members[i]->layer.need_epi()))
            return wv::Status::err(wv::kInvalid,
                                   "chain: member input is not the previous member's output");
      }
      fused = fused && g->fused;
      ch->groups.push_back(g);
    }
    WV_TRY(ch->stream.create());
    ch->fused = fused;
    if (fused) {
      std::vector<const wv::DenseGroup*> gs;
      for (auto* g : ch->groups) gs.push_back(&g->g);
      WV_TRY(wv::dense_chain_build(gs.data(), n, &ch->c,
                                   (flags & WELVET_CHAIN_INNER_NOT_KEPT) == 0));
    }
    *out = ch.release();
    return Status::ok();
  });
}

welvet_status welvet_dense_chain_execute(welvet_dense_chain* c, void* stream) {
  if (!c) return invalid("null chain");
  hipStream_t st = pick(stream, c->stream.s);
  if (c->fused) return guarded([&]() -> Status { return wv::dense_chain_forward(c->c, st); });
  for (auto* g : c->groups) {
    welvet_status r = welvet_dense_group_execute(g, st);
    if (r.code != 0) return r;
  }
  return to_c(Status::ok());
}

void welvet_dense_chain_release(welvet_dense_chain* c) { delete c; }

welvet_status welvet_dense_export_store(welvet_dense_session* s, uint8_t* native,
                                        size_t native_cap, size_t* native_len, float* row_scale,
                                        uint8_t* blk_exp, float* tensor_scale) {
  if (!s) return invalid("null session");
  if (s->layer.format)
    return to_c(Status::err(wv::kUnsupported, "packed block format session: use "
                                              "welvet_dense_export_blocks"));
  const wv::WeightStore& w = s->layer.store;
  if (native_len) *native_len = w.native.size();
  if (native) {
    if (native_cap < w.native.size()) return invalid("native buffer too small");
    std::memcpy(native, w.native.data(), w.native.size());
  }
  if (row_scale) std::memcpy(row_scale, w.row_scale.data(), w.row_scale.size() * sizeof(float));
  if (blk_exp && !w.blk_exp.empty()) std::memcpy(blk_exp, w.blk_exp.data(), w.blk_exp.size());
  if (tensor_scale) *tensor_scale = w.scale;
  return to_c(Status::ok());
}

void welvet_dense_release(welvet_dense_session* s) { delete s; }

welvet_status welvet_dense_forward_f32(int32_t batch, int32_t in, int32_t out, int32_t act,
                                       int32_t dtype, int32_t backend, const float* W_init,
                                       const double* bias, size_t bias_len, const float* x,
                                       float* pre, float* post) {
  if (batch <= 0 || in <= 0 || out <= 0 || !x || !pre || !post) return invalid("bad dims");
  welvet_dense_session* s = nullptr;
  std::vector<float> zeros;
  if (!W_init) {
    zeros.assign((size_t)in * out, 0.0f);
    W_init = zeros.data();
  }
  welvet_status st = dense_mount(batch, in, out, act, dtype, backend, W_init, bias, bias_len, &s);
  if (st.code != 0) return st;
  st = welvet_dense_execute(s, x, pre, post);
  welvet_dense_release(s);
  return st;
}

// Dense NormalBP leaf (src/interop/c_abi.cpp:119-200): forward, gradient
// (the caller's, or MSE from a target), backward over the quantized weights,
// optional SGD on the quantized store, then the updated weights as f32. The
// scale scheme comes in `backend` as for the other entry points.
welvet_status welvet_dense_normalbp_f32(int32_t batch, int32_t in, int32_t out, int32_t act,
                                        int32_t dtype, int32_t backend, const float* W_init,
                                        const double* bias, size_t bias_len, const float* x,
                                        const float* grad_or_target, int32_t use_target, double lr,
                                        float* pre, float* post, float* dX, float* dW,
                                        float* W_after, double* loss) {
  if (batch <= 0 || in <= 0 || out <= 0 || !W_init || !x || !grad_or_target || !pre || !post ||
      !dX || !dW || !W_after || !loss)
    return invalid("invalid argument");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    wv::Stream stream;
    WV_TRY(stream.create());
    hipStream_t st = stream.s;
    wv::DenseLayer L;
    wv::Workspace ws;
    int scheme = 0, terms = wv::kTerms;
    WV_TRY(wv::decode_backend(backend, &scheme, &terms));
    WV_TRY(wv::dense_build(in, out, act, dtype, scheme, W_init, bias, bias_len, &L, st));
    L.terms = terms;
    const size_t nx = (size_t)batch * in, ny = (size_t)batch * out, nw = (size_t)in * out;
    const int64_t parts = wv::dpre_blocks((int64_t)ny);
    wv::DevBuf dx_in, dpre_out, dpost, dg, dd, ddx, ddw, dwa, dloss;
    WV_TRY(dx_in.alloc(nx * sizeof(float)));
    WV_TRY(dpre_out.alloc(ny * sizeof(float)));
    WV_TRY(dpost.alloc(ny * sizeof(float)));
    WV_TRY(dg.alloc(ny * sizeof(float)));
    WV_TRY(dd.alloc(ny * sizeof(float)));
    WV_TRY(ddx.alloc(nx * sizeof(float)));
    WV_TRY(ddw.alloc(nw * sizeof(float)));
    WV_TRY(dwa.alloc(nw * sizeof(float)));
    WV_TRY(dloss.alloc((size_t)parts * sizeof(double)));
    WV_TRY(wv::copy_h2d(dx_in.p, x, nx * sizeof(float), st));
    WV_TRY(wv::copy_h2d(dg.p, grad_or_target, ny * sizeof(float), st));
    WV_TRY(wv::ensure_split(&ws, wv::dense_workspace_bytes(L, batch)));
    WV_TRY(wv::dense_forward(L, batch, dx_in.as<float>(), dpre_out.as<float>(), dpost.as<float>(),
                             &ws, st));
    WV_TRY(wv::dense_backward(L, batch, dx_in.as<float>(), dpre_out.as<float>(), dpost.as<float>(),
                              dg.as<float>(), use_target != 0, dd.as<float>(), ddx.as<float>(),
                              ddw.as<float>(), dloss.as<double>(), &ws, st));
    if (lr != 0.0) WV_TRY(wv::dense_apply_sgd(&L, ddw.as<float>(), lr, st));
    WV_TRY(wv::launch_dequant(L.dev, dwa.as<float>(), st));
    std::vector<double> lp(use_target ? (size_t)parts : 0);
    WV_TRY(wv::copy_d2h(pre, dpre_out.p, ny * sizeof(float), st));
    WV_TRY(wv::copy_d2h(post, dpost.p, ny * sizeof(float), st));
    WV_TRY(wv::copy_d2h(dX, ddx.p, nx * sizeof(float), st));
    WV_TRY(wv::copy_d2h(dW, ddw.p, nw * sizeof(float), st));
    WV_TRY(wv::copy_d2h(W_after, dwa.p, nw * sizeof(float), st));
    if (use_target)
      WV_TRY(wv::copy_d2h(lp.data(), dloss.p, lp.size() * sizeof(double), st));
    WV_HIP(hipStreamSynchronize(st));
    double sum = 0.0;
    for (double v : lp) sum += v;
    *loss = use_target ? sum / (double)ny : 0.0;
    return Status::ok();
  });
}

// SwiGLU NormalBP leaf (src/interop/c_abi.cpp:581-652): forward (pre = h,
// post = y), the gradient (gradOut or MSE from a target), the backward over
// the three quantized matrices, optional SGD on each store, then the
// updated weights as f32 [Gate | Up | Down]. Scale scheme in `backend`.
welvet_status welvet_swiglu_normalbp_f32(int32_t batch, int32_t seq, int32_t input_dim,
                                         int32_t intermediate_dim, int32_t dtype, int32_t backend,
                                         const float* Gate, const float* Up, const float* Down,
                                         const float* x, const float* grad_or_target,
                                         int32_t use_target, double lr, float* pre, float* post,
                                         float* dX, float* dW, float* W_after, double* loss) {
  if (batch <= 0 || seq <= 0 || input_dim <= 0 || intermediate_dim <= 0 || !Gate || !Up || !Down ||
      !x || !grad_or_target || !pre || !post || !dX || !dW || !W_after || !loss)
    return invalid("swiglu nbp: invalid argument");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    wv::Stream stream;
    WV_TRY(stream.create());
    hipStream_t st = stream.s;
    wv::SwiGLULayer L;
    wv::Workspace ws;
    int scheme = 0, terms = wv::kTerms;
    WV_TRY(wv::decode_backend(backend, &scheme, &terms));
    if (terms != wv::kTerms)
      return Status::err(wv::kUnsupported, "swiglu: two activation terms are for Dense layers");
    WV_TRY(wv::swiglu_build(input_dim, intermediate_dim, dtype, scheme, Gate, Up, Down, &L, st));
    const int rows = batch * seq;
    const size_t nx = (size_t)rows * input_dim, nh = (size_t)rows * intermediate_dim;
    const size_t wf = (size_t)intermediate_dim * input_dim, nw = 3 * wf;
    const int64_t parts = wv::dpre_blocks((int64_t)nx);
    wv::DevBuf dx_in, dh, dy, dg, ddx, ddw, dwa, dloss;
    WV_TRY(dx_in.alloc(nx * sizeof(float)));
    WV_TRY(dh.alloc(nh * sizeof(float)));
    WV_TRY(dy.alloc(nx * sizeof(float)));
    WV_TRY(dg.alloc(nx * sizeof(float)));
    WV_TRY(ddx.alloc(nx * sizeof(float)));
    WV_TRY(ddw.alloc(nw * sizeof(float)));
    WV_TRY(dwa.alloc(nw * sizeof(float)));
    WV_TRY(dloss.alloc((size_t)parts * sizeof(double)));
    WV_TRY(wv::copy_h2d(dx_in.p, x, nx * sizeof(float), st));
    WV_TRY(wv::copy_h2d(dg.p, grad_or_target, nx * sizeof(float), st));
    WV_TRY(wv::ensure_split(&ws, wv::swiglu_workspace_bytes(L, rows)));
    WV_TRY(wv::swiglu_forward(L, rows, dx_in.as<float>(), dh.as<float>(), dy.as<float>(), &ws, st));
    WV_TRY(wv::swiglu_backward(L, rows, dx_in.as<float>(), dh.as<float>(), dy.as<float>(),
                               dg.as<float>(), use_target != 0, ddx.as<float>(), ddw.as<float>(),
                               dloss.as<double>(), &ws, st));
    if (lr != 0.0) WV_TRY(wv::swiglu_apply_sgd(&L, ddw.as<float>(), lr, st));
    WV_TRY(wv::launch_dequant(L.gate.dev, dwa.as<float>(), st));
    WV_TRY(wv::launch_dequant(L.up.dev, dwa.as<float>() + wf, st));
    WV_TRY(wv::launch_dequant(L.down.dev, dwa.as<float>() + 2 * wf, st));
    std::vector<double> lp(use_target ? (size_t)parts : 0);
    WV_TRY(wv::copy_d2h(pre, dh.p, nh * sizeof(float), st));
    WV_TRY(wv::copy_d2h(post, dy.p, nx * sizeof(float), st));
    WV_TRY(wv::copy_d2h(dX, ddx.p, nx * sizeof(float), st));
    WV_TRY(wv::copy_d2h(dW, ddw.p, nw * sizeof(float), st));
    WV_TRY(wv::copy_d2h(W_after, dwa.p, nw * sizeof(float), st));
    if (use_target)
      WV_TRY(wv::copy_d2h(lp.data(), dloss.p, lp.size() * sizeof(double), st));
    WV_HIP(hipStreamSynchronize(st));
    double sum = 0.0;
    for (double v : lp) sum += v;
    *loss = use_target ? sum / (double)nx : 0.0;
    return Status::ok();
  });
}

// --------------------------------------------------------------- SwiGLU ----// --------------------------------------------------------------- SwiGLU ----
welvet_status welvet_swiglu_mount(int32_t batch, int32_t seq, int32_t input_dim,
                                  int32_t intermediate_dim, int32_t dtype, int32_t backend,
                                  const float* Gate, const float* Up, const float* Down,
                                  welvet_swiglu_session** out) {
  if (!out) return invalid("swiglu: invalid argument");
  *out = nullptr;
  if (batch <= 0 || seq <= 0 || input_dim <= 0 || intermediate_dim <= 0 || !Gate || !Up || !Down)
    return invalid("swiglu: invalid argument");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    auto* s = new welvet_swiglu_session();
    const int rows = batch * seq;
    Status st = s->stream.create();
    int scheme = 0, terms = wv::kTerms;
    if (st) st = wv::decode_backend(backend, &scheme, &terms);
    if (st && terms != wv::kTerms)
      st = Status::err(wv::kUnsupported, "swiglu: two activation terms are for Dense layers");
    if (st) st = wv::swiglu_build(input_dim, intermediate_dim, dtype, scheme, Gate, Up, Down,
                                  &s->layer, s->stream.s);
    if (st) st = wv::swiglu_prepare_rows(&s->layer, rows, s->stream.s);
    if (st) st = wv::ensure_split(&s->ws, wv::swiglu_workspace_bytes(s->layer, rows));
    if (st) st = s->x.alloc((size_t)rows * input_dim * sizeof(float));
    if (st) st = s->pre.alloc((size_t)rows * intermediate_dim * sizeof(float));
    if (st) st = s->post.alloc((size_t)rows * input_dim * sizeof(float));
    if (!st) {
      delete s;
      return st;
    }
    s->rows = rows;
    *out = s;
    return Status::ok();
  });
}

welvet_status welvet_swiglu_execute(welvet_swiglu_session* s, const float* x, float* pre,
                                    float* post) {
  if (!s || !x || !pre || !post) return invalid("swiglu: invalid argument");
  return guarded([&]() -> Status {
    const size_t xb = (size_t)s->rows * s->layer.in * sizeof(float);
    const size_t hb = (size_t)s->rows * s->layer.inter * sizeof(float);
    hipStream_t st = s->stream.s;
    return wv::host_call(x, s->x.p, xb, pre, s->pre.p, hb, post, s->post.p, xb, st, [&] {
      return wv::swiglu_forward(s->layer, s->rows, s->x.as<float>(), s->pre.as<float>(),
                                s->post.as<float>(), &s->ws, st);
    });
  });
}

welvet_status welvet_swiglu_execute_device(welvet_swiglu_session* s, const float* x, float* pre,
                                           float* post, void* stream) {
  if (!s || !x || !pre || !post) return invalid("swiglu: invalid argument");
  return guarded([&]() -> Status {
    return wv::swiglu_forward(s->layer, s->rows, x, pre, post, &s->ws, pick(stream, s->stream.s));
  });
}

void welvet_swiglu_release(welvet_swiglu_session* s) { delete s; }

welvet_status welvet_swiglu_forward_f32(int32_t batch, int32_t seq, int32_t input_dim,
                                        int32_t intermediate_dim, int32_t dtype, int32_t backend,
                                        const float* Gate, const float* Up, const float* Down,
                                        const float* x, float* pre, float* post) {
  if (batch <= 0 || seq <= 0 || input_dim <= 0 || intermediate_dim <= 0 || !Gate || !Up || !Down ||
      !x || !pre || !post)
    return invalid("swiglu: invalid argument");
  welvet_swiglu_session* s = nullptr;
  welvet_status st = welvet_swiglu_mount(batch, seq, input_dim, intermediate_dim, dtype, backend,
                                         Gate, Up, Down, &s);
  if (st.code != 0) return st;
  st = welvet_swiglu_execute(s, x, pre, post);
  welvet_swiglu_release(s);
  return st;
}

// ------------------------------------------------------------------ MHA ----
welvet_status welvet_mha_mount(int32_t batch, int32_t seq, int32_t d_model, int32_t num_heads,
                               int32_t num_kv_heads, int32_t head_dim, int32_t max_seq_len,
                               int32_t mask, int32_t pos, int32_t dtype, int32_t backend,
                               const float* Q, const float* K, const float* V, const float* O,
                               welvet_mha_session** out) {
  if (!out) return invalid("mha: invalid argument");
  *out = nullptr;
  if (batch <= 0 || seq <= 0 || d_model <= 0 || num_heads <= 0 || !Q || !K || !V || !O)
    return invalid("mha: invalid argument");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    wv::MHAConfig cfg;
    cfg.d_model = d_model;
    cfg.num_heads = num_heads;
    cfg.num_kv_heads = num_kv_heads;
    cfg.head_dim = head_dim;
    cfg.max_seq_len = max_seq_len;
    cfg.mask = mask;
    cfg.pos = pos;
    WV_TRY(wv::mha_validate(&cfg));
    if (seq > cfg.max_seq_len) return Status::err(wv::kInvalid, "mha: seq > MaxSeqLen");
    auto* s = new welvet_mha_session();
    const size_t T = (size_t)batch * seq;
    Status st = s->stream.create();
    int scheme = 0, terms = wv::kTerms;
    if (st) st = wv::decode_backend(backend, &scheme, &terms);
    // two-term projections leave the attention output at ~1e-3 rel-L2 (the
    // softmax amplifies the Q/K error): outside the layer bound
    if (st && terms != wv::kTerms)
      st = Status::err(wv::kUnsupported, "mha: two activation terms are for Dense layers");
    if (st) st = wv::mha_build(cfg, dtype, scheme, Q, K, V, O, &s->layer, s->stream.s);
    if (st) st = wv::mha_prepare_rows(&s->layer, batch * seq, s->stream.s);
    if (st) st = wv::mha_prepare(s->layer, batch, seq, &s->ws);
    if (st) st = s->x.alloc(T * d_model * sizeof(float));
    if (st) st = s->pre.alloc(T * cfg.q_dim() * sizeof(float));
    if (st) st = s->post.alloc(T * d_model * sizeof(float));
    if (!st) {
      delete s;
      return st;
    }
    s->batch = batch;
    s->seq = seq;
    *out = s;
    return Status::ok();
  });
}

welvet_status welvet_mha_execute(welvet_mha_session* s, const float* x, float* pre, float* post) {
  if (!s || !x || !pre || !post) return invalid("mha: invalid argument");
  return guarded([&]() -> Status {
    const size_t T = (size_t)s->batch * s->seq;
    const size_t xb = T * s->layer.cfg.d_model * sizeof(float);
    const size_t ab = T * s->layer.cfg.q_dim() * sizeof(float);
    hipStream_t st = s->stream.s;
    return wv::host_call(x, s->x.p, xb, pre, s->pre.p, ab, post, s->post.p, xb, st, [&] {
      return wv::mha_forward(s->layer, s->batch, s->seq, s->x.as<float>(), s->pre.as<float>(),
                             s->post.as<float>(), &s->ws, st);
    });
  });
}

welvet_status welvet_mha_execute_device(welvet_mha_session* s, const float* x, float* pre,
                                        float* post, void* stream) {
  if (!s || !x || !pre || !post) return invalid("mha: invalid argument");
  return guarded([&]() -> Status {
    return wv::mha_forward(s->layer, s->batch, s->seq, x, pre, post, &s->ws,
                           pick(stream, s->stream.s));
  });
}

void welvet_mha_release(welvet_mha_session* s) { delete s; }

welvet_status welvet_mha_forward_f32(int32_t batch, int32_t seq, int32_t d_model,
                                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                     int32_t max_seq_len, int32_t mask, int32_t pos, int32_t dtype,
                                     int32_t backend, const float* Q, const float* K,
                                     const float* V, const float* O, const float* x, float* pre,
                                     float* post) {
  if (!x || !pre || !post) return invalid("mha: invalid argument");
  welvet_mha_session* s = nullptr;
  welvet_status st = welvet_mha_mount(batch, seq, d_model, num_heads, num_kv_heads, head_dim,
                                      max_seq_len, mask, pos, dtype, backend, Q, K, V, O, &s);
  if (st.code != 0) return st;
  st = welvet_mha_execute(s, x, pre, post);
  welvet_mha_release(s);
  return st;
}

// ------------------------------------------------------------ K/V cache ----
welvet_status welvet_kv_mount(int32_t dtype, int32_t num_pages, int32_t page_tokens,
                              int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                              int32_t max_seqs, int32_t max_pages, int32_t flags,
                              welvet_kv_session** out) {
  if (!out) return invalid("kv: null mount args");
  *out = nullptr;
  if (num_pages <= 0 || page_tokens <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      max_seqs <= 0 || max_pages <= 0)
    return invalid("kv: bad dims");
  if (flags & ~WELVET_KV_TRACK) return invalid("kv: unknown flags");
  if (page_tokens % wv::kKvGroup != 0) return invalid("kv: page_tokens must be a multiple of 16");
  if (num_heads % num_kv_heads != 0)
    return invalid("kv: num_heads must be a multiple of num_kv_heads");
  if (dtype != wv::kKvF32 && dtype != wv::kKvBF16 && dtype != wv::kKvE4M3)
    return to_c(Status::err(wv::kUnsupported, "kv: dtype must be Float32, BFloat16 or FP8E4M3"));
  if (head_dim > wv::kKvMaxHd)
    return to_c(Status::err(wv::kUnsupported, "kv: head_dim above 256"));
  if ((int64_t)max_pages * page_tokens > (1 << 30)) return invalid("kv: capacity above 2^30");
  // (the rows of the pool and the scores of the running sums, counted so that
  // no product of their sizes leaves 64 bits)
  constexpr double kMost = 1e13;
  if ((double)num_pages * page_tokens * num_kv_heads > kMost ||
      ((flags & WELVET_KV_TRACK) && (double)max_seqs * max_pages * page_tokens * num_heads > kMost))
    return invalid("kv: too many pages, heads or sequences");
  if (max_seqs > 65535 || num_heads > 65535) return invalid("kv: more than 65535 sequences or heads");
  // (the attention cuts all sequences' tiles of 16 entries and more into shares,
  // which are counted as int)
  const int shares = wv::kv_target(num_kv_heads * wv::kv_chunks(num_heads / num_kv_heads), head_dim);
  if ((double)max_seqs * ((double)max_pages * page_tokens / 16 + 17) / shares > (1 << 30))
    return invalid("kv: max_seqs times capacity too large");
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    auto s = std::make_unique<welvet_kv_session>();
    WV_TRY(s->stream.create());
    WV_TRY(wv::kv_build(dtype, num_pages, page_tokens, num_heads, num_kv_heads, head_dim, max_seqs,
                        max_pages, (flags & WELVET_KV_TRACK) != 0, &s->cache, s->stream.s));
    *out = s.release();
    return Status::ok();
  });
}

void welvet_kv_release(welvet_kv_session* s) { delete s; }

welvet_status welvet_kv_get_buffers(welvet_kv_session* s, welvet_kv_buffers* out) {
  if (!s || !out) return invalid("kv: null buffers args");
  const wv::KvPool& p = s->cache.pool;
  *out = welvet_kv_buffers{p.k, p.v, p.ks, p.vs, p.pitch};
  return to_c(Status::ok());
}

// The sequences of a call in the kernels' form, checked against the session.
static Status kv_seqs(const welvet_kv_session* s, const welvet_kv_seqs* q, wv::KvSeqs* out) {
  if (!s || !q) return Status::err(wv::kInvalid, "kv: null session or sequences");
  if (q->nseq < 0 || q->nseq > s->cache.max_seqs)
    return Status::err(wv::kInvalid, "kv: nseq outside the mounted number of sequences");
  if (!q->table || !q->lens) return Status::err(wv::kInvalid, "kv: null table or lens");
  if (((uintptr_t)q->pos | (uintptr_t)q->weight) % 16 != 0)
    return Status::err(wv::kInvalid, "kv: pos and weight must be 16-byte aligned");
  out->nseq = q->nseq, out->table = q->table, out->lens = q->lens, out->next_pos = q->next_pos;
  out->pos = q->pos, out->weight = q->weight;
  return Status::ok();
}

// A row stride: 0 stands for rows that follow each other.
static bool kv_stride(int64_t given, int64_t width, int64_t* out) {
  *out = given == 0 ? width : given;
  return *out >= width;
}

welvet_status welvet_kv_append_device(welvet_kv_session* s, const welvet_kv_seqs* seqs,
                                      int32_t rows, const int32_t* counts, const float* k,
                                      int64_t k_stride, const float* v, int64_t v_stride,
                                      void* stream) {
  return guarded([&]() -> Status {
    wv::KvSeqs q;
    WV_TRY(kv_seqs(s, seqs, &q));
    const wv::KvPool& p = s->cache.pool;
    if (rows < 0 || rows > p.capacity()) return Status::err(wv::kInvalid, "kv append: bad rows");
    if (!k || !v) return Status::err(wv::kInvalid, "kv append: null rows");
    wv::KvRows r;
    const int64_t width = (int64_t)p.kv_heads * p.hd;
    if (!kv_stride(k_stride, width, &r.k_stride) || !kv_stride(v_stride, width, &r.v_stride))
      return Status::err(wv::kInvalid, "kv append: stride shorter than a row");
    r.rows = rows, r.counts = counts, r.k = k, r.v = v;
    return wv::launch_kv_append(p, q, r, pick(stream, s->stream.s));
  });
}

welvet_status welvet_kv_read_device(welvet_kv_session* s, const welvet_kv_seqs* seqs, int32_t count,
                                    const int32_t* first, const int32_t* counts, float* k, float* v,
                                    void* stream) {
  return guarded([&]() -> Status {
    wv::KvSeqs q;
    WV_TRY(kv_seqs(s, seqs, &q));
    if (count < 0 || count > s->cache.pool.capacity())
      return Status::err(wv::kInvalid, "kv read: bad count");
    if (!k || !v) return Status::err(wv::kInvalid, "kv read: null output");
    return wv::launch_kv_read(s->cache.pool, q, count, first, counts, k, v,
                              pick(stream, s->stream.s));
  });
}

welvet_status welvet_kv_attend_device(welvet_kv_session* s, const welvet_kv_seqs* seqs,
                                      int32_t tail, const float* q, int64_t q_stride, double scale,
                                      int32_t window, int32_t alibi, float* out,
                                      int64_t out_stride, float* lse, void* stream) {
  return guarded([&]() -> Status {
    wv::KvSeqs sq;
    WV_TRY(kv_seqs(s, seqs, &sq));
    const wv::KvPool& p = s->cache.pool;
    if (!q || !out) return Status::err(wv::kInvalid, "kv attend: null q or out");
    if (tail < 0 || tail > p.capacity()) return Status::err(wv::kInvalid, "kv attend: bad tail");
    if (window < 0) return Status::err(wv::kInvalid, "kv attend: negative window");
    if (!(scale >= 0.0) || scale > 2.0e38) return Status::err(wv::kInvalid, "kv attend: bad scale");
    if (sq.weight && !s->cache.track)
      return Status::err(wv::kInvalid, "kv attend: running sums need a session mounted with WELVET_KV_TRACK");
    wv::KvAttend a;
    const int64_t width = (int64_t)p.heads * p.hd;
    if (!kv_stride(q_stride, width, &a.q_stride) || !kv_stride(out_stride, width, &a.out_stride))
      return Status::err(wv::kInvalid, "kv attend: stride shorter than a row");
    a.q = q, a.out = out, a.lse = lse, a.tail = tail, a.window = window, a.alibi = alibi ? 1 : 0;
    a.scale2 = (float)((scale == 0.0 ? 1.0 / std::sqrt((double)p.hd) : scale) * 1.4426950408889634);
    return wv::kv_attend(s->cache, sq, a, pick(stream, s->stream.s));
  });
}

welvet_status welvet_kv_choose_device(welvet_kv_session* s, const welvet_kv_seqs* seqs,
                                      int32_t budget, int32_t sinks, int32_t recent, int32_t* src,
                                      void* stream) {
  return guarded([&]() -> Status {
    wv::KvSeqs q;
    WV_TRY(kv_seqs(s, seqs, &q));
    if (!q.weight || !src) return Status::err(wv::kInvalid, "kv choose: null weight or src");
    if (!s->cache.track)
      return Status::err(wv::kInvalid, "kv choose: needs a session mounted with WELVET_KV_TRACK");
    if (budget <= 0 || budget > s->cache.pool.capacity())
      return Status::err(wv::kInvalid, "kv choose: budget outside the capacity");
    if (sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
      return Status::err(wv::kInvalid, "kv choose: sinks and recent entries exceed the budget");
    return wv::kv_choose(s->cache, q, budget, sinks, recent, src,
                                pick(stream, s->stream.s));
  });
}

welvet_status welvet_kv_compact_device(welvet_kv_session* s, const welvet_kv_seqs* seqs,
                                       int32_t budget, const int32_t* src, void* stream) {
  return guarded([&]() -> Status {
    wv::KvSeqs q;
    WV_TRY(kv_seqs(s, seqs, &q));
    if (!src) return Status::err(wv::kInvalid, "kv compact: null src");
    if (budget <= 0 || budget > s->cache.pool.capacity())
      return Status::err(wv::kInvalid, "kv compact: budget outside the capacity");
    return wv::launch_kv_compact(s->cache.pool, q, budget, src, pick(stream, s->stream.s));
  });
}

welvet_status welvet_kv_advance_device(welvet_kv_session* s, int32_t nseq, int32_t* lens,
                                       int32_t* next_pos, const int32_t* counts, int32_t add,
                                       int32_t cap, void* stream) {
  return guarded([&]() -> Status {
    if (!s || !lens) return Status::err(wv::kInvalid, "kv advance: null session or lens");
    if (nseq < 0 || nseq > s->cache.max_seqs)
      return Status::err(wv::kInvalid, "kv: nseq outside the mounted number of sequences");
    const int capacity = s->cache.pool.capacity();
    if (add < 0 || add > capacity || cap < 0 || cap > capacity)
      return Status::err(wv::kInvalid, "kv advance: add or cap outside the capacity");
    return wv::launch_kv_advance(nseq, lens, next_pos, counts, add, cap ? cap : capacity,
                                 pick(stream, s->stream.s));
  });
}

// Whether an attention layer and a cache have the same heads.
static Status kv_matches(const wv::MHAConfig& c, const wv::KvPool& p) {
  if (c.num_heads != p.heads || c.num_kv_heads != p.kv_heads || c.head_dim != p.hd)
    return Status::err(wv::kInvalid, "mha: the cache was mounted for other heads");
  return Status::ok();
}

welvet_status welvet_mha_prefill_device(welvet_mha_session* m, welvet_kv_session* s,
                                        const welvet_kv_seqs* seqs, int32_t tokens, const float* x,
                                        float* pre, float* post, void* stream) {
  return guarded([&]() -> Status {
    if (!m || !x || !pre || !post) return Status::err(wv::kInvalid, "mha prefill: invalid argument");
    wv::KvSeqs q;
    WV_TRY(kv_seqs(s, seqs, &q));
    WV_TRY(kv_matches(m->layer.cfg, s->cache.pool));
    if (m->batch != 1 || q.nseq != 1)
      return Status::err(wv::kInvalid, "mha prefill: one sequence, in a session mounted with batch 1");
    if (tokens < 0 || tokens > m->seq || tokens > s->cache.pool.capacity())
      return Status::err(wv::kInvalid, "mha prefill: tokens outside the mounted seq or the capacity");
    return wv::mha_prefill(m->layer, s->cache, q, m->seq, tokens, x, pre, post, &m->ws,
                           pick(stream, m->stream.s));
  });
}

welvet_status welvet_mha_decode_device(welvet_mha_session* m, welvet_kv_session* s,
                                       const welvet_kv_seqs* seqs, const float* x, float* pre,
                                       float* post, void* stream) {
  return guarded([&]() -> Status {
    if (!m || !x || !pre || !post) return Status::err(wv::kInvalid, "mha decode: invalid argument");
    wv::KvSeqs q;
    WV_TRY(kv_seqs(s, seqs, &q));
    WV_TRY(kv_matches(m->layer.cfg, s->cache.pool));
    if (m->seq != 1 || q.nseq != m->batch)
      return Status::err(wv::kInvalid, "mha decode: nseq must be the batch of a session mounted with seq 1");
    if (q.weight && !s->cache.track)
      return Status::err(wv::kInvalid, "mha decode: running sums need a cache mounted with WELVET_KV_TRACK");
    return wv::mha_decode(m->layer, s->cache, q, x, pre, post, &m->ws, pick(stream, m->stream.s));
  });
}

// ---------------------------------------------------------------- model ----
struct welvet_model_session {
  std::mutex mu;
  wv::Stream stream;
  wv::Model model;
};

int32_t welvet_model_abi_version(void) { return 1; }

static welvet_status model_mount(const uint8_t* descriptor, size_t size, int32_t backend,
                                 welvet_model_session** out) {
  if (out) *out = nullptr;
  if (!out || !descriptor) return invalid("invalid mount arguments");
  return guarded([&]() -> Status {
    auto s = std::make_unique<welvet_model_session>();
    WV_TRY(wv::model_parse(descriptor, size, backend, &s->model));
    WV_TRY(wv::init_device());
    WV_TRY(s->stream.create());
    WV_TRY(wv::model_build(&s->model, s->stream.s));
    *out = s.release();
    return Status::ok();
  });
}

welvet_status welvet_model_mount(const uint8_t* descriptor, size_t size,
                                 welvet_model_session** out) {
  return model_mount(descriptor, size, 0, out);
}

welvet_status welvet_model_mount_q(const uint8_t* descriptor, size_t size, int32_t backend,
                                   welvet_model_session** out) {
  return model_mount(descriptor, size, backend, out);
}

// Input tensor wire (model_session.cpp:101-116): i32 rank (1..5), i32 dims,
// then the f32 data without a count. Output (:117-122): rank, dims, i32 count,
// data.
welvet_status welvet_model_forward(welvet_model_session* s, const uint8_t* input, size_t size,
                                   welvet_cuda_blob* out) {
  if (!s || !input || !out) return invalid("invalid forward arguments");
  out->data = nullptr;
  out->size = 0;
  return guarded([&]() -> Status {
    std::lock_guard<std::mutex> lock(s->mu);
    size_t off = 0;
    auto rd = [&](void* dst, size_t n) {
      if (size - off < n) return false;
      std::memcpy(dst, input + off, n);
      off += n;
      return true;
    };
    int32_t rank = 0;
    if (!rd(&rank, 4) || rank <= 0 || rank > 5) return Status::err(wv::kInvalid, "tensor rank must be 1..5");
    std::vector<int> shape((size_t)rank);
    size_t n = 1;
    for (auto& d : shape) {
      int32_t v = 0;
      if (!rd(&v, 4) || v <= 0 || n > (size_t(1) << 26) / (size_t)v)
        return Status::err(wv::kInvalid, "invalid tensor shape");
      d = v;
      n *= (size_t)v;
    }
    if ((size - off) / 4 < n) return Status::err(wv::kInvalid, "short tensor data");
    if (size - off != n * 4) return Status::err(wv::kInvalid, "trailing descriptor bytes");
    hipStream_t st = s->stream.s;
    // the input buffer and the pass's buffers are kept by the model
    wv::DevBuf& dx = s->model.scratch.in;
    if (dx.bytes < n * 4) WV_TRY(dx.alloc(n * 4));
    WV_TRY(wv::copy_h2d(dx.p, input + off, n * 4, st));
    std::vector<int> oshape;
    const float* dy = nullptr;
    WV_TRY(wv::model_forward_view(s->model, shape, dx.as<float>(), &oshape, &dy, st));
    size_t on = 1;
    for (int d : oshape) on *= (size_t)d;
    std::vector<uint8_t> blob;
    auto put = [&](const void* p, size_t k) {
      const uint8_t* b = static_cast<const uint8_t*>(p);
      blob.insert(blob.end(), b, b + k);
    };
    const int32_t orank = (int32_t)oshape.size();
    put(&orank, 4);
    for (int d : oshape) {
      const int32_t v = d;
      put(&v, 4);
    }
    const int32_t cnt = (int32_t)on;
    put(&cnt, 4);
    const size_t hdr = blob.size();
    blob.resize(hdr + on * 4);
    WV_TRY(wv::copy_d2h(blob.data() + hdr, dy, on * 4, st));
    WV_HIP(hipStreamSynchronize(st));
    out->data = static_cast<uint8_t*>(std::malloc(blob.size()));
    if (!out->data) return Status::err(wv::kInternal, "out of host memory");
    std::memcpy(out->data, blob.data(), blob.size());
    out->size = blob.size();
    return Status::ok();
  });
}

welvet_status welvet_model_forward_device(welvet_model_session* s, const float* x, int32_t batch,
                                          int32_t width, float* y, int32_t y_cap, void* stream) {
  if (!s || !x || !y || batch <= 0 || width <= 0 || y_cap <= 0)
    return invalid("invalid forward arguments");
  return guarded([&]() -> Status {
    std::lock_guard<std::mutex> lock(s->mu);
    std::vector<int> oshape;
    return wv::model_forward(s->model, {batch, width}, x, &oshape, y, (size_t)y_cap,
                             pick(stream, s->stream.s));
  });
}

welvet_status welvet_model_export_weights(welvet_model_session* s, welvet_cuda_blob* out) {
  if (!s || !out) return invalid("invalid export arguments");
  out->data = nullptr;
  out->size = 0;
  return guarded([&]() -> Status {
    std::lock_guard<std::mutex> lock(s->mu);
    std::vector<uint8_t> blob;
    WV_TRY(wv::model_export(s->model, &blob));
    out->data = static_cast<uint8_t*>(std::malloc(blob.size()));
    if (!out->data) return Status::err(wv::kInternal, "out of host memory");
    std::memcpy(out->data, blob.data(), blob.size());
    out->size = blob.size();
    return Status::ok();
  });
}

void welvet_model_release(welvet_model_session* s) { delete s; }

void welvet_cuda_blob_free(welvet_cuda_blob* b) {
  if (b) {
    std::free(b->data);
    b->data = nullptr;
    b->size = 0;
  }
}

// ---------------------------------------------------------- codec check ----
welvet_status welvet_codec_sweep(int32_t dtype, uint32_t first_chunk, uint32_t n_chunks,
                                 int64_t* out) {
  if (!out || n_chunks == 0 || (uint64_t)first_chunk + n_chunks > 4096u)
    return invalid("codec sweep: chunk range must lie in [0, 4096)");
  if (dtype != wv::kE4M3 && dtype != wv::kE5M2 && dtype != wv::kFP4)
    return to_c(Status::err(wv::kUnsupported, "codec sweep: dtype"));
  return guarded([&]() -> Status {
    WV_TRY(wv::init_device());
    wv::Stream s;
    WV_TRY(s.create());
    return wv::codec_sweep(dtype, first_chunk, n_chunks, out, s.s);
  });
}

// ------------------------------------------------------------- seqmix ----
// Metadata only (reference include/welvet/seqmix.hpp): kind tags.
welvet_status welvet_seqmix_kind_name(int32_t kind, char* buf, int32_t buf_len) {
  if (!buf || buf_len <= 0) return invalid("seqmix: bad buf");
  static const char* names[] = {"attention", "ssm", "linear_attn", "conv_mix"};
  if (kind < 0 || kind > 3) {
    welvet_status st{};
    st.code = wv::kInvalid;
    std::snprintf(st.message, sizeof(st.message), "seqmix: unknown kind %d", (int)kind);
    return st;
  }
  std::snprintf(buf, (size_t)buf_len, "%s", names[kind]);
  return to_c(Status::ok());
}
int32_t welvet_seqmix_mha_kind(void) { return 0; }
int32_t welvet_seqmix_mamba_kind(void) { return 1; }
int32_t welvet_seqmix_gdn_kind(void) { return 2; }

// ------------------------------------------------- outside this path ----
welvet_status welvet_model_train_credit(welvet_model_session*, int32_t, double, const uint8_t*,
                                        size_t) {
  return gap("model train credit");
}
// A model-wire tensor (model_session.cpp tensor(): int32 rank 1..5, the
// dims, float32 data) read at *off; *data points into the blob.
static Status read_tensor(const uint8_t* p, size_t size, size_t* off, std::vector<int>* shape,
                          const float** data, size_t* n) {
  auto rd = [&](void* dst, size_t k) {
    if (size - *off < k) return false;
    std::memcpy(dst, p + *off, k);
    *off += k;
    return true;
  };
  int32_t rank = 0;
  if (!rd(&rank, 4) || rank <= 0 || rank > 5) return Status::err(wv::kInvalid, "tensor rank must be 1..5");
  shape->assign((size_t)rank, 0);
  *n = 1;
  for (auto& d : *shape) {
    int32_t v = 0;
    if (!rd(&v, 4) || v <= 0 || *n > (size_t(1) << 26) / (size_t)v)
      return Status::err(wv::kInvalid, "invalid tensor shape");
    d = v;
    *n *= (size_t)v;
  }
  if ((size - *off) / 4 < *n) return Status::err(wv::kInvalid, "short tensor data");
  *data = reinterpret_cast<const float*>(p + *off);
  *off += *n * 4;
  return Status::ok();
}

static void put_tensor(std::vector<uint8_t>* blob, const std::vector<int>& shape, size_t n,
                       size_t* data_at) {
  auto put = [&](const void* q, size_t k) {
    const uint8_t* b = static_cast<const uint8_t*>(q);
    blob->insert(blob->end(), b, b + k);
  };
  const int32_t rank = (int32_t)shape.size();
  put(&rank, 4);
  for (int d : shape) {
    const int32_t v = d;
    put(&v, 4);
  }
  const int32_t cnt = (int32_t)n;
  put(&cnt, 4);
  *data_at = blob->size();
  blob->resize(blob->size() + n * 4);
}

// Segment backward (reference model_session.cpp:435-455): x and gy in, the
// input gradient and the concatenated dW (shape [1, n]) out.
welvet_status welvet_model_backward(welvet_model_session* s, const uint8_t* data, size_t size,
                                    welvet_cuda_blob* out) {
  if (!s || !data || !out) return invalid("invalid segment backward arguments");
  out->data = nullptr;
  out->size = 0;
  return guarded([&]() -> Status {
    std::lock_guard<std::mutex> lock(s->mu);
    size_t off = 0, nx = 0, ng = 0;
    std::vector<int> xs, gs;
    const float *hx = nullptr, *hg = nullptr;
    WV_TRY(read_tensor(data, size, &off, &xs, &hx, &nx));
    WV_TRY(read_tensor(data, size, &off, &gs, &hg, &ng));
    if (off != size) return Status::err(wv::kInvalid, "trailing descriptor bytes");
    hipStream_t st = s->stream.s;
    wv::DevBuf dx, dg;
    WV_TRY(dx.alloc(nx * 4));
    WV_TRY(dg.alloc(ng * 4));
    WV_TRY(wv::copy_h2d(dx.p, hx, nx * 4, st));
    WV_TRY(wv::copy_h2d(dg.p, hg, ng * 4, st));
    const float *gx = nullptr, *dw = nullptr;
    size_t nw = 0;
    WV_TRY(wv::model_backward(s->model, xs, dx.as<float>(), gs, dg.as<float>(), &gx, &dw, &nw, st));
    std::vector<uint8_t> blob;
    size_t at_x = 0, at_w = 0;
    put_tensor(&blob, xs, nx, &at_x);
    put_tensor(&blob, {1, (int)nw}, nw, &at_w);
    WV_TRY(wv::copy_d2h(blob.data() + at_x, gx, nx * 4, st));
    if (nw) WV_TRY(wv::copy_d2h(blob.data() + at_w, dw, nw * 4, st));
    WV_HIP(hipStreamSynchronize(st));
    out->data = static_cast<uint8_t*>(std::malloc(blob.size()));
    if (!out->data) return Status::err(wv::kInternal, "out of host memory");
    std::memcpy(out->data, blob.data(), blob.size());
    out->size = blob.size();
    return Status::ok();
  });
}

static Status blob_out(const std::vector<uint8_t>& blob, welvet_cuda_blob* out) {
  out->data = static_cast<uint8_t*>(std::malloc(blob.size()));
  if (!out->data) return Status::err(wv::kInternal, "out of host memory");
  std::memcpy(out->data, blob.data(), blob.size());
  out->size = blob.size();
  return Status::ok();
}

// Segment forward (reference model_session.cpp:420-434): x in; the last
// op's pre-activation and the output out.
welvet_status welvet_model_forward_pair(welvet_model_session* s, const uint8_t* data, size_t size,
                                        welvet_cuda_blob* out) {
  if (!s || !data || !out) return invalid("invalid segment forward arguments");
  out->data = nullptr;
  out->size = 0;
  return guarded([&]() -> Status {
    std::lock_guard<std::mutex> lock(s->mu);
    size_t off = 0, nx = 0;
    std::vector<int> xs;
    const float* hx = nullptr;
    WV_TRY(read_tensor(data, size, &off, &xs, &hx, &nx));
    if (off != size) return Status::err(wv::kInvalid, "trailing descriptor bytes");
    hipStream_t st = s->stream.s;
    wv::DevBuf& dx = s->model.scratch.in;
    if (dx.bytes < nx * 4) WV_TRY(dx.alloc(nx * 4));
    WV_TRY(wv::copy_h2d(dx.p, hx, nx * 4, st));
    std::vector<int> shape;
    const float *pre = nullptr, *post = nullptr;
    WV_TRY(wv::model_forward_pair(s->model, xs, dx.as<float>(), &shape, &pre, &post, st));
    size_t n = 1;
    for (int d : shape) n *= (size_t)d;
    std::vector<uint8_t> blob;
    size_t at_pre = 0, at_post = 0;
    put_tensor(&blob, shape, n, &at_pre);
    put_tensor(&blob, shape, n, &at_post);
    WV_TRY(wv::copy_d2h(blob.data() + at_pre, pre, n * 4, st));
    WV_TRY(wv::copy_d2h(blob.data() + at_post, post, n * 4, st));
    WV_HIP(hipStreamSynchronize(st));
    return blob_out(blob, out);
  });
}

// Dense proxy (reference model_session.cpp:475-493) of a Stack holding one
// Dense: x, gy, an int32 flag and (flag 1) pre in; kind 0 the linear input
// gradient [batch, in], kind 1 dW [out, in] out.
welvet_status welvet_model_dense_proxy(welvet_model_session* s, int32_t kind, const uint8_t* data,
                                       size_t size, welvet_cuda_blob* out) {
  if (!s || !data || !out || kind < 0 || kind > 1) return invalid("invalid Dense proxy arguments");
  out->data = nullptr;
  out->size = 0;
  return guarded([&]() -> Status {
    std::lock_guard<std::mutex> lock(s->mu);
    wv::Model& m = s->model;
    if (m.root != 0 || m.children.size() != 1 || m.children[0].kind != 1)
      return Status::err(wv::kInvalid, "proxy expects one Dense");
    const wv::DenseLayer& L = *m.children[0].dense;
    size_t off = 0, nx = 0, ng = 0, np = 0;
    std::vector<int> xs, gs, ps;
    const float *hx = nullptr, *hg = nullptr, *hp = nullptr;
    WV_TRY(read_tensor(data, size, &off, &xs, &hx, &nx));
    WV_TRY(read_tensor(data, size, &off, &gs, &hg, &ng));
    int32_t present = 0;
    if (size - off < 4) return Status::err(wv::kInvalid, "short descriptor");
    std::memcpy(&present, data + off, 4);
    off += 4;
    if (present != 0 && present != 1) return Status::err(wv::kInvalid, "invalid pre flag");
    if (present) WV_TRY(read_tensor(data, size, &off, &ps, &hp, &np));
    if (off != size) return Status::err(wv::kInvalid, "trailing descriptor bytes");
    if (xs.size() != 2 || xs[0] <= 0 || ng == 0 || (size_t)xs[0] * L.in != nx)
      return Status::err(wv::kInvalid, kind == 0 ? "dense: LinearGradIn shape" : "dense: GradWOnly shape");
    const size_t b = (size_t)xs[0], ny = b * L.out;
    const std::vector<float> g = wv::remap_len(hg, ng, ny);
    // kind 1 uses pre only when it is 2-D and long enough (dense.cpp:183-187)
    const bool use_pre = kind == 1 && present && ps.size() == 2 && np >= ny;
    hipStream_t st = s->stream.s;
    wv::DevBuf dx, dg, dp;
    WV_TRY(dx.alloc(nx * 4));
    WV_TRY(dg.alloc(ny * 4));
    WV_TRY(wv::copy_h2d(dx.p, hx, nx * 4, st));
    WV_TRY(wv::copy_h2d(dg.p, g.data(), ny * 4, st));
    if (use_pre) {
      WV_TRY(dp.alloc(ny * 4));
      WV_TRY(wv::copy_h2d(dp.p, hp, ny * 4, st));
    }
    const float* res = nullptr;
    WV_TRY(wv::model_dense_proxy(m, kind, xs, dx.as<float>(), dg.as<float>(),
                                 use_pre ? dp.as<float>() : nullptr, &res, st));
    const std::vector<int> shape = kind == 0 ? std::vector<int>{(int)b, L.in}
                                             : std::vector<int>{L.out, L.in};
    const size_t n = (size_t)shape[0] * shape[1];
    std::vector<uint8_t> blob;
    size_t at = 0;
    put_tensor(&blob, shape, n, &at);
    WV_TRY(wv::copy_d2h(blob.data() + at, res, n * 4, st));
    WV_HIP(hipStreamSynchronize(st));
    return blob_out(blob, out);
  });
}

// Segment SGD (reference model_session.cpp:494-507): one tensor, the
// concatenated dW; each Dense store is updated and re-quantized.
welvet_status welvet_model_apply_sgd(welvet_model_session* s, double lr, const uint8_t* data,
                                     size_t size) {
  if (!s || !data || !std::isfinite(lr)) return invalid("invalid segment SGD arguments");
  return guarded([&]() -> Status {
    std::lock_guard<std::mutex> lock(s->mu);
    size_t off = 0, n = 0;
    std::vector<int> shape;
    const float* hw = nullptr;
    WV_TRY(read_tensor(data, size, &off, &shape, &hw, &n));
    if (off != size) return Status::err(wv::kInvalid, "trailing descriptor bytes");
    hipStream_t st = s->stream.s;
    wv::DevBuf d;
    WV_TRY(d.alloc(n * 4));
    WV_TRY(wv::copy_h2d(d.p, hw, n * 4, st));
    WV_TRY(wv::model_apply_sgd(s->model, d.as<float>(), n, lr, st));
    WV_HIP(hipStreamSynchronize(st));
    return Status::ok();
  });
}
welvet_status welvet_model_train_mse(welvet_model_session*, int32_t, double, int32_t,
                                     const uint8_t*, size_t, double*) {
  return gap("model training");
}
welvet_status welvet_model_sync(welvet_model_session*, int32_t) { return gap("model sync"); }

#define WV_GAP_NBP(name, ...) \
  welvet_status name(__VA_ARGS__) { return gap(#name); }

WV_GAP_NBP(welvet_rmsnorm_forward_f32, int32_t, int32_t, int32_t, double, int32_t, int32_t,
           const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_rmsnorm_normalbp_f32, int32_t, int32_t, int32_t, double, int32_t, int32_t,
           const float*, const float*, const float*, int32_t, double, float*, float*, float*,
           float*, float*, double*)
WV_GAP_NBP(welvet_layernorm_forward_f32, int32_t, int32_t, int32_t, double, int32_t, int32_t,
           const float*, const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_layernorm_normalbp_f32, int32_t, int32_t, int32_t, double, int32_t, int32_t,
           const float*, const float*, const float*, const float*, int32_t, double, float*, float*,
           float*, float*, float*, float*, double*)
WV_GAP_NBP(welvet_softmax_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           double, double, int32_t, int32_t, int32_t, int32_t, const int32_t*, const uint8_t*,
           int32_t, const int32_t*, int32_t, const float*, float*, float*)
WV_GAP_NBP(welvet_softmax_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           double, double, int32_t, int32_t, int32_t, int32_t, const int32_t*, const uint8_t*,
           int32_t, const int32_t*, int32_t, const float*, const float*, int32_t, double, float*,
           float*, float*, double*)
WV_GAP_NBP(welvet_embedding_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_embedding_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, const float*, const float*, const float*, int32_t, double,
           float*, float*, float*, float*, float*, double*)
WV_GAP_NBP(welvet_mha_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, const float*, const float*, const float*,
           const float*, const float*, const float*, int32_t, double, float*, float*, float*,
           float*, float*, double*)
WV_GAP_NBP(welvet_cnn1_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, const float*, const double*, size_t, const float*, float*,
           float*)
WV_GAP_NBP(welvet_cnn1_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, const float*, const double*, size_t, const float*,
           const float*, int32_t, double, float*, float*, float*, float*, float*, double*)
WV_GAP_NBP(welvet_cnn2_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, const float*, const double*, size_t, const float*,
           float*, float*)
WV_GAP_NBP(welvet_cnn2_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, const float*, const double*, size_t, const float*,
           const float*, int32_t, double, float*, float*, float*, float*, float*, double*)
WV_GAP_NBP(welvet_cnn3_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, int32_t, const float*, const double*, size_t,
           const float*, float*, float*)
WV_GAP_NBP(welvet_cnn3_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, int32_t, const float*, const double*, size_t,
           const float*, const float*, int32_t, double, float*, float*, float*, float*, float*,
           double*)
WV_GAP_NBP(welvet_convt1_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_convt1_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, int32_t, const float*, const float*, const float*,
           int32_t, double, float*, float*, float*, float*, float*, double*)
WV_GAP_NBP(welvet_convt2_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, int32_t, const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_convt2_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, const float*, const float*,
           const float*, int32_t, double, float*, float*, float*, float*, float*, double*)
WV_GAP_NBP(welvet_convt3_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, const float*, const float*, float*,
           float*)
WV_GAP_NBP(welvet_convt3_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, const float*,
           const float*, const float*, int32_t, double, float*, float*, float*, float*, float*,
           double*)
WV_GAP_NBP(welvet_rnn_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_rnn_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           const float*, const float*, const float*, int32_t, double, float*, float*, float*,
           float*, float*, double*)
WV_GAP_NBP(welvet_lstm_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_lstm_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           const float*, const float*, const float*, int32_t, double, float*, float*, float*,
           float*, float*, double*)
WV_GAP_NBP(welvet_sequential_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_sequential_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, const float*, const float*, const float*, int32_t, double, float*, float*,
           float*, float*, float*, double*)
WV_GAP_NBP(welvet_residual_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_residual_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, const float*, const float*, const float*, int32_t, double, float*, float*,
           float*, float*, float*, double*)
WV_GAP_NBP(welvet_stack_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, const float*, const float*, const float*, int32_t, double, float*, float*,
           float*, float*, float*, double*)
WV_GAP_NBP(welvet_mamba_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, const float*, const float*, const float*, int32_t, double, float*, float*,
           float*, float*, float*, double*)
WV_GAP_NBP(welvet_metacognition_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t,
           const float*, const float*, const float*, int32_t, double, float*, float*, float*,
           float*, float*, double*)
WV_GAP_NBP(welvet_gdn_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, const float*, const float*, const float*, int32_t, double,
           float*, float*, float*, float*, float*, double*)
WV_GAP_NBP(welvet_kmeans_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           double, int32_t, int32_t, const float*, const float*, const float*, int32_t, double,
           float*, float*, float*, float*, float*, double*)
WV_GAP_NBP(welvet_parallel_normalbp_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, double, const float*, const float*, const float*, int32_t,
           double, float*, float*, float*, float*, float*, double*)
WV_GAP_NBP(welvet_mamba_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_metacognition_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t,
           const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_gdn_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_kmeans_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, double, int32_t,
           int32_t, int32_t, const int32_t*, const float*, const float*, float*, float*)
WV_GAP_NBP(welvet_parallel_forward_f32, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t,
           int32_t, int32_t, int32_t, double, const float*, const float*, float*, float*)

}  // extern "C"
