// C entry points of the plain mixture-of-adapters operators
// (include/tensafe_he.h): argument checks, workspace layout, launches.
#include "mixture.h"

#include "runtime.h"

namespace {

// The current device once per call: a usable gfx950, or TH_EDEVICE.
void need_device() {
  static std::atomic<uint32_t> good{0};  // bit d: device d has been looked at
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) {
    (void)hipGetLastError();
    raise(TH_EDEVICE, "no HIP device available (the mixture operators require an MI355X / gfx950 GPU)");
  }
  if (dev < 32 && (good.load(std::memory_order_relaxed) >> dev & 1)) return;
  int n = 0;
  if (hipGetDeviceCount(&n) != hipSuccess || n == 0) {
    (void)hipGetLastError();
    raise(TH_EDEVICE, "no HIP device available (the mixture operators require an MI355X / gfx950 GPU)");
  }
  hipDeviceProp_t prop;
  HIPCHK(hipGetDeviceProperties(&prop, dev));
  if (strncmp(prop.gcnArchName, "gfx950", 6) != 0)
    raise(TH_EDEVICE, std::string("device is ") + prop.gcnArchName + ", the operators are built for gfx950");
  if (dev < 32) good.fetch_or(1u << dev, std::memory_order_relaxed);
}

MixType mix_type(int dtype, bool with_float) {
  need(dtype == TH_BF16 || dtype == TH_F16 || (with_float && dtype == TH_F32),
       with_float ? "dtype must be TH_BF16, TH_F16 or TH_F32" : "dtype must be TH_BF16 or TH_F16");
  return (MixType)dtype;
}

// Consecutive pieces of the caller's workspace, each on 256 bytes; with a null
// base it only adds up their sizes.
class Pieces {
 public:
  explicit Pieces(void* base) : base_((char*)base) {}
  template <class T>
  T* take(uint64_t count) {
    T* p = base_ ? (T*)(base_ + used_) : nullptr;
    used_ += (count * sizeof(T) + 255) & ~(uint64_t)255;
    return p;
  }
  uint64_t used() const { return used_; }

 private:
  char* base_;
  uint64_t used_ = 0;
};

void need_work(const void* work, size_t have, uint64_t want) {
  need(want == 0 || work != nullptr, "this call needs a workspace");
  need(have >= want, "the workspace has " + std::to_string(have) + " bytes, " + std::to_string(want) + " are needed");
  need(((uintptr_t)work & 255) == 0, "the workspace must start on a multiple of 256 bytes");
}

void need_slots(int64_t tokens, uint32_t experts, uint32_t choices) {
  need(tokens >= 0, "negative token count");
  need(experts >= 1 && experts <= th::MIX_MAX_EXPERTS,
       "the number of experts must be in [1, " + std::to_string(th::MIX_MAX_EXPERTS) + "]");
  need(choices >= 1 && choices <= th::MIX_MAX_CHOICES,
       "choices must be in [1, " + std::to_string(th::MIX_MAX_CHOICES) + "]");
  need(tokens <= 0x7fffffff / (int64_t)choices, "tokens x choices must be below 2^31");
}

void need_rows(const void* p, int64_t rows, int64_t ld, int64_t width, const char* what) {
  need(rows == 0 || p != nullptr, std::string("null ") + what);
  need(rows <= 1 || ld >= width, std::string(what) + ": the row stride is shorter than a row");
}

uint64_t hist_words(int64_t tokens, uint32_t experts, uint32_t choices) {
  const uint64_t chunks = th::group_chunks((uint64_t)tokens, choices);
  return chunks > 1 ? chunks * (experts + 1) : 0;
}

uint32_t padded_rank(uint32_t r) { return (r + 3) & ~3u; }

// Rows of 2-byte elements that all start on 16 bytes.
bool on16(const void* p, int64_t ld, int64_t rows = 2) { return ((uintptr_t)p & 15) == 0 && (rows < 2 || ld % 8 == 0); }

// A stack of matrices as the products read it: the caller's, or a copy with
// rows of a multiple of 8 values, zeros beyond the caller's.
struct Stack {
  const void* p;
  int64_t ld, lde;
  uint32_t E, cols;
  int64_t rows;
  void* copy;
  bool ready() const { return on16(p, ld, rows) && (E < 2 || lde % 8 == 0) && cols % 8 == 0; }
  uint32_t padded() const { return (cols + 7) & ~7u; }
  void lay(Pieces& work, bool needed) {
    if (needed) copy = work.take<uint16_t>((uint64_t)E * rows * padded());
  }
  void use_copy() {
    if (!copy) return;
    cols = padded();
    p = copy;
    ld = cols;
    lde = ld * rows;
  }
};
void make_copies(Stack& a, Stack& b, Stack& c, hipStream_t s) {
  PadSet set{};
  Stack* all[3] = {&a, &b, &c};
  for (int i = 0; i < 3; ++i) {
    set.p[i] = PadArgs{all[i]->p, all[i]->copy, all[i]->ld, all[i]->lde, all[i]->E, all[i]->cols, all[i]->rows};
    all[i]->use_copy();
  }
  HIPCHK(launch_pad(set, s));
}

// ---------------------------------------------------------------- grouped products
void check_grouped(const th_grouped* d) {
  need(d != nullptr, "null descriptor");
  mix_type(d->dtype, false);
  need_slots(d->tokens, d->experts, d->choices);
  need(d->d_in >= 1 && d->d_out >= 1, "d_in and d_out must be positive");
  need_rows(d->x, d->x_per_slot ? d->tokens * d->choices : d->tokens, d->ldx, d->d_in, "x");
  need(d->w != nullptr, "null w");
  need(d->ldw >= d->d_in, "w: the row stride is shorter than a row");
  need(d->tokens == 0 || (d->order && d->offsets), "null groups");
}

struct GroupedWork {
  Stack x{}, w{}, dy{};
  float* part = nullptr;  // a token's choices, to be summed
};
GroupedWork lay_grouped_backward(Pieces& p, const th_grouped* d, const void* dy, int64_t lddy) {
  GroupedWork g;
  const int64_t slots = d->tokens * d->choices;
  g.x = Stack{d->x, d->ldx, 0, 1, d->d_in, d->x_per_slot ? slots : d->tokens, nullptr};
  g.w = Stack{d->w, d->ldw, d->ldwe, d->experts, d->d_in, d->d_out, nullptr};
  g.dy = Stack{dy, lddy, 0, 1, d->d_out, slots, nullptr};
  for (Stack* t : {&g.x, &g.w}) t->lay(p, !t->ready());
  g.dy.lay(p, d->d_out % 8 != 0);  // the workspace's size does not depend on where dy lies
  if (!d->x_per_slot && d->choices > 1) g.part = p.take<float>((uint64_t)slots * d->d_in);
  return g;
}

// ---------------------------------------------------------------- shared projection with adapters
void check_lora(const th_lora_linear_args* d) {
  need(d != nullptr, "null descriptor");
  mix_type(d->dtype, false);
  need_slots(d->tokens, d->adapters, d->choices);
  need(d->d_in >= 1 && d->d_out >= 1, "d_in and d_out must be positive");
  need(d->rank >= 1 && d->rank <= th::MIX_MAX_RANK, "rank must be in [1, " + std::to_string(th::MIX_MAX_RANK) + "]");
  need_rows(d->x, d->tokens, d->ldx, d->d_in, "x");
  need(d->weight && d->a && d->b, "null weight or adapter");
  need(d->ldw >= d->d_in, "weight: the row stride is shorter than a row");
  need(d->lda >= d->d_in, "a: the row stride is shorter than a row");
  need(d->ldb >= d->rank, "b: the row stride is shorter than a row");
  need(d->tokens == 0 || d->experts, "null experts");
  need(d->tokens == 0 || (d->order == nullptr) == (d->offsets == nullptr), "order and offsets go together");
}

struct LoraWork {
  Stack x{}, weight{}, a{}, dy{};
  int32_t *order = nullptr, *offsets = nullptr;
  uint32_t* hist = nullptr;
  float *u = nullptr, *v = nullptr, *partial[2] = {};
  uint16_t *at = nullptr, *bt = nullptr;
};
// Few slots that nothing else needs grouped: the low-rank product finds each
// adapter's slots by itself.
bool scans(const th_lora_linear_args* d, bool keep_u) {
  return !d->order && !keep_u && (uint64_t)d->tokens * d->choices <= th::NARROW_SCAN_SLOTS;
}
LoraWork lay_groups(Pieces& p, const th_lora_linear_args* d, bool own_lists = false) {
  LoraWork w;
  w.x = Stack{d->x, d->ldx, 0, 1, d->d_in, d->tokens, nullptr};
  w.weight = Stack{d->weight, d->ldw, 0, 1, d->d_in, d->d_out, nullptr};
  w.a = Stack{d->a, d->lda, d->lda_adapter, d->adapters, d->d_in, d->rank, nullptr};
  if (!d->order && !own_lists) {
    w.order = p.take<int32_t>((uint64_t)d->tokens * d->choices);
    w.offsets = p.take<int32_t>(d->adapters + 1);
    w.hist = p.take<uint32_t>(hist_words(d->tokens, d->adapters, d->choices));
  }
  return w;
}
LoraWork lay_forward(Pieces& p, const th_lora_linear_args* d, bool keep_u) {
  LoraWork w = lay_groups(p, d, scans(d, keep_u));
  for (Stack* t : {&w.x, &w.weight, &w.a}) t->lay(p, th::pad_operands(d->tokens, d->d_in) && !t->ready());
  if (!keep_u) w.u = p.take<float>((uint64_t)d->tokens * d->choices * padded_rank(d->rank));
  return w;
}
LoraWork lay_backward(Pieces& p, const th_lora_linear_args* d, const void* dy, int64_t lddy) {
  LoraWork w = lay_groups(p, d);
  w.dy = Stack{dy, lddy, 0, 1, d->d_out, d->tokens, nullptr};
  for (Stack* t : {&w.x, &w.weight}) t->lay(p, !t->ready());
  w.dy.lay(p, d->d_out % 8 != 0);  // the workspace's size does not depend on where dy lies
  const uint64_t slots = (uint64_t)d->tokens * d->choices;
  w.v = p.take<float>(slots * padded_rank(d->rank));
  w.at = p.take<uint16_t>((uint64_t)d->adapters * d->d_in * d->rank);
  w.bt = p.take<uint16_t>((uint64_t)d->adapters * w.dy.padded() * d->rank);
  for (int i = 0; i < 2; ++i) {
    const uint32_t cols = i ? d->d_out : d->d_in;
    w.partial[i] =
        p.take<float>(th::lowrank_spans(slots, d->adapters, th::lowrank_span(slots, cols)) * d->rank * cols);
  }
  return w;
}

// The groups given, or made in the workspace.
void make_groups(const th_lora_linear_args* d, LoraWork& w, hipStream_t s) {
  if (d->order) {
    w.order = const_cast<int32_t*>(d->order);
    w.offsets = const_cast<int32_t*>(d->offsets);
    return;
  }
  RouteArgs g{};
  g.T = d->tokens;
  g.E = d->adapters;
  g.k = d->choices;
  g.experts = const_cast<int32_t*>(d->experts);
  g.order = w.order;
  g.offsets = w.offsets;
  g.hist = w.hist;
  HIPCHK(launch_group(g, s));
}

// low (slots x rank floats) = one low-rank factor of every slot's adapter times
// its token's row of `wide`.
void shrink(const th_lora_linear_args* d, const LoraWork& w, const Stack& wide, const Stack& factor, float* low,
            hipStream_t s) {
  MatArgs m{};
  m.scan = w.offsets == nullptr;
  m.ids = d->experts;
  m.x = wide.p;
  m.ldx = wide.ld;
  m.w = factor.p;
  m.ldw = factor.ld;
  m.ldwe = factor.lde;
  m.y = low;
  m.ldy = padded_rank(d->rank);
  m.y_float = 1;
  m.order = w.order;
  m.offsets = w.offsets;
  m.rows = d->tokens * d->choices;
  m.n = d->rank;
  m.k = wide.cols;
  m.E = d->adapters;
  m.div = d->choices;
  m.aligned = wide.ready() && factor.ready();
  HIPCHK(launch_mat((MixType)d->dtype, m, 0, s));
}

void set_lowrank(MatArgs& m, const th_lora_linear_args* d, const float* u, const void* p, int64_t ldp, int64_t ldpe) {
  m.p = p;
  m.ldp = ldp;
  m.ldpe = ldpe;
  m.u = u;
  m.ids = d->experts;
  m.gate = d->gate;
  m.scale = d->scale;
  m.r = d->rank;
  m.ru = padded_rank(d->rank);
  m.kc = d->choices;
  m.E = d->adapters;
}

}  // namespace

extern "C" {

int th_group_workspace(int64_t tokens, uint32_t experts, uint32_t choices, size_t* bytes) {
  return guarded([&] {
    need(bytes != nullptr, "null output");
    need_slots(tokens, experts, choices);
    *bytes = hist_words(tokens, experts, choices) * 4;
  });
}

int th_group(const int32_t* experts, int64_t tokens, uint32_t n_experts, uint32_t choices, int32_t* order,
             int32_t* offsets, void* work, size_t work_bytes, void* stream) {
  return guarded([&] {
    need_slots(tokens, n_experts, choices);
    need(offsets && (tokens == 0 || (experts && order)), "null argument");
    need_work(work, work_bytes, hist_words(tokens, n_experts, choices) * 4);
    need_device();
    RouteArgs a{};
    a.T = tokens;
    a.E = n_experts;
    a.k = choices;
    a.experts = const_cast<int32_t*>(experts);
    a.order = order;
    a.offsets = offsets;
    a.hist = (uint32_t*)work;
    HIPCHK(launch_group(a, (hipStream_t)stream));
  });
}

int th_route(int dtype, const void* logits, int64_t ld, int64_t tokens, uint32_t n_experts, const uint8_t* mask,
             int64_t mask_ld, uint32_t choices, int normalize, float* weights, int32_t* experts, int32_t* order,
             int32_t* offsets, void* work, size_t work_bytes, void* stream) {
  return guarded([&] {
    const MixType type = mix_type(dtype, true);
    need_slots(tokens, n_experts, choices);
    need(n_experts <= 512, "a gate has at most 512 experts");
    need(choices <= n_experts, "choices must not exceed the number of experts");
    need_rows(logits, tokens, ld, n_experts, "logits");
    need(!mask || mask_ld == 0 || mask_ld >= n_experts, "mask: the row stride is shorter than a row");
    need(offsets && (tokens == 0 || (weights && experts && order)), "null output");
    need_work(work, work_bytes, hist_words(tokens, n_experts, choices) * 4);
    need_device();
    RouteArgs a{};
    a.logits = logits;
    a.mask = mask;
    a.T = tokens;
    a.ld = ld;
    a.mask_ld = mask_ld;
    a.E = n_experts;
    a.k = choices;
    a.normalize = normalize;
    a.weights = weights;
    a.experts = experts;
    a.order = order;
    a.offsets = offsets;
    a.hist = (uint32_t*)work;
    HIPCHK(launch_route(type, a, (hipStream_t)stream));
  });
}

int th_route_backward(int dtype, const void* logits, int64_t ld, int64_t tokens, uint32_t n_experts,
                      const uint8_t* mask, int64_t mask_ld, uint32_t choices, int normalize, const float* weights,
                      const int32_t* experts, const float* dweights, void* dlogits, void* stream) {
  return guarded([&] {
    const MixType type = mix_type(dtype, true);
    need_slots(tokens, n_experts, choices);
    need(n_experts <= 512, "a gate has at most 512 experts");
    need(choices <= n_experts, "choices must not exceed the number of experts");
    need_rows(logits, tokens, ld, n_experts, "logits");
    need(!mask || mask_ld == 0 || mask_ld >= n_experts, "mask: the row stride is shorter than a row");
    need(tokens == 0 || (weights && experts && dweights && dlogits), "null argument");
    need_device();
    if (tokens == 0) return;
    RouteArgs a{};
    a.logits = logits;
    a.mask = mask;
    a.T = tokens;
    a.ld = ld;
    a.mask_ld = mask_ld;
    a.E = n_experts;
    a.k = choices;
    a.normalize = normalize;
    a.weights = const_cast<float*>(weights);
    a.experts = const_cast<int32_t*>(experts);
    HIPCHK(launch_route_backward(type, a, dweights, dlogits, (hipStream_t)stream));
  });
}

int th_grouped_matmul(const th_grouped* d, void* y, int64_t ldy, void* stream) {
  return guarded([&] {
    check_grouped(d);
    need_rows(y, d->tokens * d->choices, ldy, d->d_out, "y");
    need_device();
    MatArgs m{};
    m.x = d->x;
    m.ldx = d->ldx;
    m.w = d->w;
    m.ldw = d->ldw;
    m.ldwe = d->ldwe;
    m.y = y;
    m.ldy = ldy;
    m.order = d->order;
    m.offsets = d->offsets;
    m.rows = d->tokens * d->choices;
    m.n = d->d_out;
    m.k = d->d_in;
    m.E = d->experts;
    m.div = d->x_per_slot ? 1 : d->choices;
    m.aligned = on16(d->x, d->ldx) && on16(d->w, d->ldw) && d->ldwe % 8 == 0 && d->d_in % 8 == 0;
    HIPCHK(launch_mat((MixType)d->dtype, m, 0, (hipStream_t)stream));
  });
}

int th_grouped_matmul_backward_workspace(const th_grouped* d, size_t* bytes) {
  return guarded([&] {
    need(bytes != nullptr, "null output");
    check_grouped(d);
    Pieces p(nullptr);
    lay_grouped_backward(p, d, nullptr, d->d_out);
    *bytes = p.used();
  });
}

int th_grouped_matmul_backward(const th_grouped* d, const void* dy, int64_t lddy, void* dx, void* dw, void* work,
                               size_t work_bytes, void* stream) {
  return guarded([&] {
    check_grouped(d);
    need_rows(dy, d->tokens * d->choices, lddy, d->d_out, "dy");
    const MixType type = (MixType)d->dtype;
    const bool summed = !d->x_per_slot && d->choices > 1;
    Pieces p(work);
    GroupedWork g = lay_grouped_backward(p, d, dy, lddy);
    need_work(work, work_bytes, p.used());
    need_device();
    const hipStream_t s = (hipStream_t)stream;
    const int64_t slots = d->tokens * d->choices;
    if (slots) make_copies(g.x, g.w, g.dy, s);
    if (dx) {
      MatArgs m{};
      m.x = g.dy.p;
      m.ldx = g.dy.ld;
      m.w = g.w.p;
      m.ldw = g.w.ld;
      m.ldwe = g.w.lde;
      m.y = summed ? (void*)g.part : dx;
      m.y_float = summed;
      m.ldy = d->d_in;
      m.order = d->order;
      m.offsets = d->offsets;
      m.rows = slots;
      m.n = d->d_in;
      m.k = d->d_out;
      m.E = d->experts;
      m.div = 1;
      m.aligned = g.dy.ready() && g.w.ready();
      HIPCHK(launch_mat(type, m, 1, s));
      if (summed) HIPCHK(launch_sum_choices(type, g.part, dx, d->tokens, d->choices, d->d_in, s));
    }
    if (dw) {
      OuterArgs o{};
      o.dy = g.dy.p;
      o.lddy = g.dy.ld;
      o.x = g.x.p;
      o.ldx = g.x.ld;
      o.out = dw;
      o.order = d->order;
      o.offsets = d->offsets;
      o.slots = slots;
      o.n = d->d_out;
      o.k = d->d_in;
      o.E = d->experts;
      o.div = d->x_per_slot ? 1 : d->choices;
      o.aligned = g.dy.ready() && g.x.ready();
      need(d->offsets != nullptr, "null groups");
      HIPCHK(launch_outer(type, o, s));
    }
  });
}

int th_lora_linear_workspace(const th_lora_linear_args* d, int keep_u, size_t* bytes) {
  return guarded([&] {
    need(bytes != nullptr, "null output");
    check_lora(d);
    Pieces p(nullptr);
    lay_forward(p, d, keep_u != 0);
    *bytes = p.used();
  });
}

int th_lora_linear(const th_lora_linear_args* d, void* y, int64_t ldy, float* u, void* work, size_t work_bytes,
                   void* stream) {
  return guarded([&] {
    check_lora(d);
    need_rows(y, d->tokens, ldy, d->d_out, "y");
    Pieces p(work);
    LoraWork w = lay_forward(p, d, u != nullptr);
    need_work(work, work_bytes, p.used());
    need_device();
    if (d->tokens == 0) return;
    const hipStream_t s = (hipStream_t)stream;
    float* low = u ? u : w.u;
    if (!scans(d, u != nullptr)) make_groups(d, w, s);
    make_copies(w.x, w.weight, w.a, s);
    shrink(d, w, w.x, w.a, low, s);
    MatArgs m{};
    m.x = w.x.p;
    m.ldx = w.x.ld;
    m.w = w.weight.p;
    m.ldw = w.weight.ld;
    m.y = y;
    m.ldy = ldy;
    m.bias = d->bias;
    m.rows = d->tokens;
    m.n = d->d_out;
    m.k = w.x.cols;
    m.div = 1;
    m.aligned = w.x.ready() && w.weight.ready();
    set_lowrank(m, d, low, d->b, d->ldb, d->ldb_adapter);
    HIPCHK(launch_mat((MixType)d->dtype, m, 0, s));
  });
}

int th_lora_linear_backward_workspace(const th_lora_linear_args* d, size_t* bytes) {
  return guarded([&] {
    need(bytes != nullptr, "null output");
    check_lora(d);
    Pieces p(nullptr);
    lay_backward(p, d, nullptr, d->d_out);
    *bytes = p.used();
  });
}

int th_lora_linear_backward(const th_lora_linear_args* d, const float* u, const void* dy, int64_t lddy, void* dx,
                            void* da, void* db, float* dgate, void* work, size_t work_bytes, void* stream) {
  return guarded([&] {
    check_lora(d);
    need_rows(dy, d->tokens, lddy, d->d_out, "dy");
    need(d->tokens == 0 || u != nullptr || !(db || dgate), "null u");
    Pieces p(work);
    LoraWork w = lay_backward(p, d, dy, lddy);
    need_work(work, work_bytes, p.used());
    need_device();
    const hipStream_t s = (hipStream_t)stream;
    const MixType type = (MixType)d->dtype;
    const uint32_t ru = padded_rank(d->rank);
    const int64_t slots = d->tokens * d->choices;
    make_groups(d, w, s);
    if (slots) make_copies(w.x, w.weight, w.dy, s);
    if (slots && (dx || da || dgate)) {
      TransposePair t{};
      t.p[0] = TransposeArgs{d->b, w.bt, d->ldb, d->ldb_adapter, d->adapters, d->d_out, d->rank, w.dy.padded()};
      if (dx) t.p[1] = TransposeArgs{d->a, w.at, d->lda, d->lda_adapter, d->adapters, d->rank, d->d_in, d->rank};
      HIPCHK(launch_transpose(t, s));
      const uint32_t n = w.dy.padded();
      shrink(d, w, w.dy, Stack{w.bt, n, (int64_t)n * d->rank, d->adapters, n, d->rank, nullptr}, w.v, s);
    }
    if (slots && dx) {
      MatArgs m{};
      m.x = w.dy.p;
      m.ldx = w.dy.ld;
      m.w = w.weight.p;
      m.ldw = w.weight.ld;
      m.y = dx;
      m.ldy = d->d_in;
      m.rows = d->tokens;
      m.n = d->d_in;
      m.k = d->d_out;
      m.div = 1;
      m.aligned = w.dy.ready() && w.weight.ready();
      set_lowrank(m, d, w.v, w.at, d->rank, (int64_t)d->d_in * d->rank);
      HIPCHK(launch_mat(type, m, 1, s));
    }
    GateGradArgs gate{u, w.v, d->experts, d->scale, dgate, slots, d->rank, ru, d->adapters};
    if (da || db) {
      LowOuterPair pair{};
      pair.gate = gate;
      for (int which = 0; which < 2; ++which) {
        LowOuterArgs& o = pair.p[which];
        o.low = which ? u : w.v;
        const Stack& wide = which ? w.dy : w.x;
        o.wide = wide.p;
        o.ldwide = wide.ld;
        o.cols = which ? d->d_out : d->d_in;
        o.out = which ? db : da;
        o.partial = w.partial[which];
        o.order = w.order;
        o.offsets = w.offsets;
        o.gate = d->gate;
        o.scale = d->scale;
        o.slots = slots;
        o.r = d->rank;
        o.ru = ru;
        o.E = d->adapters;
        o.div = d->choices;
        o.span = th::lowrank_span(slots, o.cols);
        o.aligned = !o.out || wide.ready();
        o.transposed = which;
      }
      HIPCHK(launch_low_outer(type, pair, s));
    }
    if (dgate && !(da || db)) HIPCHK(launch_gate_grad(gate, s));
  });
}

}  // extern "C"
