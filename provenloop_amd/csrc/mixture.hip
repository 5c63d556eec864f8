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

// Of a gate: a balanced one has chunks of its own.
uint64_t gate_words(const RouteArgs& a) {
  const uint64_t chunks = balanced(a) ? th::gate_chunks(a.T, a.k) : th::group_chunks(a.T, a.k);
  return chunks > 1 ? chunks * (a.E + 1) : 0;
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

// ---------------------------------------------------------------- gates
th_gate_args plain_gate(int dtype, const void* logits, int64_t ld, int64_t tokens, uint32_t n_experts,
                        const uint8_t* mask, int64_t mask_ld, uint32_t choices, int normalize) {
  return th_gate_args{dtype, TH_SOFTMAX, normalize, n_experts, choices, 1, 1, 1, tokens, ld, mask_ld, logits, mask, nullptr, 1.0f};
}
RouteArgs check_gate(const th_gate_args& d) {
  mix_type(d.dtype, true);
  need_slots(d.tokens, d.n_experts, d.choices);
  need(d.n_experts <= 512, "a gate has at most 512 experts");
  need(d.choices <= d.n_experts, "choices must not exceed the number of experts");
  need_rows(d.logits, d.tokens, d.ld, d.n_experts, "logits");
  need(!d.mask || d.mask_ld == 0 || d.mask_ld >= d.n_experts, "mask: the row stride is shorter than a row");
  need(d.score == TH_SOFTMAX || d.score == TH_SIGMOID, "score must be TH_SOFTMAX or TH_SIGMOID");
  need(d.nodes >= 1 && d.n_experts % d.nodes == 0, "the experts must lie on the nodes equally");
  need(d.top_nodes >= 1 && d.top_nodes <= d.nodes, "top_nodes must be in [1, nodes]");
  need(d.choices <= d.n_experts / d.nodes * d.top_nodes, "choices must not exceed the experts of top_nodes nodes");
  need(d.node_best == 1 || d.node_best == 2, "node_best must be 1 or 2");
  need(d.scale > 0 && d.scale < INFINITY, "scale must be a positive number");
  RouteArgs a{};
  a.logits = d.logits;
  a.mask = d.mask;
  a.T = d.tokens;
  a.ld = d.ld;
  a.mask_ld = d.mask_ld;
  a.E = d.n_experts;
  a.k = d.choices;
  a.normalize = d.normalize;
  a.bias = d.bias;
  a.scale = d.scale;
  a.sigmoid = d.score == TH_SIGMOID;
  // every node kept is no choice of nodes
  a.nodes = d.top_nodes < d.nodes ? d.nodes : 1;
  a.top_nodes = d.top_nodes < d.nodes ? d.top_nodes : 1;
  a.node_best = d.node_best;
  return a;
}
void gate_forward(const th_gate_args& d, float* weights, int32_t* experts, int32_t* order, int32_t* offsets, void* work,
                  size_t work_bytes, void* stream) {
  RouteArgs a = check_gate(d);
  need(offsets && (d.tokens == 0 || (weights && experts && order)), "null output");
  need_work(work, work_bytes, gate_words(a) * 4);
  need_device();
  a.weights = weights;
  a.experts = experts;
  a.order = order;
  a.offsets = offsets;
  a.hist = (uint32_t*)work;
  HIPCHK(launch_route((MixType)d.dtype, a, (hipStream_t)stream));
}
void gate_backward(const th_gate_args& d, const float* weights, const int32_t* experts, const float* dweights,
                   void* dlogits, void* stream) {
  RouteArgs a = check_gate(d);
  need(d.tokens == 0 || (weights && experts && dweights && dlogits), "null argument");
  need_device();
  if (d.tokens == 0) return;
  a.weights = const_cast<float*>(weights);
  a.experts = const_cast<int32_t*>(experts);
  HIPCHK(launch_route_backward((MixType)d.dtype, a, dweights, dlogits, (hipStream_t)stream));
}

// ---------------------------------------------------------------- 4-bit weights
th::FourLayout check_weight4(const th_weight4* w, bool data = true) {
  need(w != nullptr, "null weight");
  mix_type(w->dtype, false);
  need(w->matrices >= 1 && w->d_in >= 1 && w->d_out >= 1, "matrices, d_in and d_out must be positive");
  need(w->d_in <= 1u << 30 && w->d_out <= 1u << 30, "d_in and d_out must be at most 2^30");
  // a workgroup of 256 threads for 16 rows, below 2^32 threads in a launch
  need(th::ceil_div(w->d_out, 16) * w->matrices < 1u << 24, "the matrices' rows in all must be below 2^28");
  need(w->group >= th::FOUR_MIN_GROUP && w->group <= th::FOUR_MAX_GROUP && (w->group & (w->group - 1)) == 0,
       "group must be a power of two from 32 to 2^30");
  if (data) {
    need(w->data != nullptr, "null data of a 4-bit weight");
    need(((uintptr_t)w->data & 15) == 0, "the data of a 4-bit weight must start on a multiple of 16 bytes");
  }
  return th::four_layout(w->d_out, w->d_in, w->group);
}
FourArgs four_of(const th_weight4* w) {
  return four_args(w->data, th::four_layout(w->d_out, w->d_in, w->group), w->matrices, w->zeros != 0);
}
// The 4-bit weight of a product, or null.
void check_operand4(const th_weight4* w, int dtype, uint32_t matrices, uint32_t d_out, uint32_t d_in) {
  check_weight4(w);
  need(w->dtype == dtype, "the 4-bit weight must have the other operands' dtype");
  need(w->matrices == matrices && w->d_out == d_out && w->d_in == d_in, "the 4-bit weight has other sizes");
}
FourRows four_rows(const th_weight4* w, int64_t ld, int64_t ld_matrix) {
  FourRows a{};
  a.four = four_of(w);
  a.ld = ld;
  a.lde = ld_matrix;
  a.E = w->matrices;
  a.rows = w->d_out;
  a.cols = w->d_in;
  a.out_cols = w->d_in;
  a.scale_cols = (uint32_t)th::ceil_div(w->d_in, w->group);
  return a;
}
// The place of its values in a workspace, as a stack of rows of a multiple of 8.
Stack values4(Pieces& p, const th_weight4* w) {
  Stack t{nullptr, 0, 0, w->matrices, w->d_in, w->d_out, nullptr};
  t.lay(p, true);
  return t;
}
void make_values4(Stack& t, const th_weight4* w, hipStream_t s) {
  t.use_copy();
  FourRows a = four_rows(w, t.ld, t.lde);
  a.out = t.copy;
  a.out_cols = t.cols;
  HIPCHK(launch_dequantize4((MixType)w->dtype, a, s));
}

// ---------------------------------------------------------------- grouped products
void check_grouped(const th_grouped* d, const th_weight4* four = nullptr) {
  need(d != nullptr, "null descriptor");
  mix_type(d->dtype, false);
  need_slots(d->tokens, d->experts, d->choices);
  need(d->d_in >= 1 && d->d_out >= 1, "d_in and d_out must be positive");
  need_rows(d->x, d->x_per_slot ? d->tokens * d->choices : d->tokens, d->ldx, d->d_in, "x");
  if (four) {
    check_operand4(four, d->dtype, d->experts, d->d_out, d->d_in);
  } else {
    need(d->w != nullptr, "null w");
    need(d->ldw >= d->d_in, "w: the row stride is shorter than a row");
  }
  need(d->tokens == 0 || (d->order && d->offsets), "null groups");
}

struct GroupedWork {
  Stack x{}, w{}, dy{};
  float* part = nullptr;  // a token's choices, to be summed
};
// y = w x of a product with 4-bit weights: whether small tiles take the codes
// themselves; larger products go through the values.
bool four_narrow(const th_grouped* d) {
  return th::four_narrow(d->tokens * d->choices, d->d_out, d->d_in, d->experts);
}
bool four_narrow(const th_lora_linear_args* d) { return th::four_narrow(d->tokens, d->d_out, d->d_in, 1); }

GroupedWork lay_grouped4(Pieces& p, const th_grouped* d, const th_weight4* w) {
  GroupedWork g;
  g.x = Stack{d->x, d->ldx, 0, 1, d->d_in, d->x_per_slot ? d->tokens * d->choices : d->tokens, nullptr};
  g.x.lay(p, !g.x.ready());
  if (!four_narrow(d)) g.w = values4(p, w);
  return g;
}
GroupedWork lay_grouped4_backward(Pieces& p, const th_grouped* d, const th_weight4* w, const void* dy, int64_t lddy) {
  GroupedWork g;
  const int64_t slots = d->tokens * d->choices;
  g.w = values4(p, w);
  g.dy = Stack{dy, lddy, 0, 1, d->d_out, slots, nullptr};
  g.dy.lay(p, d->d_out % 8 != 0);  // the workspace's size does not depend on where dy lies
  if (!d->x_per_slot && d->choices > 1) g.part = p.take<float>((uint64_t)slots * d->d_in);
  return g;
}
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

// dx of grouped products, a token's choices summed.
void grouped_dx(const th_grouped* d, const GroupedWork& g, void* dx, hipStream_t s) {
  const int64_t slots = d->tokens * d->choices;
  const bool summed = !d->x_per_slot && d->choices > 1;
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
  HIPCHK(launch_mat((MixType)d->dtype, m, 1, s));
  if (summed) HIPCHK(launch_sum_choices((MixType)d->dtype, g.part, dx, d->tokens, d->choices, d->d_in, s));
}

// ---------------------------------------------------------------- shared projection with adapters
void check_lora(const th_lora_linear_args* d, const th_weight4* four = nullptr) {
  need(d != nullptr, "null descriptor");
  mix_type(d->dtype, false);
  need_slots(d->tokens, d->adapters, d->choices);
  need(d->d_in >= 1 && d->d_out >= 1, "d_in and d_out must be positive");
  need(d->rank >= 1 && d->rank <= th::MIX_MAX_RANK, "rank must be in [1, " + std::to_string(th::MIX_MAX_RANK) + "]");
  need_rows(d->x, d->tokens, d->ldx, d->d_in, "x");
  need((four || d->weight) && d->a && d->b, "null weight or adapter");
  if (four) check_operand4(four, d->dtype, 1, d->d_out, d->d_in);
  else need(d->ldw >= d->d_in, "weight: the row stride is shorter than a row");
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
LoraWork lay_forward(Pieces& p, const th_lora_linear_args* d, bool keep_u, const th_weight4* four = nullptr) {
  LoraWork w = lay_groups(p, d, scans(d, keep_u));
  const bool pad = four || th::pad_operands(d->tokens, d->d_in);
  for (Stack* t : {&w.x, &w.a}) t->lay(p, pad && !t->ready());
  if (!four) w.weight.lay(p, pad && !w.weight.ready());
  else if (!four_narrow(d)) w.weight = values4(p, four);
  if (!keep_u) w.u = p.take<float>((uint64_t)d->tokens * d->choices * padded_rank(d->rank));
  return w;
}
LoraWork lay_backward(Pieces& p, const th_lora_linear_args* d, const void* dy, int64_t lddy,
                      const th_weight4* four = nullptr) {
  LoraWork w = lay_groups(p, d);
  w.dy = Stack{dy, lddy, 0, 1, d->d_out, d->tokens, nullptr};
  w.x.lay(p, !w.x.ready());
  if (four) w.weight = values4(p, four);
  else w.weight.lay(p, !w.weight.ready());
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

// ---------------------------------------------------------------- the shared projection, its weight of 16 or 4 bits
void lora_workspace(const th_lora_linear_args* d, const th_weight4* four, int keep_u, size_t* bytes) {
  need(bytes != nullptr, "null output");
  check_lora(d, four);
  Pieces p(nullptr);
  lay_forward(p, d, keep_u != 0, four);
  *bytes = p.used();
}
void lora_forward(const th_lora_linear_args* d, const th_weight4* four, void* y, int64_t ldy, float* u, void* work,
                  size_t work_bytes, void* stream) {
  check_lora(d, four);
  need_rows(y, d->tokens, ldy, d->d_out, "y");
  Pieces p(work);
  LoraWork w = lay_forward(p, d, u != nullptr, four);
  need_work(work, work_bytes, p.used());
  need_device();
  if (d->tokens == 0) return;
  const hipStream_t s = (hipStream_t)stream;
  float* low = u ? u : w.u;
  if (!scans(d, u != nullptr)) make_groups(d, w, s);
  const bool codes = four && four_narrow(d);  // the product takes the codes, with no values of them in memory
  Stack none{};
  make_copies(w.x, four ? none : w.weight, w.a, s);
  if (four && !codes) make_values4(w.weight, four, s);
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
  m.aligned = w.x.ready() && (codes || w.weight.ready());
  set_lowrank(m, d, low, d->b, d->ldb, d->ldb_adapter);
  if (codes) {
    m.four = four_of(four);
    HIPCHK(launch_narrow4((MixType)d->dtype, m, s));
  } else {
    HIPCHK(launch_mat((MixType)d->dtype, m, 0, s));
  }
}
void lora_backward_workspace(const th_lora_linear_args* d, const th_weight4* four, size_t* bytes) {
  need(bytes != nullptr, "null output");
  check_lora(d, four);
  Pieces p(nullptr);
  lay_backward(p, d, nullptr, d->d_out, four);
  *bytes = p.used();
}
void lora_backward(const th_lora_linear_args* d, const th_weight4* four, const float* u, const void* dy, int64_t lddy,
                   void* dx, void* da, void* db, float* dgate, void* work, size_t work_bytes, void* stream) {
  check_lora(d, four);
  need_rows(dy, d->tokens, lddy, d->d_out, "dy");
  need(d->tokens == 0 || u != nullptr || !(db || dgate), "null u");
  Pieces p(work);
  LoraWork w = lay_backward(p, d, dy, lddy, four);
  need_work(work, work_bytes, p.used());
  need_device();
  const hipStream_t s = (hipStream_t)stream;
  const MixType type = (MixType)d->dtype;
  const uint32_t ru = padded_rank(d->rank);
  const int64_t slots = d->tokens * d->choices;
  make_groups(d, w, s);
  Stack none{};
  if (slots) make_copies(w.x, four ? none : w.weight, w.dy, s);
  if (slots && (dx || da || dgate)) {
    TransposePair t{};
    t.p[0] = TransposeArgs{d->b, w.bt, d->ldb, d->ldb_adapter, d->adapters, d->d_out, d->rank, w.dy.padded()};
    if (dx) t.p[1] = TransposeArgs{d->a, w.at, d->lda, d->lda_adapter, d->adapters, d->rank, d->d_in, d->rank};
    HIPCHK(launch_transpose(t, s));
    const uint32_t n = w.dy.padded();
    shrink(d, w, w.dy, Stack{w.bt, n, (int64_t)n * d->rank, d->adapters, n, d->rank, nullptr}, w.v, s);
  }
  if (slots && dx) {
    if (four) make_values4(w.weight, four, s);
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
    const th_gate_args d = plain_gate(dtype, logits, ld, tokens, n_experts, mask, mask_ld, choices, normalize);
    gate_forward(d, weights, experts, order, offsets, work, work_bytes, stream);
  });
}
int th_gate_workspace(const th_gate_args* d, size_t* bytes) {
  return guarded([&] {
    need(d != nullptr, "null descriptor");
    need(bytes != nullptr, "null output");
    *bytes = gate_words(check_gate(*d)) * 4;
  });
}
int th_gate(const th_gate_args* d, float* weights, int32_t* experts, int32_t* order, int32_t* offsets, void* work,
            size_t work_bytes, void* stream) {
  return guarded([&] {
    need(d != nullptr, "null descriptor");
    gate_forward(*d, weights, experts, order, offsets, work, work_bytes, stream);
  });
}

int th_route_backward(int dtype, const void* logits, int64_t ld, int64_t tokens, uint32_t n_experts,
                      const uint8_t* mask, int64_t mask_ld, uint32_t choices, int normalize, const float* weights,
                      const int32_t* experts, const float* dweights, void* dlogits, void* stream) {
  return guarded([&] {
    const th_gate_args d = plain_gate(dtype, logits, ld, tokens, n_experts, mask, mask_ld, choices, normalize);
    gate_backward(d, weights, experts, dweights, dlogits, stream);
  });
}
int th_gate_backward(const th_gate_args* d, const float* weights, const int32_t* experts, const float* dweights,
                     void* dlogits, void* stream) {
  return guarded([&] {
    need(d != nullptr, "null descriptor");
    gate_backward(*d, weights, experts, dweights, dlogits, stream);
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
    Pieces p(work);
    GroupedWork g = lay_grouped_backward(p, d, dy, lddy);
    need_work(work, work_bytes, p.used());
    need_device();
    const hipStream_t s = (hipStream_t)stream;
    const int64_t slots = d->tokens * d->choices;
    if (slots) make_copies(g.x, g.w, g.dy, s);
    if (dx) grouped_dx(d, g, dx, s);
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
  return guarded([&] { lora_workspace(d, nullptr, keep_u, bytes); });
}
int th_lora_linear4_workspace(const th_lora_linear_args* d, const th_weight4* w, int keep_u, size_t* bytes) {
  return guarded([&] {
    check_weight4(w);
    lora_workspace(d, w, keep_u, bytes);
  });
}

int th_lora_linear(const th_lora_linear_args* d, void* y, int64_t ldy, float* u, void* work, size_t work_bytes,
                   void* stream) {
  return guarded([&] { lora_forward(d, nullptr, y, ldy, u, work, work_bytes, stream); });
}
int th_lora_linear4(const th_lora_linear_args* d, const th_weight4* w, void* y, int64_t ldy, float* u, void* work,
                    size_t work_bytes, void* stream) {
  return guarded([&] {
    check_weight4(w);
    lora_forward(d, w, y, ldy, u, work, work_bytes, stream);
  });
}

int th_lora_linear_backward_workspace(const th_lora_linear_args* d, size_t* bytes) {
  return guarded([&] { lora_backward_workspace(d, nullptr, bytes); });
}
int th_lora_linear4_backward_workspace(const th_lora_linear_args* d, const th_weight4* w, size_t* bytes) {
  return guarded([&] {
    check_weight4(w);
    lora_backward_workspace(d, w, bytes);
  });
}

int th_lora_linear_backward(const th_lora_linear_args* d, const float* u, const void* dy, int64_t lddy, void* dx,
                            void* da, void* db, float* dgate, void* work, size_t work_bytes, void* stream) {
  return guarded([&] { lora_backward(d, nullptr, u, dy, lddy, dx, da, db, dgate, work, work_bytes, stream); });
}
int th_lora_linear4_backward(const th_lora_linear_args* d, const th_weight4* w, const float* u, const void* dy,
                             int64_t lddy, void* dx, void* da, void* db, float* dgate, void* work, size_t work_bytes,
                             void* stream) {
  return guarded([&] {
    check_weight4(w);
    lora_backward(d, w, u, dy, lddy, dx, da, db, dgate, work, work_bytes, stream);
  });
}

// ---------------------------------------------------------------- 4-bit weights
int th_weight4_bytes(const th_weight4* w, size_t* bytes) {
  return guarded([&] {
    need(bytes != nullptr, "null output");
    const th::FourLayout f = check_weight4(w, false);
    *bytes = th::four_bytes(f, w->matrices, w->zeros != 0);
  });
}

int th_pack4(const th_weight4* w, const uint8_t* codes, int64_t ldc, int64_t ldc_matrix, const void* scales,
             const uint8_t* zeros, void* stream) {
  return guarded([&] {
    check_weight4(w);
    need_rows(codes, w->d_out, ldc, w->d_in, "codes");
    need(scales != nullptr, "null scales");
    need((zeros != nullptr) == (w->zeros != 0), "zeros are given exactly for a weight that has them");
    need_device();
    FourRows a = four_rows(w, ldc, ldc_matrix);
    a.in = codes;
    a.scales = scales;
    a.zeros = zeros;
    HIPCHK(launch_pack4((MixType)w->dtype, a, (hipStream_t)stream));
  });
}

int th_quantize4(const th_weight4* w, const void* values, int64_t ldv, int64_t ldv_matrix, void* stream) {
  return guarded([&] {
    check_weight4(w);
    need_rows(values, w->d_out, ldv, w->d_in, "values");
    need_device();
    FourRows a = four_rows(w, ldv, ldv_matrix);
    a.in = values;
    HIPCHK(launch_quantize4((MixType)w->dtype, a, (hipStream_t)stream));
  });
}

int th_dequantize4(const th_weight4* w, void* values, int64_t ldv, int64_t ldv_matrix, void* stream) {
  return guarded([&] {
    check_weight4(w);
    need_rows(values, w->d_out, ldv, w->d_in, "values");
    need_device();
    FourRows a = four_rows(w, ldv, ldv_matrix);
    a.out = values;
    HIPCHK(launch_dequantize4((MixType)w->dtype, a, (hipStream_t)stream));
  });
}

int th_grouped_matmul4_workspace(const th_grouped* d, const th_weight4* w, size_t* bytes) {
  return guarded([&] {
    need(bytes != nullptr, "null output");
    check_weight4(w);
    check_grouped(d, w);
    Pieces p(nullptr);
    lay_grouped4(p, d, w);
    *bytes = p.used();
  });
}

int th_grouped_matmul4(const th_grouped* d, const th_weight4* w, void* y, int64_t ldy, void* work, size_t work_bytes,
                       void* stream) {
  return guarded([&] {
    check_weight4(w);
    check_grouped(d, w);
    const int64_t slots = d->tokens * d->choices;
    need_rows(y, slots, ldy, d->d_out, "y");
    Pieces p(work);
    GroupedWork g = lay_grouped4(p, d, w);
    need_work(work, work_bytes, p.used());
    need_device();
    if (slots == 0) return;
    const hipStream_t s = (hipStream_t)stream;
    const bool codes = four_narrow(d);
    Stack none{};
    make_copies(g.x, none, none, s);
    if (!codes) make_values4(g.w, w, s);
    MatArgs m{};
    m.x = g.x.p;
    m.ldx = g.x.ld;
    m.w = g.w.p;
    m.ldw = g.w.ld;
    m.ldwe = g.w.lde;
    m.y = y;
    m.ldy = ldy;
    m.order = d->order;
    m.offsets = d->offsets;
    m.rows = slots;
    m.n = d->d_out;
    m.k = g.x.cols;
    m.E = d->experts;
    m.div = d->x_per_slot ? 1 : d->choices;
    m.aligned = 1;
    if (codes) {
      m.four = four_of(w);
      HIPCHK(launch_narrow4((MixType)d->dtype, m, s));
    } else {
      HIPCHK(launch_mat((MixType)d->dtype, m, 0, s));
    }
  });
}

int th_grouped_matmul4_backward_workspace(const th_grouped* d, const th_weight4* w, size_t* bytes) {
  return guarded([&] {
    need(bytes != nullptr, "null output");
    check_weight4(w);
    check_grouped(d, w);
    Pieces p(nullptr);
    lay_grouped4_backward(p, d, w, nullptr, d->d_out);
    *bytes = p.used();
  });
}

int th_grouped_matmul4_backward(const th_grouped* d, const th_weight4* w, const void* dy, int64_t lddy, void* dx,
                                void* work, size_t work_bytes, void* stream) {
  return guarded([&] {
    check_weight4(w);
    check_grouped(d, w);
    const int64_t slots = d->tokens * d->choices;
    need_rows(dy, slots, lddy, d->d_out, "dy");
    need(slots == 0 || dx != nullptr, "null dx");
    Pieces p(work);
    GroupedWork g = lay_grouped4_backward(p, d, w, dy, lddy);
    need_work(work, work_bytes, p.used());
    need_device();
    if (slots == 0) return;
    const hipStream_t s = (hipStream_t)stream;
    Stack none{};
    make_copies(none, none, g.dy, s);
    make_values4(g.w, w, s);
    grouped_dx(d, g, dx, s);
  });
}

}  // extern "C"
