// layers.cc -- the layer calls (include/hexir_b200/layers.h): argument
// checks, kernel choice and launches of the kernels in kernels/layers.cu.

#include "hexir_b200/layers.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <limits>

#include "../kernels/launch_abi.h"
#include "../kernels/layers_abi.h"
#include "cuda_driver.h"
#include "kernel_lib.h"

extern "C" {
extern const unsigned char hexir_layers_cubin_begin[];
}

namespace hexir {

namespace {

// How a norm's rows lie: in whole 16-byte packs; in packs that every tensor's
// row cuts at the same place; or anyhow.
enum Layout { kWhole, kShifted, kAny };

// The norm kernels: the name's end in layer_norm.cu, threads per row (blocks
// have 256 at least, several rows where a row has less), elements per thread,
// layout, and the gradient's rows of the ring.  A row runs the first kernel of
// its layout that holds it.
struct NormShape {
  const char *name;
  uint32_t threads, elements;
  Layout layout;
  uint32_t depth;
  uint32_t rows() const { return threads < 256 ? 256 / threads : 1; }
  uint32_t block() const { return rows() * threads; }
};
constexpr int kMaxShapes = 21;
// By the kind of type: 16-bit, f32, f64.
constexpr NormShape kNorm[3][kMaxShapes] = {
    {{"w32x8", 32, 8, kWhole, 0},
     {"w32x16", 32, 16, kWhole, 0},
     {"w32x24", 32, 24, kWhole, 0},
     {"w32x32", 32, 32, kWhole, 0},
     {"w128x16", 128, 16, kWhole, 0},
     {"w256x16", 256, 16, kWhole, 0},
     {"w256x24", 256, 24, kWhole, 0},
     {"w256x32", 256, 32, kWhole, 0},
     {"w512x32", 512, 32, kWhole, 0},
     {"h32x8", 32, 8, kShifted, 0},
     {"h32x16", 32, 16, kShifted, 0},
     {"h64x16", 64, 16, kShifted, 0},
     {"h128x16", 128, 16, kShifted, 0},
     {"h256x16", 256, 16, kShifted, 0},
     {"h320x16", 320, 16, kShifted, 0},
     {"h384x16", 384, 16, kShifted, 0},
     {"h512x16", 512, 16, kShifted, 0},
     {"h1024x16", 1024, 16, kShifted, 0},
     {"s32x32", 32, 32, kAny, 0},
     {"s256x16", 256, 16, kAny, 0},
     {"s512x32", 512, 32, kAny, 0}},
    {{"w32x8", 32, 8, kWhole, 0},
     {"w32x16", 32, 16, kWhole, 0},
     {"w32x32", 32, 32, kWhole, 0},
     {"w128x16", 128, 16, kWhole, 0},
     {"w256x16", 256, 16, kWhole, 0},
     {"w512x16", 512, 16, kWhole, 0},
     {"w1024x16", 1024, 16, kWhole, 0},
     {"h256x8", 256, 8, kShifted, 0},
     {"h320x8", 320, 8, kShifted, 0},
     {"h512x8", 512, 8, kShifted, 0},
     {"h640x8", 640, 8, kShifted, 0},
     {"h512x16", 512, 16, kShifted, 0},
     {"h1024x16", 1024, 16, kShifted, 0},
     {"s32x8", 32, 8, kAny, 0},
     {"s32x16", 32, 16, kAny, 0},
     {"s128x8", 128, 8, kAny, 0},
     {"s320x8", 320, 8, kAny, 0},
     {"s512x8", 512, 8, kAny, 0},
     {"s512x16", 512, 16, kAny, 0},
     {"s1024x16", 1024, 16, kAny, 0}},
    {{"w32x8", 32, 8, kWhole, 0},
     {"w64x8", 64, 8, kWhole, 0},
     {"w128x8", 128, 8, kWhole, 0},
     {"w256x8", 256, 8, kWhole, 0},
     {"w512x8", 512, 8, kWhole, 0},
     {"w512x16", 512, 16, kWhole, 0},
     {"s32x8", 32, 8, kAny, 0},
     {"s64x8", 64, 8, kAny, 0},
     {"s192x8", 192, 8, kAny, 0},
     {"s256x8", 256, 8, kAny, 0},
     {"s512x8", 512, 8, kAny, 0},
     {"s512x16", 512, 16, kAny, 0}}};
constexpr NormShape kNormGrad[3][kMaxShapes] = {
    {{"w32x8", 32, 8, kWhole, 6},
     {"w32x16", 32, 16, kWhole, 4},
     {"w64x16", 64, 16, kWhole, 4},
     {"w128x16", 128, 16, kWhole, 3},
     {"w256x16", 256, 16, kWhole, 3},
     {"w384x16", 384, 16, kWhole, 4},
     {"w512x16", 512, 16, kWhole, 3},
     {"w1024x16", 1024, 16, kWhole, 2},
     {"h32x8", 32, 8, kShifted, 6},
     {"h32x16", 32, 16, kShifted, 4},
     {"h64x16", 64, 16, kShifted, 4},
     {"h128x16", 128, 16, kShifted, 4},
     {"h256x16", 256, 16, kShifted, 4},
     {"h384x16", 384, 16, kShifted, 4},
     {"h512x16", 512, 16, kShifted, 3},
     {"h1024x16", 1024, 16, kShifted, 2},
     {"s32x32", 32, 32, kAny, 2},
     {"s1024x16", 1024, 16, kAny, 2}},
    {{"w32x8", 32, 8, kWhole, 4},
     {"w64x8", 64, 8, kWhole, 4},
     {"w128x8", 128, 8, kWhole, 4},
     {"w256x8", 256, 8, kWhole, 4},
     {"w512x8", 512, 8, kWhole, 3},
     {"w512x16", 512, 16, kWhole, 2},
     {"h256x8", 256, 8, kShifted, 4},
     {"h320x8", 320, 8, kShifted, 4},
     {"h512x8", 512, 8, kShifted, 3},
     {"h640x8", 640, 8, kShifted, 2},
     {"h512x16", 512, 16, kShifted, 2},
     {"s64x8", 64, 8, kAny, 4},
     {"s128x8", 128, 8, kAny, 4},
     {"s320x8", 320, 8, kAny, 4},
     {"s512x8", 512, 8, kAny, 3},
     {"s512x16", 512, 16, kAny, 2}},
    {{"w32x8", 32, 8, kWhole, 3},
     {"w64x8", 64, 8, kWhole, 3},
     {"w128x8", 128, 8, kWhole, 3},
     {"w256x8", 256, 8, kWhole, 3},
     {"w512x8", 512, 8, kWhole, 2},
     {"s32x8", 32, 8, kAny, 3},
     {"s64x8", 64, 8, kAny, 3},
     {"s192x8", 192, 8, kAny, 3},
     {"s256x8", 256, 8, kAny, 3},
     {"s512x8", 512, 8, kAny, 2}}};

int kind_of(uint32_t dtype) {
  return dtype == HEXIR_DTYPE_F64 ? 2 : (dtype == HEXIR_DTYPE_F32 ? 1 : 0);
}

Layout norm_layout(uint32_t size, uint32_t cols, bool parameters16,
                   std::initializer_list<std::pair<const void *, uint64_t>> tensors) {
  bool whole = cols * static_cast<uint64_t>(size) % 16 == 0 && parameters16;
  // Shifted packs against single elements: f32 16384 x 4097 137 against 171 us,
  // 4099 x 1025 11.9 against 14.6, 8192 x 257 8.2 against 6.5; f64 4099 x 1025
  // 16.9 against 13.7 (its single elements are wide enough).
  bool same = size == 2 || (size == 4 && cols >= 1024);
  const auto first = *tensors.begin();
  auto phase = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16; };
  for (const auto &t : tensors) {
    if (!t.first)
      continue;
    whole = whole && phase(t.first) == 0 && t.second * size % 16 == 0;
    same = same && phase(t.first) == phase(first.first) &&
           t.second * size % 16 == first.second * size % 16;
  }
  return whole ? kWhole : (same ? kShifted : kAny);
}

// -1: a longer row than any kernel holds.
int norm_shape(const NormShape (&shapes)[kMaxShapes], uint32_t cols, uint32_t size,
               Layout layout) {
  // A shifted row may begin and end inside a pack.
  const uint64_t need = cols + (layout == kShifted ? 16ull / size - 1 : 0ull);
  for (int s = 0; s < kMaxShapes && shapes[s].name; ++s)
    if (shapes[s].layout == layout && need <= shapes[s].threads * shapes[s].elements)
      return s;
  return -1;
}

// Persistent blocks; those of a shifted layout stay a multiple of 8 rows
// apart, so that all rows of a thread are cut at the same place.
uint64_t norm_blocks(const NormShape &shape, Layout layout, uint64_t rows,
                     uint64_t resident) {
  const uint64_t blocks = (rows + shape.rows() - 1) / shape.rows();
  if (blocks <= resident)
    return blocks;
  return layout == kShifted ? std::max<uint64_t>(8, resident / 8 * 8) : resident;
}

// Blocks of a kernel that fit an SM, by its registers and shared memory.
uint32_t blocks_per_sm(uint32_t registers, uint32_t threads, uint32_t smem) {
  const uint32_t per_warp = (registers + 7) / 8 * 8 * 32;
  const uint32_t warps = 65536u / std::max(per_warp, 1u) / 4 * 4;
  uint32_t n = std::min(2048u / threads, warps / ((threads + 31) / 32));
  n = std::min(n, 227u * 1024u / (smem + 9216u));
  return std::max(n, 1u);
}

const char *const kDtypeName[4] = {"f64", "f32", "bf16", "f16"};
constexpr uint32_t kDtypeSize[4] = {8, 4, 2, 2};

}  // namespace

struct LayersLib {
  CUmodule module = nullptr;
  CUdeviceptr error_word = 0;
  // By HEXIR_PRODUCT_*; skinny is the forward's only.
  CUfunction pair[3] = {}, single[3] = {}, guarded[3] = {}, skinny = nullptr;
  // By dtype.
  struct Sized {
    CUfunction fn = nullptr;
    int registers = 0;
  };
  Sized norm[4][kMaxShapes] = {}, norm_grad[4][kMaxShapes] = {};
  CUfunction norm_wide[4] = {}, norm_grad_wide[4] = {},
             norm_grad_columns[4] = {}, norm_grad_join[4] = {};
  Sized output_grad[4] = {};
  CUfunction output_grad_join[4] = {};
};

CUdeviceptr layers_error_word(const LayersLib *lib) { return lib->error_word; }

namespace {

// The most dynamic shared memory a product kernel is launched with, beside up
// to 5 KiB of its own.
constexpr uint32_t kSmemLimit = 221u * 1024u;
// The same of the norm kernels, beside up to 8 KiB of their own.
constexpr uint32_t kNormSmemLimit = 218u * 1024u;

LayersLib *layers_library(DeviceState *dev, std::string *error) {
  std::lock_guard<std::mutex> lock(dev->mu);
  if (dev->layers)
    return dev->layers;
  const Driver &d = driver();
  ContextGuard guard(dev->context);
  auto lib = std::make_unique<LayersLib>();
  CUresult r = d.ModuleLoadData(&lib->module, hexir_layers_cubin_begin);
  if (r != CUDA_SUCCESS) {
    fail(error, cuda_message("cuModuleLoadData", r) +
                    " (the layer kernels are built for sm_100a)");
    return nullptr;
  }
  std::string missing;
  auto get = [&](CUfunction *slot, const std::string &name) {
    if (d.ModuleGetFunction(slot, lib->module, name.c_str()) != CUDA_SUCCESS &&
        missing.empty())
      missing = name;
  };
  const char *const products[3] = {"hexir_linear_16", "hexir_linear_16_input_grad",
                                   "hexir_linear_16_weight_grad"};
  for (int i = 0; i < 3; ++i) {
    const std::string base = products[i];
    get(&lib->pair[i], base + "_pair");
    get(&lib->single[i], base + "_single");
    get(&lib->guarded[i], base + "_guarded");
  }
  get(&lib->skinny, "hexir_linear_16_skinny");
  for (int t = 0; t < 4; ++t) {
    const std::string norm = std::string("hexir_layer_norm_") + kDtypeName[t];
    const std::string grad = std::string("hexir_layer_norm_grad_") + kDtypeName[t];
    const int kind = kind_of(t);
    for (int s = 0; s < kMaxShapes; ++s) {
      if (kNorm[kind][s].name)
        get(&lib->norm[t][s].fn, norm + "_" + kNorm[kind][s].name);
      if (kNormGrad[kind][s].name)
        get(&lib->norm_grad[t][s].fn, grad + "_" + kNormGrad[kind][s].name);
    }
    get(&lib->norm_wide[t], norm + "_wide");
    get(&lib->norm_grad_wide[t], grad + "_wide");
    get(&lib->norm_grad_columns[t], grad + "_columns");
    get(&lib->norm_grad_join[t], grad + "_join");
    if (t >= static_cast<int>(HEXIR_DTYPE_BF16)) {
      const std::string out = std::string("hexir_linear_output_grad_") + kDtypeName[t];
      get(&lib->output_grad[t].fn, out);
      get(&lib->output_grad_join[t], out + "_join");
    }
  }
  if (!missing.empty()) {
    d.ModuleUnload(lib->module);
    fail(error, "the layer kernels lack " + missing);
    return nullptr;
  }
  size_t bytes = 0;
  r = d.ModuleGetGlobal(&lib->error_word, &bytes, lib->module,
                        "hexir_device_error_word");
  for (int i = 0; i < 3 && r == CUDA_SUCCESS; ++i)
    for (CUfunction fn : {lib->pair[i], lib->single[i], lib->guarded[i]})
      if (r == CUDA_SUCCESS)
        r = d.FuncSetAttribute(fn, CU_FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES,
                               kSmemLimit);
  if (r == CUDA_SUCCESS)
    r = d.FuncSetAttribute(lib->skinny,
                           CU_FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES,
                           kSmemLimit);
  for (int t = HEXIR_DTYPE_BF16; t < 4 && r == CUDA_SUCCESS; ++t)
    r = d.FuncGetAttribute(&lib->output_grad[t].registers, CU_FUNC_ATTRIBUTE_NUM_REGS,
                           lib->output_grad[t].fn);
  for (int t = 0; t < 4; ++t)
    for (int s = 0; s < kMaxShapes; ++s)
      for (LayersLib::Sized *k : {&lib->norm[t][s], &lib->norm_grad[t][s]}) {
        if (!k->fn || r != CUDA_SUCCESS)
          continue;
        r = d.FuncGetAttribute(&k->registers, CU_FUNC_ATTRIBUTE_NUM_REGS, k->fn);
        if (r == CUDA_SUCCESS)
          r = d.FuncSetAttribute(k->fn,
                                 CU_FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES,
                                 kNormSmemLimit);
      }
  if (r != CUDA_SUCCESS) {
    d.ModuleUnload(lib->module);
    fail(error, cuda_message("layer kernels setup", r));
    return nullptr;
  }
  dev->layers = lib.release();
  return dev->layers;
}

struct Call {
  DeviceState *dev = nullptr;
  LayersLib *lib = nullptr;
  std::string error;
  bool open(int ordinal) {
    dev = device_state(ordinal, &error);
    lib = dev ? layers_library(dev, &error) : nullptr;
    return lib != nullptr;
  }
  hexir_status_t finish(hexir_status_t status) {
    if (status != HEXIR_OK)
      set_last_error(error.empty() ? hexir_status_string(status) : error);
    return status;
  }
  hexir_status_t refuse(std::string message,
                        hexir_status_t status = HEXIR_ERROR_INVALID_ARGUMENT) {
    error = std::move(message);
    return finish(status);
  }
};

uint32_t ceil_div(uint64_t a, uint64_t b) {
  return static_cast<uint32_t>((a + b - 1) / b);
}

bool off(const void *p, uint32_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes != 0;
}

// Rows that start on 16-byte boundaries: what TMA and 16-byte accesses need.
bool rows16(const void *p, uint64_t ld, uint32_t size) {
  return !off(p, 16) && ld * size % 16 == 0;
}

// One tensor argument: its row stride made explicit, and checked.
struct Tensor {
  const char *name;
  const void *p;
  uint64_t *ld;
  uint64_t rows, cols;
};

// Empty if fine.  Element alignment matters: a kernel's access off it faults.
std::string check_tensors(const char *op, uint32_t size,
                          std::initializer_list<Tensor> tensors) {
  for (const Tensor &t : tensors) {
    if (*t.ld == 0)
      *t.ld = t.cols;
    if (t.p && off(t.p, size))
      return std::string(op) + ": " + t.name + " is not aligned to its elements";
    if (*t.ld < t.cols)
      return std::string(op) + ": the row stride of " + t.name +
             " is smaller than its row";
    // Byte offsets stay within 63 bits.
    if (t.rows && *t.ld > (std::numeric_limits<uint64_t>::max() >> 4) / t.rows)
      return std::string(op) + ": " + t.name + " is too large";
    if (t.rows <= 1)  // one row has no stride: leave it aligned
      *t.ld = (t.cols + 15) / 16 * 16;
  }
  return std::string();
}

bool linear_activation(uint32_t a) {
  return a == HEXIR_ACTIVATION_NONE || a == HEXIR_ACTIVATION_RELU ||
         (a >= HEXIR_ACTIVATION_LEAKY_RELU && a <= HEXIR_ACTIVATION_MISH &&
          a != HEXIR_ACTIVATION_SOFTMAX);
}

// What the linear calls share.
std::string check_linear(const char *op, uint32_t dtype, uint32_t activation,
                         uint32_t flags, hexir_status_t *status) {
  *status = HEXIR_ERROR_INVALID_ARGUMENT;
  if (dtype == HEXIR_DTYPE_F64 || dtype == HEXIR_DTYPE_F32) {
    *status = HEXIR_ERROR_UNIMPLEMENTED;
    return std::string(op) + ": bf16 or f16 only (f64: hexir_cuda_matmul_add_f64)";
  }
  if (dtype > HEXIR_DTYPE_F16)
    return std::string(op) + ": unknown dtype " + std::to_string(dtype);
  if (!linear_activation(activation))
    return std::string(op) + ": no such elementwise activation " +
           std::to_string(activation);
  const uint32_t forces = flags & 0xF00u;
  if ((flags & ~0xFFFF0F00u) || (forces & (forces - 1)))
    return std::string(op) + ": unknown flags";
  const uint32_t split = flags >> 16 & 0xFFu;
  const uint32_t tile = flags >> 24 << 4;
  if (tile && !((forces == HEXIR_LINEAR_FORCE_PAIR && (tile == 256 || tile == 128)) ||
                (forces == HEXIR_LINEAR_FORCE_SINGLE && (tile == 128 || tile == 64))))
    return std::string(op) + ": no such tile of the kernel asked for";
  if (split && split != 1 && split != 2 && split != 4 && split != 8)
    return std::string(op) + ": the split is 1, 2, 4 or 8";
  return std::string();
}

// ------------------------------------------------------------ the products

enum ProductVariant { kPair = 1, kSingle = 2, kSkinny = 3, kGuardedLoads = 4 };

struct ProductPlan {
  uint32_t variant = 0;
  uint32_t tile_n = 0, split = 1, stages = 0;
  uint32_t tiles_m = 0, tiles_n = 0, full_tiles = 0;
  uint32_t tmem_cols = 0, ring = 0, smem = 0;
  std::string refusal;  // a forced kernel that cannot run this
};

uint32_t stage_bytes(uint32_t tile_n) {
  return HEXIR_PRODUCT_BM * 128u + tile_n * 128u;
}

// Tiles that CTA pairs take whole.  Those of a last turn that fills at most half
// of the pairs are cut into halves of 128 columns, which take 0.7 of its time.
uint64_t pair_full_tiles(uint64_t tiles, uint32_t tile_n, uint64_t pairs) {
  const uint64_t over = tiles % pairs;
  return tile_n == 256 && tiles > pairs && 2 * over <= pairs ? tiles - over : tiles;
}

// Modelled microseconds of a product: a base, and per wave of tiles (of pairs,
// or of clusters of `split` CTAs, resident at once) a fixed part and a part per
// 64 of the summed index.  Fitted on B200 to 27 shapes of 65-8192 rows and
// 256-8192 columns and depths, each in its three forms and every tile and
// split (within 6-15 % of the measured times; what it chose took 0.6 % more
// than the best, on average).  An epilogue that reads or stores through shared
// memory (slots) costs more per tile and leaves one single CTA per SM.
double modelled_us(uint32_t variant, uint32_t tile_n, uint32_t split, uint32_t rows,
                   uint32_t cols, uint32_t k_tiles, bool slots, uint32_t guarded,
                   uint32_t sms) {
  struct Cost {
    double k_tile, wave, base;
  };
  static constexpr Cost kPairCost[2][2] = {{{0.219, 1.9, 4.1}, {0.312, 3.2, 4.4}},
                                           {{0.230, 3.1, 4.4}, {0.322, 5.2, 5.1}}};
  static constexpr Cost kSingleCost[2][4] = {
      {{0.224, 4.0, 0.8}, {0.227, 4.9, 1.1}, {0.264, 5.3, 1.9}, {0.381, 6.4, 3.4}},
      {{0.272, 5.5, 1.0}, {0.283, 6.1, 1.3}, {0.311, 7.4, 0.6}, {0.631, 6.7, 2.8}}};
  const uint32_t wide = tile_n >= (variant == kPair ? 256u : 128u) ? 1 : 0;
  if (variant == kPair) {
    const Cost &c = kPairCost[slots][wide];
    const uint64_t tiles =
        static_cast<uint64_t>(ceil_div(rows, 256)) * ceil_div(cols, tile_n);
    const uint64_t pairs = sms / 2, whole = pair_full_tiles(tiles, tile_n, pairs);
    const Cost &half = kPairCost[slots][0];
    return c.base + (whole + pairs - 1) / pairs * (k_tiles * c.k_tile + c.wave) +
           (whole < tiles ? k_tiles * half.k_tile + half.wave : 0.0);
  }
  const Cost &c = kSingleCost[wide][split >= 8 ? 3 : split / 2];
  const uint64_t ctas =
      static_cast<uint64_t>(ceil_div(rows, 128)) * ceil_div(cols, tile_n) * split;
  // Clusters are placed inside a GPC: 32 of 4 CTAs and 16 of 8 are resident.
  const uint64_t resident = split >= 4 ? sms * 7 / 8 / split * split : sms;
  const uint64_t waves = (ctas + resident - 1) / std::max<uint64_t>(resident, 1);
  const double k_tile = c.k_tile + 0.23 * guarded;  // operands of guarded loads
  return c.base + waves * (ceil_div(k_tiles, split) * k_tile + c.wave);
}

// slots: the epilogue reads or stores through shared memory.
// guarded: operands that TMA cannot describe.
ProductPlan plan_product(uint32_t op, uint32_t m, uint32_t n, uint32_t k,
                         uint32_t guarded, bool slots, uint32_t flags, uint32_t sms) {
  // out [rows][cols], summed over depth.
  const uint32_t rows = op == HEXIR_PRODUCT_WEIGHT_GRAD ? k : m;
  const uint32_t cols = op == HEXIR_PRODUCT_INPUT_GRAD ? k : n;
  const uint32_t depth = op == HEXIR_PRODUCT_FORWARD      ? k
                         : op == HEXIR_PRODUCT_INPUT_GRAD ? n
                                                          : m;
  const uint32_t k_tiles = ceil_div(depth, HEXIR_PRODUCT_BK);
  const uint32_t forced_split = flags >> 16 & 0xFFu;
  const uint32_t forced_tile = flags >> 24 << 4;
  ProductPlan p;
  const bool tma = !guarded && depth > 0;
  const bool skinny = tma && op == HEXIR_PRODUCT_FORWARD && m <= 64;
  if (flags & HEXIR_LINEAR_FORCE_GUARDED) {
    p.variant = kGuardedLoads;
  } else if (flags & HEXIR_LINEAR_FORCE_SKINNY) {
    p.variant = kSkinny;
    if (!skinny)
      p.refusal = "the skinny kernel needs aligned rows, the forward and m <= 64";
  } else if (flags & (HEXIR_LINEAR_FORCE_PAIR | HEXIR_LINEAR_FORCE_SINGLE)) {
    p.variant = flags & HEXIR_LINEAR_FORCE_PAIR ? kPair : kSingle;
    if (!tma)
      p.refusal = "the TMA kernels need aligned rows and a sum that is not empty";
  } else if (!tma) {
    p.variant = kGuardedLoads;
  } else if (skinny) {
    p.variant = kSkinny;
  }
  if (!p.refusal.empty())
    return p;

  if (p.variant == kSkinny) {
    const uint32_t max_split = std::max<uint32_t>(
        1, k_tiles >= 32 ? 8 : (k_tiles >= 16 ? 4 : (k_tiles >= 8 ? 2 : 1)));
    p.tile_n = (std::max<uint32_t>(m, 1) + 15) / 16 * 16;
    p.tiles_m = ceil_div(n, HEXIR_PRODUCT_BM);
    p.tiles_n = 1;
    // The weight stream is the cost: CTAs for every SM, two per SM.
    while (p.split < max_split && p.tiles_m * p.split * 2 <= 2 * sms)
      p.split *= 2;
    p.tmem_cols = p.tile_n <= 32 ? 32 : 64;
  } else {
    // The kernel, tile and split of the least modelled time.
    double best = 0;
    uint32_t best_variant = 0;
    auto consider = [&](uint32_t variant, uint32_t tile_n, uint32_t split) {
      if ((p.variant && p.variant != variant) || (forced_tile && tile_n != forced_tile) ||
          (forced_split && split != forced_split))
        return;
      const double t =
          modelled_us(variant, tile_n, split, rows, cols, k_tiles, slots, guarded, sms);
      if (best_variant == 0 || t < best) {
        best = t;
        best_variant = variant;
        p.tile_n = tile_n;
        p.split = split;
      }
    };
    for (uint32_t tile_n : {256u, 128u})
      consider(kPair, tile_n, 1);
    const uint32_t single = p.variant == kGuardedLoads ? kGuardedLoads : kSingle;
    for (uint32_t tile_n : {128u, 64u})
      for (uint32_t split = 1; split <= 8; split *= 2)
        if (split == 1 || split * 2 <= k_tiles || split == forced_split)
          if (tile_n == 128 || single == kSingle)
            consider(single, tile_n, split);
    if (!best_variant) {
      p.refusal = "CTA pairs do not split the sum";
      return p;
    }
    p.variant = best_variant;
    if (p.variant == kPair) {
      p.tiles_m = ceil_div(rows, 2 * HEXIR_PRODUCT_BM);
      p.tiles_n = ceil_div(cols, p.tile_n);
      p.full_tiles = static_cast<uint32_t>(pair_full_tiles(
          static_cast<uint64_t>(p.tiles_m) * p.tiles_n, p.tile_n, sms / 2));
      p.smem = HEXIR_PAIR_SMEM_BYTES;
      return p;
    }
    p.tiles_m = ceil_div(rows, HEXIR_PRODUCT_BM);
    p.tiles_n = ceil_div(cols, p.tile_n);
    p.tmem_cols = p.tile_n;
  }
  if (forced_split)
    p.split = forced_split;
  // One CTA per SM with a deep ring, or, where there are more and their
  // epilogues need no slots, two whose main loops and epilogues overlap (the
  // same shared memory for guarded loads, of which one fits by its registers).
  const uint64_t ctas = static_cast<uint64_t>(p.tiles_m) * p.tiles_n * p.split;
  const uint32_t epilogue =
      slots && p.variant != kSkinny
          ? HEXIR_EPILOGUE_BYTES(HEXIR_SINGLE_EPILOGUE_WARPS) : 0u;
  const bool two = p.variant == kSkinny || (ctas > sms && !epilogue);
  const uint32_t room = (two ? 108u : 216u) * 1024u - epilogue;
  p.stages = std::min<uint32_t>(HEXIR_SINGLE_MAX_STAGES, room / stage_bytes(p.tile_n));
  // The ring also holds a split tile's sums.
  p.ring = std::max<uint32_t>(p.stages * stage_bytes(p.tile_n),
                              p.split > 1 ? HEXIR_PRODUCT_BM * p.tile_n * 4u : 0u);
  // Shared memory: at least what keeps the TMEM columns of the CTAs that fit
  // an SM within its 512 (a CTA that waits for columns while it holds a place
  // in a cluster could wait on a cluster that waits for it): 227 KiB / 512
  // columns = 454 bytes per column.
  p.smem = std::max<uint32_t>(p.ring + epilogue, p.tmem_cols * 512u) + 1024u;
  return p;
}

struct Operand {
  const void *p;
  uint64_t ld;
  bool mn;             // MN-major: rows along the summed index
  uint32_t side, box;  // extent of the tile's side, and of a box along it
};

CUresult encode(CUtensorMap *map, const Operand &o, uint32_t depth, bool f16) {
  const cuuint64_t dims[2] = {o.mn ? o.side : depth, o.mn ? depth : o.side};
  const cuuint64_t strides[1] = {o.ld * 2};
  const cuuint32_t box[2] = {64, o.mn ? 64u : o.box};
  const cuuint32_t unit[2] = {1, 1};
  return driver().TensorMapEncodeTiled(
      map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
      2, const_cast<void *>(o.p), dims, strides, box, unit,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// out[rows][cols] = a . b over depth with op's epilogue (args: everything but
// the tiling).  a and b as the product has them: x and w, dz and w, x and dz.
hexir_status_t launch_product(Call &call, uint32_t op, uint32_t m, uint32_t n,
                              uint32_t k, uint32_t flags,
                              hexir_product_args_t &args, CUstream stream) {
  if (args.rows == 0 || args.cols == 0)
    return HEXIR_OK;
  const bool a_mn = op == HEXIR_PRODUCT_WEIGHT_GRAD;
  const bool b_mn = op != HEXIR_PRODUCT_INPUT_GRAD;
  const bool aligned_a = rows16(args.a, args.lda, 2) && args.lda < 1ull << 39;
  const bool aligned_b = rows16(args.b, args.ldb, 2) && args.ldb < 1ull << 39;
  const uint32_t sms = static_cast<uint32_t>(std::max(call.dev->sm_count, 2));
  args.vec = rows16(args.out, args.ldo, 2) &&
             (!args.preact_out || rows16(args.preact_out, args.ldp, 2)) &&
             (!args.residual || rows16(args.residual, args.ldr, 2)) &&
             (!args.slope_at || rows16(args.slope_at, args.lds, 2));
  if (args.vec && !off(args.out, 32) && args.ldo % 16 == 0 &&
      (!args.preact_out || (!off(args.preact_out, 32) && args.ldp % 16 == 0)))
    args.vec = 2;
  const bool slots = !args.vec || args.residual || args.slope_at;
  const ProductPlan p = plan_product(
      op, m, n, k, (aligned_a ? 0u : 1u) + (aligned_b ? 0u : 1u), slots, flags, sms);
  if (!p.refusal.empty())
    return fail(&call.error, "linear: " + p.refusal, HEXIR_ERROR_INVALID_ARGUMENT);
  const uint64_t tiles = static_cast<uint64_t>(p.tiles_m) * p.tiles_n;
  if (tiles * p.split > 0x7FFFFFFFull)
    return fail(&call.error, "linear: too many tiles", HEXIR_ERROR_INVALID_ARGUMENT);

  args.tiles_m = p.tiles_m;
  args.tiles_n = p.tiles_n;
  args.group_m = std::min<uint32_t>(8, p.tiles_m);
  args.full_tiles = p.full_tiles;
  args.tile_n = p.tile_n;
  args.k_tiles = ceil_div(args.depth, HEXIR_PRODUCT_BK);
  args.split = p.split;
  args.stages = p.stages;
  args.tmem_cols = p.tmem_cols;
  args.ring_bytes = p.ring;
  args.timeout_ns = kWaitTimeoutNs;

  const unsigned grid = static_cast<unsigned>(tiles * p.split);
  Operand a = {args.a, args.lda, a_mn, args.rows, HEXIR_PRODUCT_BM};
  Operand b = {args.b, args.ldb, b_mn, args.cols,
               p.variant == kPair ? 64u : p.tile_n};
  if (p.variant == kSkinny) {
    // The transposed product: the weight's columns are the tile's rows.
    const Operand x = {args.a, args.lda, false, args.rows, p.tile_n};
    a = {args.b, args.ldb, true, args.cols, HEXIR_PRODUCT_BM};
    b = x;
  }
  // Guarded: by TMA what TMA can describe (forced: neither).
  if (p.variant != kGuardedLoads)
    args.tma_operands = 3;
  else if (!(flags & HEXIR_LINEAR_FORCE_GUARDED) && args.depth)
    args.tma_operands = (aligned_a ? 1u : 0u) | (aligned_b ? 2u : 0u);
  CUtensorMap map_a, map_b;
  std::memset(&map_a, 0, sizeof(map_a));
  std::memset(&map_b, 0, sizeof(map_b));
  CUresult r = CUDA_SUCCESS;
  if (args.tma_operands & 1u)
    r = encode(&map_a, a, args.depth, args.is_f16 != 0);
  if (r == CUDA_SUCCESS && (args.tma_operands & 2u))
    r = encode(&map_b, b, args.depth, args.is_f16 != 0);
  if (r != CUDA_SUCCESS)
    return fail(&call.error, cuda_message("cuTensorMapEncodeTiled", r));
  void *params[] = {&map_a, &map_b, &args};
  if (p.variant == kPair) {
    const uint64_t pairs = std::min<uint64_t>(tiles, sms / 2);
    return launch_after(call.lib->pair[op], static_cast<unsigned>(2 * pairs), 1,
                        HEXIR_PAIR_THREADS, stream, params,
                        "launch hexir_linear_16 pair", &call.error, p.smem);
  }
  CUfunction fn = p.variant == kSkinny         ? call.lib->skinny
                  : p.variant == kGuardedLoads ? call.lib->guarded[op]
                                               : call.lib->single[op];
  const char *what = p.variant == kSkinny         ? "launch hexir_linear_16 skinny"
                     : p.variant == kGuardedLoads ? "launch hexir_linear_16 guarded"
                                                  : "launch hexir_linear_16 single";
  return launch_after(fn, grid, 1,
                      p.variant == kGuardedLoads ? HEXIR_GUARDED_THREADS
                                                    : HEXIR_SINGLE_THREADS,
                      stream, params, what,
                      &call.error, p.smem, p.split);
}

// TMA coordinates are signed 32-bit numbers.
bool extents_ok(uint32_t m, uint32_t n, uint32_t k) {
  constexpr uint32_t kMost = 0x7FFFFF00u;
  return m <= kMost && n <= kMost && k <= kMost;
}

// ----------------------------------------------------------- the norms

constexpr uint32_t kSumsPerColumn = 640;  // hexir_cuda_grad_workspace

}  // namespace

}  // namespace hexir

using namespace hexir;

extern "C" uint64_t hexir_cuda_grad_workspace(uint32_t cols, uint32_t dtype) {
  return static_cast<uint64_t>(kSumsPerColumn) * cols *
         (dtype == HEXIR_DTYPE_F64 ? 8 : 4);
}

extern "C" hexir_status_t hexir_cuda_linear_plan(
    int ordinal, uint32_t op, uint32_t m, uint32_t n, uint32_t k, int aligned,
    uint32_t flags, uint32_t *variant, uint32_t *tile_n, uint32_t *split) {
  Call call;
  hexir_status_t status;
  const bool reads =
      op != HEXIR_PRODUCT_WEIGHT_GRAD && !(flags & HEXIR_LINEAR_PLAN_PLAIN);
  flags &= ~HEXIR_LINEAR_PLAN_PLAIN;
  std::string bad = check_linear("linear_plan", HEXIR_DTYPE_BF16, 0, flags, &status);
  if (op > HEXIR_PRODUCT_WEIGHT_GRAD || !bad.empty())
    return call.refuse(bad.empty() ? "linear_plan: op is 0, 1 or 2" : bad);
  if (!extents_ok(m, n, k))
    return call.refuse("linear_plan: m, n or k is too large");
  if (aligned & ~15)
    return call.refuse("linear_plan: unknown bits in aligned");
  auto is_aligned = [&](int part) {
    return (aligned & (HEXIR_LINEAR_ALIGNED_ALL | part)) != 0;
  };
  // Without a GPU: B200's 148 SMs.
  std::string error;
  DeviceState *dev = device_state(ordinal, &error);
  ProductPlan p;
  if ((op == HEXIR_PRODUCT_WEIGHT_GRAD ? k : m) &&
      (op == HEXIR_PRODUCT_INPUT_GRAD ? k : n))
    p = plan_product(op, m, n, k,
                     (is_aligned(HEXIR_LINEAR_ALIGNED_FIRST) ? 0u : 1u) +
                         (is_aligned(HEXIR_LINEAR_ALIGNED_SECOND) ? 0u : 1u),
                     reads || !is_aligned(HEXIR_LINEAR_ALIGNED_REST), flags,
                     dev ? std::max(dev->sm_count, 2) : 148);
  if (!p.refusal.empty())
    return call.refuse("linear_plan: " + p.refusal);
  if (variant)
    *variant = p.variant;
  if (tile_n)
    *tile_n = p.tile_n;
  if (split)
    *split = p.variant ? p.split : 0;
  return HEXIR_OK;
}

extern "C" hexir_status_t hexir_cuda_linear(int ordinal,
                                            const hexir_linear_call_t *given,
                                            void *stream) {
  Call call;
  if (!given)
    return call.refuse("linear: null call");
  hexir_linear_call_t c = *given;
  hexir_status_t status;
  std::string bad = check_linear("linear", c.dtype, c.activation, c.flags, &status);
  if (!bad.empty())
    return call.refuse(bad, status);
  const bool some = c.m && c.n;
  if (some && (!c.y || (c.k && (!c.x || !c.w))))
    return call.refuse("linear: null pointer");
  if (!extents_ok(c.m, c.n, c.k))
    return call.refuse("linear: m, n or k is too large");
  uint64_t dense = 0;
  bad = check_tensors("linear", 2,
                      {{"x", c.x, &c.ldx, c.m, c.k},
                       {"w", c.w, &c.ldw, c.k, c.n},
                       {"bias", c.bias, &dense, 1, c.n},
                       {"residual", c.residual, &c.ldr, c.m, c.n},
                       {"preact", c.preact, &c.ldp, c.m, c.n},
                       {"y", c.y, &c.ldy, c.m, c.n}});
  if (!bad.empty())
    return call.refuse(bad);
  if (!call.open(ordinal))
    return call.finish(HEXIR_ERROR_DEVICE);
  hexir_product_args_t args;
  std::memset(&args, 0, sizeof(args));
  args.a = c.x;
  args.lda = c.ldx;
  args.b = c.w;
  args.ldb = c.ldw;
  args.out = c.y;
  args.ldo = c.ldy;
  args.preact_out = c.preact;
  args.ldp = c.ldp;
  args.bias = c.bias;
  args.residual = c.residual;
  args.ldr = c.ldr;
  args.rows = c.m;
  args.cols = c.n;
  args.depth = c.k;
  args.activation = c.activation;
  args.is_f16 = c.dtype == HEXIR_DTYPE_F16;
  ContextGuard guard(call.dev->context);
  return call.finish(launch_product(call, HEXIR_PRODUCT_FORWARD, c.m, c.n, c.k,
                                    c.flags, args, static_cast<CUstream>(stream)));
}

extern "C" hexir_status_t hexir_cuda_linear_input_grad(
    int ordinal, const hexir_linear_input_grad_call_t *given, void *stream) {
  Call call;
  if (!given)
    return call.refuse("linear_input_grad: null call");
  hexir_linear_input_grad_call_t c = *given;
  hexir_status_t status;
  std::string bad =
      check_linear("linear_input_grad", c.dtype, c.activation, c.flags, &status);
  if (!bad.empty())
    return call.refuse(bad, status);
  const bool some = c.m && c.k;
  if (some && (!c.dx || (c.n && (!c.dz || !c.w)) || (c.activation && !c.preact)))
    return call.refuse("linear_input_grad: null pointer");
  if (!extents_ok(c.m, c.n, c.k))
    return call.refuse("linear_input_grad: m, n or k is too large");
  bad = check_tensors("linear_input_grad", 2,
                      {{"dz", c.dz, &c.lddz, c.m, c.n},
                       {"w", c.w, &c.ldw, c.k, c.n},
                       {"preact", c.preact, &c.ldp, c.m, c.k},
                       {"residual", c.residual, &c.ldr, c.m, c.k},
                       {"dx", c.dx, &c.lddx, c.m, c.k}});
  if (!bad.empty())
    return call.refuse(bad);
  if (!call.open(ordinal))
    return call.finish(HEXIR_ERROR_DEVICE);
  hexir_product_args_t args;
  std::memset(&args, 0, sizeof(args));
  args.a = c.dz;
  args.lda = c.lddz;
  args.b = c.w;
  args.ldb = c.ldw;
  args.out = c.dx;
  args.ldo = c.lddx;
  args.slope_at = c.activation ? c.preact : nullptr;
  args.lds = c.ldp;
  args.residual = c.residual;
  args.ldr = c.ldr;
  args.rows = c.m;
  args.cols = c.k;
  args.depth = c.n;
  args.activation = c.activation;
  args.is_f16 = c.dtype == HEXIR_DTYPE_F16;
  ContextGuard guard(call.dev->context);
  return call.finish(launch_product(call, HEXIR_PRODUCT_INPUT_GRAD, c.m, c.n, c.k,
                                    c.flags, args, static_cast<CUstream>(stream)));
}

extern "C" hexir_status_t hexir_cuda_linear_weight_grad(
    int ordinal, const hexir_linear_weight_grad_call_t *given, void *stream) {
  Call call;
  if (!given)
    return call.refuse("linear_weight_grad: null call");
  hexir_linear_weight_grad_call_t c = *given;
  hexir_status_t status;
  std::string bad = check_linear("linear_weight_grad", c.dtype, 0, c.flags, &status);
  if (!bad.empty())
    return call.refuse(bad, status);
  if (c.reserved)
    return call.refuse("linear_weight_grad: reserved is not 0");
  const bool some = c.k && c.n;
  if (some && (!c.dw || (c.m && (!c.x || !c.dz))))
    return call.refuse("linear_weight_grad: null pointer");
  if (!extents_ok(c.m, c.n, c.k))
    return call.refuse("linear_weight_grad: m, n or k is too large");
  bad = check_tensors("linear_weight_grad", 2,
                      {{"x", c.x, &c.ldx, c.m, c.k},
                       {"dz", c.dz, &c.lddz, c.m, c.n},
                       {"dw", c.dw, &c.lddw, c.k, c.n}});
  if (!bad.empty())
    return call.refuse(bad);
  if (!call.open(ordinal))
    return call.finish(HEXIR_ERROR_DEVICE);
  hexir_product_args_t args;
  std::memset(&args, 0, sizeof(args));
  args.a = c.x;
  args.lda = c.ldx;
  args.b = c.dz;
  args.ldb = c.lddz;
  args.out = c.dw;
  args.ldo = c.lddw;
  args.rows = c.k;
  args.cols = c.n;
  args.depth = c.m;
  args.is_f16 = c.dtype == HEXIR_DTYPE_F16;
  ContextGuard guard(call.dev->context);
  return call.finish(launch_product(call, HEXIR_PRODUCT_WEIGHT_GRAD, c.m, c.n, c.k,
                                    c.flags, args, static_cast<CUstream>(stream)));
}

extern "C" hexir_status_t hexir_cuda_linear_output_grad(
    int ordinal, const hexir_linear_output_grad_call_t *given, void *stream) {
  Call call;
  if (!given)
    return call.refuse("linear_output_grad: null call");
  hexir_linear_output_grad_call_t c = *given;
  hexir_status_t status;
  std::string bad = check_linear("linear_output_grad", c.dtype, c.activation, 0, &status);
  if (!bad.empty())
    return call.refuse(bad, status);
  const bool some = c.m && c.n;
  if (some && (!c.dy || (c.activation && (!c.preact || !c.dz))))
    return call.refuse("linear_output_grad: null pointer");
  bad = check_tensors("linear_output_grad", 2,
                      {{"dy", c.dy, &c.lddy, c.m, c.n},
                       {"preact", c.preact, &c.ldp, c.m, c.n},
                       {"dz", c.dz, &c.lddz, c.m, c.n}});
  if (!bad.empty())
    return call.refuse(bad);
  if (c.dbias && off(c.dbias, 2))
    return call.refuse("linear_output_grad: dbias is not aligned to its elements");
  if (c.dbias && c.n &&
      (!c.workspace || off(c.workspace, 16) ||
       c.workspace_bytes < hexir_cuda_grad_workspace(c.n, c.dtype)))
    return call.refuse("linear_output_grad: dbias needs a 16-byte aligned "
                       "workspace of hexir_cuda_grad_workspace(n, dtype) bytes");
  if (!call.open(ordinal))
    return call.finish(HEXIR_ERROR_DEVICE);
  if (!c.n || (!c.dz && !c.dbias))
    return HEXIR_OK;
  ContextGuard guard(call.dev->context);
  CUstream s = static_cast<CUstream>(stream);
  hexir_output_grad_args_t args;
  std::memset(&args, 0, sizeof(args));
  args.dy = c.dy;
  args.lddy = c.lddy;
  args.preact = c.preact;
  args.ldp = c.ldp;
  args.dz = c.dz == c.dy && !c.activation ? nullptr : c.dz;
  args.lddz = c.lddz;
  args.dbias = c.dbias;
  args.partials = c.dbias ? static_cast<float *>(c.workspace) : nullptr;
  args.m = c.m;
  args.n = c.n;
  args.activation = c.activation;
  args.vec = rows16(c.dy, c.lddy, 2) &&
             (!c.activation || rows16(c.preact, c.ldp, 2)) &&
             (!args.dz || rows16(c.dz, c.lddz, 2));
  const uint32_t gx = ceil_div(c.n, 256);
  hexir_status_t st = HEXIR_OK;
  if (c.m) {
    // One wave of blocks where the rows allow it.
    const LayersLib::Sized &kernel = call.lib->output_grad[c.dtype];
    const uint64_t resident = static_cast<uint64_t>(std::max(call.dev->sm_count, 1)) *
                              blocks_per_sm(kernel.registers, 256, 8192);
    const uint64_t want = std::max<uint64_t>(1, resident / gx);
    args.parts = static_cast<uint32_t>(std::min<uint64_t>(
        {want, static_cast<uint64_t>(ceil_div(c.m, 32)), uint64_t(kSumsPerColumn)}));
    args.rows_per_part = ceil_div(c.m, args.parts);
    args.parts = ceil_div(c.m, args.rows_per_part);
    void *params[] = {&args};
    st = launch_after(kernel.fn, gx, args.parts, 256, s, params,
                      "launch hexir_linear_output_grad", &call.error);
  }
  if (st == HEXIR_OK && c.dbias) {
    void *params[] = {&args};
    st = launch_after(call.lib->output_grad_join[c.dtype], ceil_div(c.n, 32), 1,
                      1024, s, params, "launch hexir_linear_output_grad_join",
                      &call.error);
  }
  return call.finish(st);
}

extern "C" hexir_status_t hexir_cuda_layer_norm(int ordinal,
                                                const hexir_layer_norm_call_t *given,
                                                void *stream) {
  Call call;
  if (!given)
    return call.refuse("layer_norm: null call");
  hexir_layer_norm_call_t c = *given;
  if (c.dtype > HEXIR_DTYPE_F16)
    return call.refuse("layer_norm: unknown dtype " + std::to_string(c.dtype));
  if (!c.cols)
    return call.refuse("layer_norm: a row needs at least one column");
  if (!(c.eps >= 0.0) || std::isinf(c.eps))
    return call.refuse("layer_norm: eps is not a finite number >= 0");
  if (c.rows && (!c.x || !c.y))
    return call.refuse("layer_norm: null pointer");
  const uint32_t size = kDtypeSize[c.dtype];
  const uint32_t real = c.dtype == HEXIR_DTYPE_F64 ? 8 : 4;
  uint64_t dense = 0;
  std::string bad = check_tensors("layer_norm", size,
                                  {{"x", c.x, &c.ldx, c.rows, c.cols},
                                   {"y", c.y, &c.ldy, c.rows, c.cols},
                                   {"gamma", c.gamma, &dense, 1, c.cols},
                                   {"beta", c.beta, &dense, 1, c.cols}});
  if (bad.empty())
    bad = check_tensors("layer_norm", real,
                        {{"mean", c.mean, &dense, 1, 1}, {"rstd", c.rstd, &dense, 1, 1}});
  if (!bad.empty())
    return call.refuse(bad);
  if (!call.open(ordinal))
    return call.finish(HEXIR_ERROR_DEVICE);
  if (!c.rows)
    return HEXIR_OK;
  hexir_layer_norm_args_t args;
  std::memset(&args, 0, sizeof(args));
  args.x = c.x;
  args.ldx = c.ldx;
  args.y = c.y;
  args.ldy = c.ldy;
  args.gamma = c.gamma;
  args.beta = c.beta;
  args.mean = c.mean;
  args.rstd = c.rstd;
  args.rows = c.rows;
  args.cols = c.cols;
  args.eps = c.eps;
  const Layout layout = norm_layout(size, c.cols, !off(c.gamma, 16) && !off(c.beta, 16),
                                    {{c.x, c.ldx}, {c.y, c.ldy}});
  void *params[] = {&args};
  ContextGuard guard(call.dev->context);
  CUstream s = static_cast<CUstream>(stream);
  const int kind = kind_of(c.dtype);
  const int at = norm_shape(kNorm[kind], c.cols, size, layout);
  if (at < 0)
    return call.finish(
        launch_after(call.lib->norm_wide[c.dtype],
                     static_cast<unsigned>(std::min<uint64_t>(c.rows, 1u << 24)), 1, 512,
                     s, params, "launch hexir_layer_norm wide", &call.error));
  const NormShape &shape = kNorm[kind][at];
  const LayersLib::Sized &kernel = call.lib->norm[c.dtype][at];
  // Shifted rows: gamma and beta as the rows lie.
  const uint32_t copies =
      layout == kShifted ? 2 * shape.block() * shape.elements * size : 0;
  const uint64_t resident =
      static_cast<uint64_t>(std::max(call.dev->sm_count, 1)) *
      blocks_per_sm(kernel.registers, shape.block(), copies);
  return call.finish(launch_after(
      kernel.fn, static_cast<unsigned>(norm_blocks(shape, layout, c.rows, resident)), 1,
      shape.block(), s, params, "launch hexir_layer_norm", &call.error, copies));
}

extern "C" hexir_status_t hexir_cuda_layer_norm_grad(
    int ordinal, const hexir_layer_norm_grad_call_t *given, void *stream) {
  Call call;
  if (!given)
    return call.refuse("layer_norm_grad: null call");
  hexir_layer_norm_grad_call_t c = *given;
  if (c.dtype > HEXIR_DTYPE_F16)
    return call.refuse("layer_norm_grad: unknown dtype " + std::to_string(c.dtype));
  if (!c.cols)
    return call.refuse("layer_norm_grad: a row needs at least one column");
  if (c.rows && (!c.dy || !c.x || !c.mean || !c.rstd))
    return call.refuse("layer_norm_grad: null pointer");
  const uint32_t size = kDtypeSize[c.dtype];
  const uint32_t real = c.dtype == HEXIR_DTYPE_F64 ? 8 : 4;
  uint64_t dense = 0;
  std::string bad = check_tensors("layer_norm_grad", size,
                                  {{"dy", c.dy, &c.lddy, c.rows, c.cols},
                                   {"x", c.x, &c.ldx, c.rows, c.cols},
                                   {"residual", c.residual, &c.ldr, c.rows, c.cols},
                                   {"dx", c.dx, &c.lddx, c.rows, c.cols},
                                   {"gamma", c.gamma, &dense, 1, c.cols},
                                   {"dgamma", c.dgamma, &dense, 1, c.cols},
                                   {"dbeta", c.dbeta, &dense, 1, c.cols}});
  if (bad.empty())
    bad = check_tensors("layer_norm_grad", real,
                        {{"mean", c.mean, &dense, 1, 1}, {"rstd", c.rstd, &dense, 1, 1}});
  if (!bad.empty())
    return call.refuse(bad);
  const bool sums = c.dgamma || c.dbeta;
  if (sums && (!c.workspace || off(c.workspace, 16) ||
               c.workspace_bytes < hexir_cuda_grad_workspace(c.cols, c.dtype)))
    return call.refuse("layer_norm_grad: dgamma and dbeta need a 16-byte aligned "
                       "workspace of hexir_cuda_grad_workspace(cols, dtype) bytes");
  if (!call.open(ordinal))
    return call.finish(HEXIR_ERROR_DEVICE);
  if (!sums && (!c.dx || !c.rows))
    return HEXIR_OK;
  hexir_layer_norm_grad_args_t args;
  std::memset(&args, 0, sizeof(args));
  args.dy = c.dy;
  args.lddy = c.lddy;
  args.x = c.x;
  args.ldx = c.ldx;
  args.mean = c.mean;
  args.rstd = c.rstd;
  args.gamma = c.gamma;
  args.residual = c.residual;
  args.ldr = c.ldr;
  args.dx = c.dx;
  args.lddx = c.lddx;
  args.dgamma = c.dgamma;
  args.dbeta = c.dbeta;
  args.partials = sums ? c.workspace : nullptr;
  args.rows = c.rows;
  args.cols = c.cols;
  const Layout layout = norm_layout(
      size, c.cols, !off(c.gamma, 16),
      {{c.x, c.ldx}, {c.dy, c.lddy}, {c.dx, c.lddx}, {c.residual, c.ldr}});
  ContextGuard guard(call.dev->context);
  CUstream s = static_cast<CUstream>(stream);
  const uint64_t sms = static_cast<uint64_t>(std::max(call.dev->sm_count, 1));
  const int kind = kind_of(c.dtype);
  const int at = norm_shape(kNormGrad[kind], c.cols, size, layout);
  hexir_status_t st = HEXIR_OK;
  void *params[] = {&args};
  if (c.rows && at >= 0) {
    const NormShape &shape = kNormGrad[kind][at];
    const LayersLib::Sized &kernel = call.lib->norm_grad[c.dtype][at];
    // The ring of rows; its place then holds the column sums of a block's rows.
    const uint32_t ring = shape.depth * (c.residual && c.dx ? 3 : 2) * shape.block() *
                          shape.elements * size;
    const uint64_t resident = std::min<uint64_t>(
        sms * blocks_per_sm(kernel.registers, shape.block(), ring), kSumsPerColumn / 2);
    args.parts =
        static_cast<uint32_t>(norm_blocks(shape, layout, c.rows, resident));
    st = launch_after(kernel.fn, args.parts, 1, shape.block(), s, params,
                      "launch hexir_layer_norm_grad", &call.error, ring);
  } else if (c.rows) {
    // The column sums first: dx may be dy.
    if (sums) {
      args.parts = static_cast<uint32_t>(
          std::min<uint64_t>(kSumsPerColumn / 2, (c.rows + 63) / 64));
      st = launch_after(call.lib->norm_grad_columns[c.dtype], ceil_div(c.cols, 32),
                        args.parts, 256, s, params,
                        "launch hexir_layer_norm_grad columns", &call.error);
    }
    if (st == HEXIR_OK && c.dx)
      st = launch_after(call.lib->norm_grad_wide[c.dtype],
                        static_cast<unsigned>(std::min<uint64_t>(c.rows, 1u << 24)), 1,
                        512, s, params, "launch hexir_layer_norm_grad wide",
                        &call.error);
  }
  if (st == HEXIR_OK && sums)
    st = launch_after(call.lib->norm_grad_join[c.dtype], ceil_div(c.cols, 32), 2,
                      1024, s, params, "launch hexir_layer_norm_grad_join",
                      &call.error);
  return call.finish(st);
}
