// One training pass of SBLocal attention through the C ABI, on the models, under a number of schedules: the results have
// to be those of the definition in 64 bits, and the same bits under every schedule.
//   driver DATA_SEED B H T S D W SMS SCHEDULES FIRST_SCHEDULE [lengths, repeated over the batch]
// prints "errors out .. dq .. dk .. dv .." and "N schedules, M differ"; exits with 3 where something cannot go on.
#include "device_model.h"

#include <random>
#include <vector>

#include "sblocal_b200.h"

extern "C" {
cudaError_t cudaGetDevice(int* device) {
  *device = 0;
  return cudaSuccess;
}
cudaError_t cudaDeviceGetAttribute(int* value, cudaDeviceAttr, int) {
  *value = model::sms;
  return cudaSuccess;
}
const char* cudaGetErrorString(cudaError_t) { return "an error"; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* dst, const void* src, size_t n, cudaMemcpyKind, cudaStream_t) {
  memcpy(dst, src, n);
  return cudaSuccess;
}
}

struct Tensor {                       // (B, rows, H, D) bf16
  int rows, H, D;
  uint16_t* data;
  size_t size;
  Tensor(int B, int rows, int H, int D) : rows(rows), H(H), D(D), size((size_t)B * rows * H * D) {
    data = static_cast<uint16_t*>(aligned_alloc(256, (2 * size + 255) / 256 * 256));
    clear();
  }
  void clear() { memset(data, 0xff, 2 * size); }
  size_t at(int b, int r, int h) const { return (((size_t)b * rows + r) * H + h) * D; }
  double get(size_t i) const { return __uint_as_float((uint32_t)data[i] << 16); }
  int64_t batch() const { return (int64_t)rows * H * D; }
};
struct Doubles {
  std::vector<double> v;
  explicit Doubles(const Tensor& t) : v(t.size, 0.0) {}
  double error(const Tensor& t) const {
    double e = 0, n = 0;
    for (size_t i = 0; i < v.size(); ++i) {
      e += (t.get(i) - v[i]) * (t.get(i) - v[i]);
      n += v[i] * v[i];
    }
    return std::sqrt(n > 0 ? e / n : e);
  }
};

int main(int argc, char** argv) {
  if (argc < 11) return 2;
  int a = 1;
  auto next = [&] { return atoi(argv[a++]); };
  const int data_seed = next(), B = next(), H = next(), T = next(), S = next(), D = next(), w = next();
  model::sms = next();
  const int schedules = next(), first_schedule = next(), m = 4 * D, r = 2 * D;
  std::vector<int64_t> given, lengths;
  while (a < argc) given.push_back(next());
  for (int b = 0; b < B && !given.empty(); ++b) lengths.push_back(given[b % given.size()]);

  std::mt19937 g(data_seed);
  std::normal_distribution<float> normal;
  Tensor q(B, T, H, D), k(B, S, H, D), v(B, S, H, D), dout(B, T, H, D), out(B, T, H, D), dq(B, T, H, D), dk(B, S, H, D),
      dv(B, S, H, D);
  auto fill = [&](Tensor& t, float scale) {
    for (size_t i = 0; i < t.size; ++i) t.data[i] = as<uint16_t>(__float2bfloat16(normal(g) * scale));
  };
  const float scale = std::pow((float)D, -0.25f);
  fill(q, scale);
  fill(k, scale);
  fill(v, 1.f);
  fill(dout, 1.f);
  std::vector<float> W((size_t)r * D);
  for (auto& x : W) x = normal(g);

  SblParams p{};
  p.dtype = SBL_DTYPE_BF16;
  p.B = B; p.H = H; p.T = T; p.S = S; p.E = p.D = D; p.r = r; p.w = w;
  p.softmax_temp = 1.f / std::sqrt((float)D);
  p.q = q.data; p.q_stride_b = q.batch(); p.q_stride_t = (int64_t)H * D; p.q_stride_h = D;
  p.k = k.data; p.k_stride_b = k.batch(); p.k_stride_s = (int64_t)H * D; p.k_stride_h = D;
  p.v = v.data; p.v_stride_b = v.batch(); p.v_stride_s = (int64_t)H * D; p.v_stride_h = D;
  p.out = out.data; p.o_stride_b = out.batch(); p.o_stride_t = (int64_t)H * D; p.o_stride_h = D;
  p.W = W.data();
  p.key_lengths = lengths.empty() ? nullptr : lengths.data();
  p.S_total = p.sum_hi = S;

  // the definition: every weight of every row
  Doubles ro(out), rq(dq), rk(dk), rv(dv);
  const double tau = p.softmax_temp;
  for (int b = 0; b < B; ++b)
    for (int h = 0; h < H; ++h) {
      const int len = lengths.empty() ? S : (int)std::max<int64_t>(0, std::min<int64_t>(lengths[b], S));
      if (len == 0) continue;
      auto features = [&](const Tensor& x, int rows) {
        std::vector<double> f((size_t)rows * m);
        for (int i = 0; i < rows; ++i) {
          const size_t at = x.at(b, i, h);
          double sq = 0;
          for (int e = 0; e < D; ++e) sq += x.get(at + e) * x.get(at + e);
          for (int j = 0; j < r; ++j) {
            double u = 0;
            for (int e = 0; e < D; ++e) u += (double)W[(size_t)j * D + e] * x.get(at + e);
            u *= std::sqrt(tau);
            f[(size_t)i * m + j] = std::exp(u - tau * sq / 2 - std::log((double)m) / 2);
            f[(size_t)i * m + r + j] = std::exp(-u - tau * sq / 2 - std::log((double)m) / 2);
          }
        }
        return f;
      };
      auto through = [&](double* dx, const Tensor& x, size_t at, const double* f, const double* df) {
        double sum = 0;
        for (int j = 0; j < m; ++j) sum += f[j] * df[j];
        for (int j = 0; j < r; ++j) {
          const double z = std::sqrt(tau) * (f[j] * df[j] - f[r + j] * df[r + j]);
          for (int e = 0; e < D; ++e) dx[e] += z * W[(size_t)j * D + e];
        }
        for (int e = 0; e < D; ++e) dx[e] -= tau * x.get(at + e) * sum;
      };
      const std::vector<double> fq = features(q, T), fk = features(k, S);
      std::vector<double> dfk((size_t)S * m, 0.0), weight(len);
      for (int i = 0; i < T; ++i) {
        const size_t qi = q.at(b, i, h);
        auto near = [&](int s) { return s >= i - w / 2 && s <= i - w / 2 + w - 1; };
        double total = 0, delta = 0;
        for (int s = 0; s < len; ++s) {
          double x = 0;
          if (near(s)) {
            for (int e = 0; e < D; ++e) x += q.get(qi + e) * k.get(k.at(b, s, h) + e);
            x = std::exp(tau * x);
          } else {
            for (int f = 0; f < m; ++f) x += fq[(size_t)i * m + f] * fk[(size_t)s * m + f];
          }
          weight[s] = x;
          total += x;
        }
        for (int s = 0; s < len; ++s)
          for (int e = 0; e < D; ++e) ro.v[qi + e] += (weight[s] / total) * v.get(v.at(b, s, h) + e);
        for (int e = 0; e < D; ++e) delta += ro.v[qi + e] * dout.get(qi + e);
        std::vector<double> dfq(m, 0.0);
        for (int s = 0; s < len; ++s) {
          const size_t ks = k.at(b, s, h);
          double pull = -delta;
          for (int e = 0; e < D; ++e) {
            pull += dout.get(qi + e) * v.get(ks + e);
            rv.v[ks + e] += weight[s] / total * dout.get(qi + e);
          }
          if (near(s)) {
            for (int e = 0; e < D; ++e) {
              rq.v[qi + e] += tau * weight[s] / total * pull * k.get(ks + e);
              rk.v[ks + e] += tau * weight[s] / total * pull * q.get(qi + e);
            }
          } else {
            for (int f = 0; f < m; ++f) {
              dfq[f] += pull / total * fk[(size_t)s * m + f];
              dfk[(size_t)s * m + f] += pull / total * fq[(size_t)i * m + f];
            }
          }
        }
        through(&rq.v[qi], q, qi, &fq[(size_t)i * m], dfq.data());
      }
      for (int s = 0; s < len; ++s)
        through(&rk.v[k.at(b, s, h)], k, k.at(b, s, h), &fk[(size_t)s * m], &dfk[(size_t)s * m]);
    }

  size_t forward_bytes = 0, backward_bytes = 0;
  if (sbl_workspace_bytes(&p, &forward_bytes) || sbl_backward_workspace_bytes(&p, &backward_bytes)) {
    printf("refused: %s\n", sbl_last_error());
    return 2;
  }
  auto* forward_ws = static_cast<uint8_t*>(aligned_alloc(256, (forward_bytes + 255) / 256 * 256));
  auto* backward_ws = static_cast<uint8_t*>(aligned_alloc(256, (backward_bytes + 255) / 256 * 256));
  std::vector<float> stats(2 * (size_t)B * H * T + (size_t)B * H);
  std::vector<uint16_t> first;
  int differ = 0;
  double worst[4] = {};
  for (int n = 0; n < schedules; ++n) {
    model::seed(first_schedule + n);
    memset(forward_ws, 0xff, forward_bytes);
    memset(backward_ws, 0xff, backward_bytes);
    std::fill(stats.begin(), stats.end(), NAN);
    for (Tensor* t : {&out, &dq, &dk, &dv}) t->clear();
    int rc = sbl_forward_train(&p, forward_ws, forward_bytes, stats.data(), nullptr);
    SblGrads grads{};
    grads.dout = dout.data; grads.do_stride_b = dout.batch(); grads.do_stride_t = (int64_t)H * D; grads.do_stride_h = D;
    grads.row_stats = stats.data();
    grads.dq = dq.data; grads.dq_stride_b = dq.batch(); grads.dq_stride_t = (int64_t)H * D; grads.dq_stride_h = D;
    grads.dk = dk.data; grads.dk_stride_b = dk.batch(); grads.dk_stride_s = (int64_t)H * D; grads.dk_stride_h = D;
    grads.dv = dv.data; grads.dv_stride_b = dv.batch(); grads.dv_stride_s = (int64_t)H * D; grads.dv_stride_h = D;
    if (rc == SBL_OK) rc = sbl_backward(&p, &grads, backward_ws, backward_bytes, nullptr);
    if (rc != SBL_OK) {
      printf("refused: %s\n", sbl_last_error());
      return 2;
    }
    std::vector<uint16_t> bits;
    for (const Tensor* t : {&out, &dq, &dk, &dv}) bits.insert(bits.end(), t->data, t->data + t->size);
    if (n == 0) first = bits;
    differ += bits != first;
    const double e[4] = {ro.error(out), rq.error(dq), rk.error(dk), rv.error(dv)};
    for (int i = 0; i < 4; ++i) worst[i] = e[i] <= worst[i] ? worst[i] : e[i];   // (a NaN stays)
  }
  printf("errors out %.3e dq %.3e dk %.3e dv %.3e\n%d schedules, %d differ\n", worst[0], worst[1], worst[2], worst[3],
         schedules, differ);
  return 0;
}
