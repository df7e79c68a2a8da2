// A batch over a KV cache in pages through hip_ops.hpp, beside the same sequences one by one over contiguous caches: prompts of
// --prompt tokens (less 13 for each later sequence), then --steps generated tokens, for --batch sequences.  Flags as of
// op_test_attention_layer (--head_num --kv_head_num --dtype --is_neox --theta --max_seq_len), --page_size, --eight 1: an 8-bit
// cache.  16 bits: rotated q and rows read back are the contiguous path's bit for bit, attention within --tol of it; 8 bits:
// rows within half a step of e4m3, attention within 16 times that.
#include <algorithm>

#include "op_test_common.hpp"

using namespace llm_simple_amd;

int main(int argc, char **argv) {
  const int H = optest::flag_int(argc, argv, "head_num", 28), Hkv = optest::flag_int(argc, argv, "kv_head_num", 4);
  const int batch = optest::flag_int(argc, argv, "batch", 3), prompt = optest::flag_int(argc, argv, "prompt", 100);
  const int steps = optest::flag_int(argc, argv, "steps", 4), max_seq_len = optest::flag_int(argc, argv, "max_seq_len", 512);
  const int page_size = optest::flag_int(argc, argv, "page_size", 16);
  const bool is_neox = optest::flag_int(argc, argv, "is_neox", 1) != 0, eight = optest::flag_int(argc, argv, "eight", 0) != 0;
  const float theta = std::atof(optest::flag(argc, argv, "theta", "1000000").c_str());
  const DataType dt = optest::parse_dtype(optest::flag(argc, argv, "dtype", "bf16")), cache_dt = eight ? DT_FLOAT8_E4M3 : dt;
  // two roundings each of the weights and the results, of values up to about 4 (16 bits)
  const float tol = std::atof(optest::flag(argc, argv, "tol", dt == DT_BFLOAT16 ? "6.25e-2" : "7.8125e-3").c_str());
  std::printf("paged op test {batch=%d,prompt=%d,steps=%d,head_num=%d,kv_head_num=%d,page_size=%d,%s%s}\n", batch, prompt, steps, H, Hkv, page_size,
              dt == DT_BFLOAT16 ? "bf16" : "fp16", eight ? ",8 bits" : "");
  if (prompt - 13 * (batch - 1) < 1 || prompt + steps > max_seq_len || H % Hkv != 0) {
    std::printf("sizes do not fit\n");
    return 2;
  }
  if (llmhip_device_count() < 1) {
    std::printf("no GPU\n");
    return 3;
  }
  auto table = MakeFreqCIS(128, max_seq_len, theta, dt)->to(DEV_GPU);
  const int pps = (max_seq_len + page_size - 1) / page_size, num_pages = pps * batch;
  const size_t page_bytes = llmhip_paged_page_bytes(page_size, Hkv, 128, cache_dt);
  auto k_pages = Tensor::MakeGPUTensor(page_bytes * num_pages, DT_UINT8), v_pages = Tensor::MakeGPUTensor(page_bytes * num_pages, DT_UINT8);
  std::vector<int32_t> pages(num_pages);
  for (int i = 0; i < num_pages; ++i) pages[i] = (i * 7 + 3) % num_pages;  // (a permutation where 7 does not divide their number)
  if (num_pages % 7 == 0)
    for (int i = 0; i < num_pages; ++i) pages[i] = num_pages - 1 - i;
  auto d_pages = optest::to_gpu(pages.data(), pages.size(), DT_INT32);
  const size_t row = (size_t)Hkv * 128;
  std::vector<std::shared_ptr<Tensor>> kc, vc;  // contiguous
  for (int b = 0; b < batch; ++b) {
    kc.push_back(Tensor::MakeGPUTensor(row * max_seq_len, dt));
    vc.push_back(Tensor::MakeGPUTensor(row * max_seq_len, dt));
  }
  gpuStream_t stream = nullptr;
  CHECK_LLMHIP(llmhip_stream_create(&stream));

  std::vector<int32_t> lens(batch, 0);
  size_t differ = 0;
  double worst = 0.0, worst_row = 0.0;
  for (int step = 0; step <= steps; ++step) {
    std::vector<int32_t> starts(batch + 1, 0);
    int most = 0, longest = 0;
    for (int b = 0; b < batch; ++b) {
      const int fresh = step == 0 ? prompt - 13 * b : 1;
      starts[b + 1] = starts[b] + fresh;
      lens[b] += fresh;
      most = std::max(most, fresh);
      longest = std::max(longest, (int)lens[b]);
    }
    const int tokens = starts[batch];
    const size_t nq = (size_t)tokens * H * 128, nk = (size_t)tokens * row;
    auto q = optest::to_gpu(optest::normal_bits(100 + step, nq, dt).data(), nq, dt);
    auto k = optest::to_gpu(optest::normal_bits(200 + step, nk, dt).data(), nk, dt);
    auto v = optest::to_gpu(optest::normal_bits(300 + step, nk, dt).data(), nk, dt);
    auto q_rot = Tensor::MakeGPUTensor(nq, dt), out = Tensor::MakeGPUTensor(nq, dt), back_k = Tensor::MakeGPUTensor(nk, dt), back_v = Tensor::MakeGPUTensor(nk, dt);
    auto q_one = Tensor::MakeGPUTensor(nq, dt), out_one = Tensor::MakeGPUTensor(nq, dt);
    auto d_starts = optest::to_gpu(starts.data(), starts.size(), DT_INT32), d_lens = optest::to_gpu(lens.data(), lens.size(), DT_INT32);
    const int *t = static_cast<const int *>(d_pages->data_ptr), *qs = static_cast<const int *>(d_starts->data_ptr), *kl = static_cast<const int *>(d_lens->data_ptr);
    const size_t ws_bytes = llmhip_paged_flash_attn_workspace_bytes(tokens, batch, most, longest, 0, 0, H / Hkv, Hkv, 128);
    auto ws = Tensor::MakeGPUTensor(ws_bytes + 16, DT_UINT8);
    hip_paged_rope_kv_append_layer(q_rot->data_ptr, k_pages->data_ptr, v_pages->data_ptr, t, qs, kl, table->data_ptr, q->data_ptr, k->data_ptr, v->data_ptr,
                                   tokens, batch, pps, num_pages, page_size, (int64_t)page_bytes, max_seq_len, H, Hkv, 128, is_neox, cache_dt, dt, stream);
    hip_paged_flash_attn_gqa_layer(out->data_ptr, q_rot->data_ptr, k_pages->data_ptr, v_pages->data_ptr, t, qs, kl, ws->data_ptr, ws_bytes, tokens, batch, most,
                                   longest, pps, num_pages, page_size, (int64_t)page_bytes, 0, 0, H / Hkv, Hkv, 128, cache_dt, dt, stream);
    hip_paged_kv_read_layer(back_k->data_ptr, back_v->data_ptr, k_pages->data_ptr, v_pages->data_ptr, t, qs, kl, tokens, batch, pps, num_pages, page_size,
                            (int64_t)page_bytes, Hkv, 128, cache_dt, dt, stream);
    auto at = [](const std::shared_ptr<Tensor> &x, size_t elements) { return static_cast<char *>(x->data_ptr) + 2 * elements; };
    for (int b = 0; b < batch; ++b) {
      const int fresh = starts[b + 1] - starts[b], past = lens[b] - fresh;
      const size_t q0 = (size_t)starts[b] * H * 128, k0 = starts[b] * row;
      hip_rope_kv_append_layer(at(q_one, q0), kc[b]->data_ptr, vc[b]->data_ptr, table->data_ptr, at(q, q0), at(k, k0), at(v, k0), past, fresh, H, Hkv, 128,
                               is_neox, dt, stream);
      hip_flash_attn_gqa_layer(at(out_one, q0), at(q_one, q0), kc[b]->data_ptr, vc[b]->data_ptr, fresh, lens[b], past, H / Hkv, Hkv, 128, dt, stream);
    }
    CHECK_LLMHIP(llmhip_stream_sync(stream));
    auto host = [&](const std::shared_ptr<Tensor> &x, size_t n) {
      auto h = x->to(DEV_CPU);
      std::vector<float> f(n);
      orc_widen_array(f.data(), static_cast<const uint16_t *>(h->data_ptr), (int64_t)n, dt);
      return f;
    };
    const auto a = host(q_rot, nq), c = host(q_one, nq), o = host(out, nq), o1 = host(out_one, nq), bk = host(back_k, nk), bv = host(back_v, nk);
    for (size_t i = 0; i < nq; ++i) {
      differ += a[i] != c[i];
      worst = std::max(worst, (double)std::fabs(o[i] - o1[i]));
    }
    for (int b = 0; b < batch; ++b) {
      const size_t n = (starts[b + 1] - starts[b]) * row, first = (lens[b] - (starts[b + 1] - starts[b])) * row, k0 = starts[b] * row;
      const auto ck = host(kc[b], row * max_seq_len), cv = host(vc[b], row * max_seq_len);
      for (size_t i = 0; i < n; ++i) {
        // (half a step of e4m3 is 2^-4 of a value, or 2^-10 of the row's power of two, itself at most 2^-7 of its largest magnitude, here below 8)
        const double ek = std::fabs(bk[k0 + i] - ck[first + i]), ev = std::fabs(bv[k0 + i] - cv[first + i]);
        const double mk = eight ? std::fabs(ck[first + i]) / 16 + 8.0 / (1 << 17) : 0.0, mv = eight ? std::fabs(cv[first + i]) / 16 + 8.0 / (1 << 17) : 0.0;
        differ += ek > mk;
        differ += ev > mv;
        worst_row = std::max(worst_row, std::max(ek, ev));
      }
    }
  }
  std::printf("%zu elements differ; attention off by %.3g at most, rows by %.3g\n", differ, worst, worst_row);
  for (auto *x : {&kc, &vc}) x->clear();
  CHECK_LLMHIP(llmhip_stream_destroy(stream));
  const bool ok = differ == 0 && worst <= (eight ? 16 * tol : tol) && hip_last_status() == 0;
  std::printf(ok ? "PASS\n" : "FAIL\n");
  return ok ? 0 : 1;
}
