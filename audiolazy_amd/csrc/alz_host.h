// alz_host.h -- host-side copies of the host-block entry point (alz_bank_process_host, alz_api.hip): rows of a caller's array to and
// from page-locked buffers, several threads at a time.
#pragma once

#include <stdint.h>
#include <string.h>

#include <condition_variable>
#include <mutex>
#include <thread>
#include <vector>

namespace alz {

// A few threads that copy one rectangle of rows together with the thread that asks for it.  One thread moves less than the link
// does in one direction, and the pipeline copies for both.  They live for one call of the entry point (the calls that use them
// move 64 MiB and more); on a machine that gives no more threads the copies are made with fewer, down to the caller alone.
class CopyCrew {
 public:
  explicit CopyCrew(int helpers) {
    try {
      threads_.reserve((size_t)helpers);
      for (int i = 0; i < helpers; ++i) threads_.emplace_back([this, i] { serve(i + 1); });
    } catch (...) {
    }
  }
  ~CopyCrew() {
    {
      std::lock_guard<std::mutex> lock(mu_);
      stop_ = true;
    }
    start_.notify_all();
    for (std::thread &t : threads_) t.join();
  }
  CopyCrew(const CopyCrew &) = delete;
  CopyCrew &operator=(const CopyCrew &) = delete;

  // `rows` rows of `width` bytes, `dpitch` / `spitch` bytes apart
  void copy(void *dst, size_t dpitch, const void *src, size_t spitch, size_t width, size_t rows) {
    {
      std::lock_guard<std::mutex> lock(mu_);
      dst_ = (char *)dst; src_ = (const char *)src;
      dpitch_ = dpitch; spitch_ = spitch; width_ = width; rows_ = rows;
      parts_ = threads_.size() + 1;
      busy_ = threads_.size();
      ++job_;
    }
    start_.notify_all();
    part(0);
    std::unique_lock<std::mutex> lock(mu_);
    done_.wait(lock, [this] { return busy_ == 0; });
  }

 private:
  void serve(size_t index) {
    uint64_t seen = 0;
    for (;;) {
      {
        std::unique_lock<std::mutex> lock(mu_);
        start_.wait(lock, [&] { return stop_ || job_ != seen; });
        if (stop_) return;
        seen = job_;
      }
      part(index);
      std::lock_guard<std::mutex> lock(mu_);
      if (--busy_ == 0) done_.notify_one();
    }
  }
  // the index-th of parts_ shares: whole rows where there are enough of them, a range of columns otherwise
  void part(size_t index) const {
    size_t r0 = 0, r1 = rows_, c0 = 0, c1 = width_;
    if (rows_ >= parts_) {
      r0 = rows_ * index / parts_;
      r1 = rows_ * (index + 1) / parts_;
    } else {
      c0 = width_ / 64 * index / parts_ * 64;
      if (index + 1 < parts_) c1 = width_ / 64 * (index + 1) / parts_ * 64;
    }
    if (c0 >= c1) return;
    if (dpitch_ == width_ && spitch_ == width_ && c0 == 0 && c1 == width_) {
      memcpy(dst_ + r0 * width_, src_ + r0 * width_, (r1 - r0) * width_);
      return;
    }
    for (size_t r = r0; r < r1; ++r) memcpy(dst_ + r * dpitch_ + c0, src_ + r * spitch_ + c0, c1 - c0);
  }

  std::vector<std::thread> threads_;
  std::mutex mu_;
  std::condition_variable start_, done_;
  bool stop_ = false;
  uint64_t job_ = 0;
  size_t busy_ = 0, parts_ = 1;
  char *dst_ = nullptr;
  const char *src_ = nullptr;
  size_t dpitch_ = 0, spitch_ = 0, width_ = 0, rows_ = 0;
};

// The pieces of one rectangle that a buffer of `cap` bytes holds one after the other: as many whole rows as fit, or a part of a row
// that is longer than the buffer.
struct Pieces {
  size_t width, rows, cap;
  size_t row = 0, col = 0;          // where the next piece starts
  size_t p_row = 0, p_col = 0, p_rows = 0, p_width = 0;
  Pieces(size_t width_, size_t rows_, size_t cap_) : width(width_), rows(rows_), cap(cap_) {}
  bool next() {
    if (row >= rows || width == 0) return false;
    p_row = row; p_col = col;
    if (width <= cap) {
      p_width = width;
      p_rows = cap / width < rows - row ? cap / width : rows - row;
      row += p_rows;
    } else {
      p_rows = 1;
      p_width = width - col < cap ? width - col : cap;
      col += p_width;
      if (col == width) { col = 0; ++row; }
    }
    return true;
  }
};

}  // namespace alz
