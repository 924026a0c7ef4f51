// The matrix instructions, conversions and loads into LDS that the dense library's kernels use (csrc/dense/k_device.inc), for the CPU
// emulation of hip_emu.h.  TEST INFRASTRUCTURE.  Lane layouts as measured on MI355X; sums in double, rounded once.
#pragma once
#include "hip_emu.h"

#include <math.h>
#include <string.h>

struct uint2 { unsigned x, y; };

#define DENSE_ORDER_READS(n) ((void)0)
#define DENSE_ORDER_MATRIX(n) ((void)0)
#define DENSE_KEEP_READS() ((void)0)

namespace dense {
typedef int v4i __attribute__((vector_size(16)));
typedef int v8i __attribute__((vector_size(32)));
typedef float f4 __attribute__((vector_size(16)));
typedef float f16v __attribute__((vector_size(64)));

static inline float half_value_of(unsigned short b) {
  const int e = (b >> 10) & 31, m = b & 1023;
  float v = e == 31 ? (m ? NAN : INFINITY) : e ? ldexpf(1024 + m, e - 25) : ldexpf(m, -24);
  return b & 0x8000 ? -v : v;
}
struct Halves {
  float of[65536];
  Halves() {
    for (int i = 0; i < 65536; ++i) of[i] = half_value_of((unsigned short)i);
  }
};
inline const Halves g_halves;
static inline float half_value(unsigned short b) { return g_halves.of[b]; }
static inline unsigned half_bits(float v) {
  unsigned b;
  memcpy(&b, &v, 4);
  const unsigned s = (b >> 16) & 0x8000;
  const float a = fabsf(v);
  if (a != a) return s | 0x7e00;
  if (a >= 65520.0f) return s | 0x7c00;
  if (a == 0) return s;
  int e;
  frexpf(a, &e);
  e = e - 1 < -14 ? -14 : e - 1;
  const long m = lrintf(ldexpf(a, 10 - e));                   // nearest even
  return s | (unsigned)(m >= 1024 ? ((e + 15) << 10) + (m - 1024) : m);
}
static inline float e4m3_value_of(unsigned char b) {
  const int e = (b >> 3) & 15, m = b & 7;
  float v = (b & 0x7f) == 0x7f ? NAN : e ? ldexpf(8 + m, e - 10) : ldexpf(m, -9);
  return b & 0x80 ? -v : v;
}
struct Bytes {
  float of[256];
  Bytes() {
    for (int i = 0; i < 256; ++i) of[i] = e4m3_value_of((unsigned char)i);
  }
};
inline const Bytes g_bytes;
static inline float e4m3_value(unsigned char b) { return g_bytes.of[b]; }
static inline unsigned e4m3_bits(float v) {
  unsigned b;
  memcpy(&b, &v, 4);
  const unsigned s = (b >> 24) & 0x80;
  const float a = fabsf(v);
  if (!(a <= 464.0f)) return s | 0x7f;
  if (a == 0) return s;
  int e;
  frexpf(a, &e);
  e = e - 1 < -6 ? -6 : e - 1;
  const long m = lrintf(ldexpf(a, 3 - e));
  unsigned r = (unsigned)(m >= 8 ? ((e + 7) << 3) + (m - 8) : m);
  return s | (r > 0x7e ? 0x7e : r);
}
static inline int pack_fp8(float a, float b, float c, float d) {
  return (int)(e4m3_bits(a) | (e4m3_bits(b) << 8) | (e4m3_bits(c) << 16) | (e4m3_bits(d) << 24));
}
static inline v4i halves_of_fp8(int lo, int hi) {
  v4i r;
  for (int i = 0; i < 4; ++i) {
    const unsigned w = (unsigned)(i < 2 ? lo : hi) >> (16 * (i & 1));
    r[i] = (int)(half_bits(e4m3_value(w & 255)) | (half_bits(e4m3_value((w >> 8) & 255)) << 16));
  }
  return r;
}

// what the lanes of a wavefront hand to a matrix instruction
struct Handed {
  v8i a, b;
  int sa, sb;
};
inline Handed* handed() {
  static thread_local Handed h[1024];
  return h + (hipemu::cur().flat & ~63u);
}
static inline f16v mma_f16(v4i a, v4i b, f16v c) {
  Handed* h = handed();
  const int l = (int)(hipemu::cur().flat & 63u);
  memcpy(&h[l].a, &a, 16), memcpy(&h[l].b, &b, 16);
  hipemu::wave_sync();
  for (int e = 0; e < 16; ++e) {
    const int row = 8 * (e / 4) + 4 * (l / 32) + e % 4, col = l % 32;
    double s = c[e];
    for (int k = 0; k < 2; ++k) {
      const unsigned short* x = reinterpret_cast<const unsigned short*>(&h[row + 32 * k].a);
      const unsigned short* y = reinterpret_cast<const unsigned short*>(&h[col + 32 * k].b);
      for (int i = 0; i < 8; ++i) s += (double)half_value(x[i]) * half_value(y[i]);
    }
    c[e] = (float)s;
  }
  hipemu::wave_sync();
  return c;
}
static inline f4 mma_f16_16(v4i a, v4i b, f4 c) {
  Handed* h = handed();
  const int l = (int)(hipemu::cur().flat & 63u);
  memcpy(&h[l].a, &a, 16), memcpy(&h[l].b, &b, 16);
  hipemu::wave_sync();
  for (int e = 0; e < 4; ++e) {
    double s = c[e];
    for (int k = 0; k < 4; ++k) {
      const unsigned short* x = reinterpret_cast<const unsigned short*>(&h[4 * (l / 16) + e + 16 * k].a);
      const unsigned short* y = reinterpret_cast<const unsigned short*>(&h[l % 16 + 16 * k].b);
      for (int i = 0; i < 8; ++i) s += (double)half_value(x[i]) * half_value(y[i]);
    }
    c[e] = (float)s;
  }
  hipemu::wave_sync();
  return c;
}
static inline f16v mma_f8(v8i a, v8i b, f16v c, int sa, int i, int sb, int j) {
  Handed* h = handed();
  const int l = (int)(hipemu::cur().flat & 63u);
  h[l] = Handed{a, b, (sa >> (8 * i)) & 255, (sb >> (8 * j)) & 255};
  hipemu::wave_sync();
  for (int e = 0; e < 16; ++e) {
    const int row = 8 * (e / 4) + 4 * (l / 32) + e % 4, col = l % 32;
    double s = c[e];
    for (int k = 0; k < 2; ++k) {
      const unsigned char* x = reinterpret_cast<const unsigned char*>(&h[row + 32 * k].a);
      const unsigned char* y = reinterpret_cast<const unsigned char*>(&h[col + 32 * k].b);
      double t = 0;
      for (int i = 0; i < 32; ++i) t += (double)e4m3_value(x[i]) * e4m3_value(y[i]);
      s += ldexp(t, h[row + 32 * k].sa + h[col + 32 * k].sb - 254);
    }
    c[e] = (float)s;
  }
  hipemu::wave_sync();
  return c;
}
static inline f4 mma_f8_16(v8i a, v8i b, f4 c, int sa, int sb) {
  Handed* h = handed();
  const int l = (int)(hipemu::cur().flat & 63u);
  h[l] = Handed{a, b, sa & 255, sb & 255};
  hipemu::wave_sync();
  for (int e = 0; e < 4; ++e) {
    const int row = 4 * (l / 16) + e, col = l % 16;
    double s = c[e];
    for (int k = 0; k < 4; ++k) {
      const unsigned char* x = reinterpret_cast<const unsigned char*>(&h[row + 16 * k].a);
      const unsigned char* y = reinterpret_cast<const unsigned char*>(&h[col + 16 * k].b);
      double t = 0;
      for (int i = 0; i < 32; ++i) t += (double)e4m3_value(x[i]) * e4m3_value(y[i]);
      s += ldexp(t, h[row + 16 * k].sa + h[col + 16 * k].sb - 254);
    }
    c[e] = (float)s;
  }
  hipemu::wave_sync();
  return c;
}
typedef const unsigned char* Window;
static inline Window window(const void* p) { return static_cast<const unsigned char*>(p); }
static inline void load_lds16(Window w, void* base, unsigned offset, unsigned line) {
  memcpy(static_cast<unsigned char*>(base) + 16 * (hipemu::cur().flat & 63u), w + (size_t)offset + line, 16);
}
static inline void load_lds_byte(Window w, void* base, unsigned offset) {
  static_cast<unsigned*>(base)[hipemu::cur().flat & 63u] = w[offset];
}
template <int N>
static inline void line_barrier() { hipemu::sync(); }
typedef double d4 __attribute__((vector_size(32)));
static inline d4 mma_f64(double a, double b, d4 c) {
  static thread_local double x[1024], y[1024];
  const unsigned f = hipemu::cur().flat, w = f & ~63u, l = f & 63u;
  x[f] = a, y[f] = b;
  hipemu::wave_sync();
  for (unsigned e = 0; e < 4; ++e)
    for (unsigned k = 0; k < 4; ++k) c[e] += x[w + l / 16 + 4 * e + 16 * k] * y[w + l % 16 + 16 * k];
  hipemu::wave_sync();
  return c;
}
static inline unsigned max_of_16(unsigned v) {
  for (int d = 8; d >= 1; d >>= 1) {
    float f;
    memcpy(&f, &v, 4);
    f = __shfl_xor(f, d);
    unsigned w;
    memcpy(&w, &f, 4);
    v = v > w ? v : w;
  }
  return v;
}
static inline int __shfl(int v, int lane) {
  float f;
  memcpy(&f, &v, 4);
  f = ::__shfl(f, lane);
  memcpy(&v, &f, 4);
  return v;
}
static inline int uniform(int v) { return v; }
}  // namespace dense
