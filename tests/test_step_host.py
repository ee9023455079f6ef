"""Host-side parts of the serving-step operators, compiled into small host programs: the keys
that pages are chosen by, the kernels' shared memory, the order of launches."""
import ctypes
import os
import shutil
import subprocess
import sys
import sysconfig

import numpy as np
import pytest

from conftest import PKG

CSRC = os.path.join(PKG, "csrc")
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")
pytestmark = pytest.mark.skipif(
    shutil.which("g++") is None or not os.path.exists(os.path.join(CUDA, "include")),
    reason="needs g++ and the CUDA headers")


def host_library(tmp_path, source, *flags):
    src, out = tmp_path / "host.cpp", tmp_path / "host.so"
    src.write_text(source)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-shared", "-fPIC", "-pthread",
                    f"-I{CSRC}", f"-I{CUDA}/include", "-o", str(out), str(src), *flags], check=True)
    return ctypes.CDLL(str(out))


# --------------------------------------------------------------------------- the pages' keys
@pytest.fixture
def page_key(tmp_path):
    lib = host_library(tmp_path, '''
        #include "page_key.h"
        extern "C" unsigned key(float best, float sc) { return fe::step::page_key(best, sc); }
        extern "C" unsigned forced() { return fe::step::kForced; }''')
    lib.key.argtypes, lib.key.restype = [ctypes.c_float] * 2, ctypes.c_uint
    lib.forced.restype = ctypes.c_uint
    return lib


def floats(*bits):
    return [float(x) for x in np.array(bits, np.uint32).view(np.float32)]


def test_no_score_has_the_key_of_an_always_chosen_page(page_key):
    """More always-chosen keys than pages are kept would be listed past the list's end."""
    inf = float("inf")
    scales = [0.0, -0.0, 1.0, -1.0, inf, -inf, 2.0 ** -120, 2.0 ** 122] + floats(
        0x7fffffff, 0xffffffff, 0x7fc00000, 0xffc00000, 0x7f800001, 0xff800001)  # NaN
    sums = [0.0, -0.0, 1.0, -1.0, 2.0 ** 24, -2.0 ** 24, inf, -inf, 3e38, -3e38]
    for sc in scales:
        for best in sums:
            k = page_key.key(best, sc)
            assert 0 < k < page_key.forced(), (best, sc, hex(k))


def test_keys_are_in_the_order_of_the_scores(page_key):
    inf, nan = float("inf"), float("nan")
    scores = [-inf, -3e38, -1.5, -1.0, -1e-45, 0.0, 1e-45, 1.0, 1.5, 3e38, inf]
    keys = [page_key.key(x, 1.0) for x in scores]
    assert keys == sorted(set(keys))
    assert page_key.key(-0.0, 1.0) == page_key.key(0.0, 1.0)
    for sc, best in ((inf, -5.0), (inf, 0.0), (nan, 1.0), (nan, -1.0), (-inf, 0.0), (0.0, inf)):
        assert page_key.key(best, sc) == keys[-1], (sc, best)


# ----------------------------------------------------------- the shared memory of the kernels
def test_shared_memory_opt_in_never_shrinks(tmp_path):
    """Threads that launch kernels of changing sizes: at each launch the attribute (the last
    value set) covers what it needs, and a kernel's sizes take one record however many."""
    run = host_library(tmp_path, '''
        #include "smem_optin.h"
        #include <atomic>
        #include <thread>
        #include <vector>
        // Returns launches that would fail; calls[0] counts the sets.
        extern "C" int run(int threads, int rounds, int kernels, int fail_every, int* calls) {
          fe::SmemOptin optin;
          std::vector<std::atomic<int>> attribute(kernels);
          for (auto& a : attribute) a = 48 * 1024;
          std::atomic<int> bad{0}, sets{0};
          std::vector<std::thread> all;
          for (int t = 0; t < threads; ++t)
            all.emplace_back([&, t] {
              unsigned x = 12345u + 777u * t;
              for (int i = 0; i < rounds; ++i) {
                x = x * 1664525u + 1013904223u;
                const int k = (x >> 8) % kernels, bytes = 50000 + (x >> 12) % 150000;
                const int e = optin.ensure(&attribute[k], 0, bytes, [&](int n) {
                  const int at = ++sets;
                  if (fail_every && at % fail_every == 0) return 1;
                  std::this_thread::yield();
                  attribute[k] = n;
                  return 0;
                }, 2);
                if (e == 0 && attribute[k] < bytes) ++bad;
              }
            });
          for (auto& t : all) t.join();
          calls[0] = sets;
          return bad;
        }
        extern "C" int devices() {  // one function on two devices: two records
          fe::SmemOptin optin;
          int n = 0, f = 0;
          auto set = [&](int) { ++n; return 0; };
          for (int i : {0, 1, 0}) optin.ensure(&f, i, 100, set, 2);
          optin.ensure(&f, 1, 90, set, 2);
          optin.ensure(&f, 1, 101, set, 2);
          return n;
        }''')
    calls = ctypes.c_int()
    for fail_every in (0, 7):
        for kernels in (1, 3, 700):
            assert run.run(8, 20000, kernels, fail_every, ctypes.byref(calls)) == 0
            # running maxima of random sizes: a few sets a kernel
            assert calls.value < 40 * kernels + (20 if fail_every else 0)
    assert run.devices() == 3


# -------------------------------------------------------------------- the order of the launches
def test_a_decode_right_behind_a_writer_of_tables_starts_after_it(tmp_path):
    lib = host_library(tmp_path, '''
        #include "launch_order.h"
        #include <thread>
        static fe::TableWriters w;
        extern "C" void wrote(int d, long s) { w.wrote(d, reinterpret_cast<void*>(s)); }
        extern "C" int passed(int d, long s) { return w.passed(d, reinterpret_cast<void*>(s)); }
        // Threads with a stream each: every decode after a plan has to see it.
        extern "C" int race(int threads, int rounds) {
          fe::TableWriters x;
          std::vector<std::thread> all;
          std::atomic<int> bad{0};
          for (long t = 0; t < threads; ++t)
            all.emplace_back([&, t] {
              const void* s = reinterpret_cast<const void*>(t);
              for (int i = 0; i < rounds; ++i) {
                x.wrote(0, s);
                if (i & 1) x.wrote(0, s);
                bad += !x.passed(0, s);
                bad += x.passed(0, s);
              }
            });
          for (auto& t : all) t.join();
          return bad;
        }''')
    lib.wrote.argtypes = lib.passed.argtypes = [ctypes.c_int, ctypes.c_long]
    assert not lib.passed(0, 0)                      # nothing written yet
    lib.wrote(0, 0)                                  # plan -> decode -> decode
    assert lib.passed(0, 0) and not lib.passed(0, 0)
    lib.wrote(0, 7)                                  # another stream, another device
    assert not lib.passed(0, 0) and not lib.passed(1, 7)
    lib.wrote(0, 0)
    lib.wrote(0, 0)
    lib.wrote(1, 0)
    assert lib.passed(0, 0) and not lib.passed(0, 0)
    assert lib.passed(0, 7) and lib.passed(1, 0) and not lib.passed(1, 0)
    assert lib.race(8, 20000) == 0


# ------------------------------------------------------------------------- the native binding
def test_package_works_without_the_native_binding():
    """Only the serving-step operators need it, and they say what is missing when called."""
    code = '''
import sys
import sysconfig
class Absent:
    def find_spec(self, name, path=None, target=None):
        if name.endswith("_step_native"):
            raise ImportError("not built")
sys.meta_path.insert(0, Absent())
import torch, flash_engine as F
z = torch.zeros(1)
for call in (lambda: F.paged_attention(z, z, z, z, z), lambda: F.flash_attention(z, z, z)):
    try:
        call()
    except TypeError:
        pass
    else:
        raise AssertionError
F.new_page_bounds(2, 1, 64, "cpu")
for call in (lambda: F.plan_paged_step(z, z, z, z, z, max_tokens=4),
             lambda: F.paged_qkv_append(z, z, z, z, z, 4),
             lambda: F.update_page_bounds(z, (z, z), z),
             lambda: F.sparse_paged_attention(z, z, z, (z, z), z, z, 4)):
    try:
        call()
    except ImportError as e:
        assert "make -C" in str(e) and "not built" in str(e), e
    else:
        raise AssertionError
'''
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=PKG),
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def make(*args):
    r = subprocess.run(["make", "-C", CSRC, *args], capture_output=True, text=True)
    return r.returncode, r.stdout + r.stderr


@pytest.mark.skipif(shutil.which("make") is None, reason="needs make")
def test_library_builds_without_torch(tmp_path):
    """Dry runs into an empty folder, with an interpreter that has no torch."""
    to = (f"OBJDIR={tmp_path}/obj", f"OUTDIR={tmp_path}/lib", "PYTHON=false")
    for goal in ((), ("lib",)):
        rc, out = make("-n", *to, *goal)
        assert rc == 0 and "libflash_engine_b200.so" in out and "step_binding.cpp" not in out
    rc, out = make(*to, "binding")
    assert rc != 0 and "torch" in out


@pytest.mark.skipif(shutil.which("make") is None, reason="needs make")
def test_binding_is_built_again_for_another_interpreter_or_torch(tmp_path):
    binding, stamp = tmp_path / "native.so", tmp_path / "obj" / "binding.stamp"
    to = (f"OBJDIR={tmp_path}/obj", f"PYTHON={sys.executable}", "binding")
    as_named, given = to, to + (f"BINDING={binding}",)
    rc, out = make("-n", *as_named)
    suffix = sysconfig.get_config_var("EXT_SUFFIX")
    assert rc == 0 and (f"_step_native{suffix} " in out or "up to date" in out or
                        "Nothing to be done" in out)
    rc, out = make("-n", *given)
    assert rc == 0 and "step_binding.cpp" in out      # not there yet
    binding.touch()
    rc, out = make("-n", *given)
    assert rc == 0 and "step_binding.cpp" not in out  # newer than all it comes from
    stamp.write_text("another torch\n")
    past = binding.stat().st_mtime - 100
    os.utime(stamp, (past, past))
    rc, out = make("-n", *given)
    assert rc == 0 and "step_binding.cpp" in out


# ------------------------------------------------------------------------- the C++ launchers
def test_cpp_launchers_pass_their_arguments_in_order(tmp_path):
    """serving_step.cuh against the library: what each launcher refuses, one field at a time
    (nothing is launched: no tokens, no sequences)."""
    lib = os.path.join(PKG, "flash_engine", "lib")
    if not os.path.exists(os.path.join(lib, "libflash_engine_b200.so")):
        pytest.skip("the library is not built")
    source = '''
        #include "serving_step.cuh"
        using namespace flash_engine::serving;
        static char at[64] __attribute__((aligned(64)));
        template <typename T> T* p() { return reinterpret_cast<T*>(at); }
        static int plan(StepPlanConfig c) {  // no outputs: refused by then if all else is right
          return launch_plan_paged_step(p<int>(), p<int>(), nullptr, p<int>(), p<int>(), p<int>(),
                                        p<int>(), p<int>(), p<int>(), p<long long>(), nullptr, c);
        }
        static int append(int tokens, int heads, long long stride, CacheConfig c, float eps = 0,
                          RopeTables r = {}) {
          return launch_paged_qkv_append(p<void>(), stride, p<void>(), p<void>(), p<void>(),
                                         p<int>(), p<long long>(), nullptr, nullptr, false, eps, r,
                                         tokens, heads, c);
        }
        static int bounds(int tokens, CacheConfig c) {
          return launch_update_page_bounds(p<void>(), p<signed char>(), p<float>(),
                                           p<long long>(), tokens, c);
        }
        static int sparse(int seqs, int heads, int width, int pages, int first, int last,
                          CacheConfig c) {
          return launch_sparse_paged_attention(
              p<void>(), p<void>(), p<void>(), p<void>(), p<signed char>(), p<float>(), p<int>(),
              p<int>(), p<int>(), p<int>(), seqs, heads, width, pages, first, last, 0.1f, c);
        }
        extern "C" int run() {
          const CacheConfig c{4, 2, 64, 16};
          const int bad = cudaErrorInvalidValue;
          int n = 0;  // the first check that fails
        #define CHECK(x) ++n; if (!(x)) return n;
          CHECK(plan({1, 2, 8, 16, 4}) == bad)
          CHECK(append(0, 4, 512, c) == 0)
          CHECK(append(0, 4, 511, c) == bad)
          CHECK(append(0, 0, 512, c) == bad)
          CHECK(append(-1, 4, 512, c) == bad)
          CHECK(append(0, 4, 512, c, -1.f) == bad)
          RopeTables r{p<float>(), p<float>(), 64, 8, true};
          CHECK(append(0, 4, 512, c, 0.f, r) == 0)
          r.rotary_dim = 66;
          CHECK(append(0, 4, 512, c, 0.f, r) == bad)
          r.rotary_dim = 64;
          r.max_pos = 0;
          CHECK(append(0, 4, 512, c, 0.f, r) == bad)
          CHECK(append(0, 4, 512, {4, 2, 64, 16, DType::kFp32, KvLayout::kVllm}) == bad)
          CHECK(append(0, 4, 512, {4, 2, 64, 16, DType::kFp32}) == 0)
          CHECK(bounds(0, c) == 0 && bounds(-1, c) == bad)
          CHECK(bounds(0, {4, 2, 96, 16}) == bad && bounds(0, {4, 2, 64, 8}) == bad)
          CHECK(bounds(0, {0, 2, 64, 16}) == bad && bounds(0, {4, 0, 64, 16}) == bad)
          CHECK(bounds(0, {4, 2, 128, 32}) == 0)
          CHECK(sparse(0, 4, 8, 3, 1, 2, c) == 0)
          CHECK(sparse(0, 4, 8, 3, 1, 3, c) == bad)
          CHECK(sparse(0, 4, 8, 3, 2, 0, c) == bad)
          CHECK(sparse(0, 5, 8, 3, 1, 2, c) == bad)
          CHECK(sparse(0, 4, 0, 3, 1, 2, c) == bad)
          CHECK(sparse(-1, 4, 8, 3, 1, 2, c) == bad)
          CHECK(sparse(0, 4, 8, 3, 1, 2, {4, 2, 64, 32, DType::kBf16, KvLayout::kVllm}) == bad)
          return 0;
        }'''
    include = os.path.join(os.path.dirname(PKG), "include")
    assert host_library(tmp_path, source, f"-I{include}", f"-L{lib}", f"-Wl,-rpath,{lib}",
                        "-l:libflash_engine_b200.so").run() == 0


def test_bookkeeping_throws_nothing_through_the_c_entries(tmp_path):
    """Without memory for a record: a status, and every stream counted as one to wait for."""
    lib = host_library(tmp_path, '''
        #include <cstdlib>
        #include <new>
        static bool none = false;
        void* take(std::size_t n) {
          if (none) throw std::bad_alloc();
          return std::malloc(n);
        }
        template <typename T>
        struct Failing {  // in place of std::allocator in the two headers
          using value_type = T;
          Failing() = default;
          template <typename U> Failing(const Failing<U>&) {}
          T* allocate(std::size_t n) { return static_cast<T*>(take(n * sizeof(T))); }
          void deallocate(T* p, std::size_t) { std::free(p); }
          template <typename U> bool operator==(const Failing<U>&) const { return true; }
          template <typename U> bool operator!=(const Failing<U>&) const { return false; }
        };
        #include <algorithm>
        #include <atomic>
        #include <map>
        #include <mutex>
        #include <utility>
        #include <vector>
        namespace poor {
        template <typename T> using vector = std::vector<T, Failing<T>>;
        template <typename K, typename V>
        using map = std::map<K, V, std::less<K>, Failing<std::pair<const K, V>>>;
        }
        namespace std { namespace host_test { using poor::vector; using poor::map; } }
        #define vector host_test::vector
        #define map host_test::map
        #include "launch_order.h"
        #include "smem_optin.h"
        #undef vector
        #undef map
        extern "C" int run() {
          static fe::TableWriters w;
          static fe::SmemOptin o;
          auto set = [](int) { return 0; };
          int f = 0, n = 0;
        #define CHECK(x) ++n; if (!(x)) return n;
          CHECK(o.ensure(&f, 0, 100, set, 2) == 0 && !w.passed(0, nullptr))
          none = true;
          CHECK(o.ensure(&f, 1, 100, set, 2) == 2 && o.ensure(&f, 0, 200, set, 2) == 0)
          w.wrote(0, nullptr);
          CHECK(w.passed(0, nullptr) && w.passed(0, &f) && w.passed(1, nullptr))
          none = false;
          CHECK(o.ensure(&f, 1, 100, set, 2) == 0 && w.passed(0, nullptr))
          return 0;
        }''')
    assert lib.run() == 0
