"""The serving calls' host layer at the ends of its arguments' ranges, on the CPU, in child
processes: built with UndefinedBehaviorSanitizer (a report ends the child) over the HIP
runtime that runs nothing (tests/cpp/fake_hip.cpp)."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CPP = os.path.join(HERE, "cpp")
SAN = os.path.join(CPP, "build", "libtmac_fake_san.so")
ENV = {k: v for k, v in os.environ.items() if k not in ("LD_PRELOAD", "TMAC_ATTN_LIB", "TMAC_ORACLE_LIB")}


@pytest.fixture(scope="module")
def sanitized():
    subprocess.run(["make", "-s", "-C", CPP, "sanitize"], check=True, env=ENV)
    return SAN


def child(lib, code):
    """What `code` prints in a process of its own, `fake` being the host layer in `lib`."""
    head = ("import sys; sys.path[:0] = [%r, %r]; import test_serving_refusals as t; t.FAKE = %r; fake = t.Fake();"
            % (HERE, os.path.join(os.path.dirname(HERE), "tmac_gguf.cpp_amd"), lib))
    res = subprocess.run([sys.executable, "-c", head + "\n" + code], capture_output=True, text=True,
                         env={**ENV, "UBSAN_OPTIONS": "print_stacktrace=1"}, timeout=300)
    assert res.returncode == 0, (res.stdout + res.stderr)[-3000:]
    return res.stdout.split()


def test_largest_numbers_overflow_nothing(sanitized):
    """Every number of a call at the largest int, alone and together with another: no product of them overflows.  (An
    append's max_len builds a table of that many rows and is left as it is.)"""
    child(sanitized, """
big = 2 ** 31 - 1
for name, good in t.GOOD.items():
    ints = [k for k, v in good.items() if isinstance(v, int) and v < t.P and k not in ("kv_dtype", "head_dim")]
    ints = [k for k in ints if not (name == "tmac_kv_append_paged" and k == "max_len")]
    for i in ints:
        for j in ints:
            fake.call(name, **{i: big, j: big})
            fake.call(name, **{**{k: big for k in ("n_head", "n_kv_head") if k in good}, i: big, j: big})
""")


def test_a_rotation_table_too_large_for_memory_is_an_error(sanitized):
    """An append whose max_len asks for more host memory than there is returns a status; no exception leaves the C entry,
    and the next call finds the context as it was."""
    status = child(sanitized, """
import resource
resource.setrlimit(resource.RLIMIT_AS, (8 << 30, 8 << 30))  # the table of 2^26 positions is 16 GiB
print(fake.call("tmac_kv_append_paged", max_pages=2 ** 23, max_len=2 ** 26, base=1e4))
print(fake.call("tmac_kv_append_paged", base=1e4))
""")
    assert "".join(status) == "(1002,[])(0,[('tmac_append_f32',5)])"
