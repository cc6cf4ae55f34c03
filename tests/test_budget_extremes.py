"""The host layer of the calls for long contexts in a small cache at the ends of its arguments' ranges, on the CPU, in
child processes, as in test_serving_extremes.py."""
from test_serving_extremes import child, sanitized  # noqa: F401  (the fixture)


def test_largest_numbers_overflow_nothing(sanitized):  # noqa: F811
    """Every number of a call at the largest of its type, alone and together with another.  (An append's max_pos builds a
    table of that many rows and is left as it is.)"""
    child(sanitized, """
import test_budget_refusals as b
big, wide = 2 ** 31 - 1, 2 ** 63 - 1
for name, good in b.GOOD.items():
    ints = [k for k, v in good.items() if isinstance(v, int) and v < t.P and k not in ("kv_dtype", "head_dim", "max_pos")]
    top = {k: wide if k.endswith("stride") else big for k in ints}
    for dt in (0, 2, 3, 16) if "kv_dtype" in good else (None,):
        more = {} if dt is None else {"kv_dtype": dt}
        for i in ints:
            for j in ints:
                b.call(fake, name, **{i: top[i], j: top[j]}, **more)
                b.call(fake, name, **{**{k: big for k in ("n_head", "n_kv_head") if k in good}, i: top[i], j: top[j]}, **more)
                b.call(fake, name, **{**{k: -v - 1 for k, v in top.items() if k == j}, i: top[i]}, **more)
        b.call(fake, name, **top, **more)
""")
