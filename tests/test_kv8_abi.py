"""CPU checks of the 8-bit serving entry points: struct layouts, refusals, random arguments. Nothing is launched: the
calls that pass their checks run in a process whose device is disabled."""
import ctypes
import os
import pathlib
import subprocess
import sys

import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]


@pytest.mark.parametrize("struct,cname", [("Kv8CacheArgs", "tsfm_kv8_cache"), ("Kv8PlanArgs", "tsfm_kv8_plan_args"),
                                          ("Kv8ReleaseArgs", "tsfm_kv8_release_args"),
                                          ("Kv8AppendArgs", "tsfm_kv8_append_args"),
                                          ("Kv8AttendArgs", "tsfm_kv8_attend_args"),
                                          ("F8QuantizeArgs", "tsfm_f8_quantize_args"),
                                          ("F8GemmArgs", "tsfm_f8_gemm_args")])
def test_layouts_match_the_header(ta, struct, cname, tmp_path):
    cls = getattr(ta, struct)
    fields = [f[0] for f in cls._fields_]
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "tsfm_attn.h"\nint main(void){\n'
    src += f'printf("%zu\\n", sizeof({cname}));\n' + "".join(f'printf("%zu\\n", offsetof({cname}, {f}));\n' for f in fields)
    (tmp_path / "l.c").write_text(src + "return 0;}\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    out = [int(x) for x in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    assert out[0] == ctypes.sizeof(cls)
    assert out[1:] == [getattr(cls, f).offset for f in fields]


P = 1 << 12  # an address that is aligned and is never read


def _cache(ta, **over):
    kw = dict(dtype=ta.DTYPE_BF16, code=ta.CODE_E4M3, requests=2, kv_heads=2, head_dim=64, blocks=8, table_width=4, k=P, v=P,
              scales=P, k_tail=P, v_tail=P, table=P, len=P)
    kw.update(over)
    return ta.Kv8CacheArgs(**kw)


def _append(ta, cache=None, **over):
    kw = dict(cache=_cache(ta, **(cache or {})), max_tokens=3, max_items=3, flags=ta.DEVICE_PTRS, cu_tokens=P, items=P, k=P,
              k_tok=128, v=P, v_tok=128)
    kw.update(over)
    return ta.Kv8AppendArgs(**kw)


def _attend(ta, cache=None, **over):
    kw = dict(cache=_cache(ta, **(cache or {})), heads=4, max_tokens=3, flags=ta.DEVICE_PTRS, scale=0.5, cu_tokens=P, q=P,
              q_tok=256, o=P, o_tok=256, workspace=P, workspace_bytes=1 << 40)
    kw.update(over)
    return ta.Kv8AttendArgs(**kw)


def _plan(ta, **over):
    kw = dict(requests=2, blocks=8, table_width=4, max_tokens=100, max_items=100, flags=ta.DEVICE_PTRS)
    kw.update({f: P for f, t in ta.Kv8PlanArgs._fields_ if t is ctypes.c_void_p and f != "stream"})
    kw.update(over)
    return ta.Kv8PlanArgs(**kw)


def _release(ta, **over):
    kw = dict(requests=2, blocks=8, table_width=4, flags=ta.DEVICE_PTRS, drop=P, len=P, table=P, free_list=P, free_count=P,
              status=P)
    kw.update(over)
    return ta.Kv8ReleaseArgs(**kw)


def _quantize(ta, **over):
    kw = dict(dtype=ta.DTYPE_BF16, rows=4, cols=128, group_rows=1, flags=ta.DEVICE_PTRS, x=P, x_ld=128, codes=P, codes_ld=128,
              scales=P, scales_ld=1)
    kw.update(over)
    return ta.F8QuantizeArgs(**kw)


def _gemm(ta, **over):
    kw = dict(m=4, n=130, k=256, out_dtype=ta.DTYPE_F32, flags=ta.DEVICE_PTRS, a=P, a_ld=256, a_scales=P, a_scales_ld=2, b=P,
              b_ld=256, b_scales=P, b_scales_ld=2, c=P, c_ld=130)
    kw.update(over)
    return ta.F8GemmArgs(**kw)


INVALID, UNSUPPORTED = "E_INVALID", "E_UNSUPPORTED"
CACHE = [(dict(dtype=0), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED), (dict(code=2), INVALID), (dict(head_dim=96), UNSUPPORTED),
         (dict(kv_heads=0), INVALID), (dict(requests=0), INVALID), (dict(requests=65537), UNSUPPORTED), (dict(blocks=0), INVALID),
         (dict(blocks=-1), INVALID), (dict(blocks=0x7fffffff), UNSUPPORTED), (dict(table_width=0), INVALID),
         (dict(table_width=1 << 25), UNSUPPORTED), (dict(k=0), INVALID), (dict(v=0), INVALID), (dict(scales=0), INVALID),
         (dict(k_tail=0), INVALID), (dict(v_tail=0), INVALID), (dict(table=0), INVALID), (dict(len=0), INVALID),
         (dict(k=P + 8), UNSUPPORTED), (dict(v_tail=P + 2), UNSUPPORTED), (dict(scales=P + 4), UNSUPPORTED),
         (dict(blocks=1 << 30, kv_heads=1 << 12), UNSUPPORTED)]


@pytest.mark.parametrize("over,code", CACHE)
def test_cache_refusals(ta, over, code):
    for a, fn in ((_append(ta, over), ta.load().tsfm_kv8_append), (_attend(ta, over), ta.load().tsfm_kv8_attend)):
        assert fn(ctypes.byref(a)) == getattr(ta, code), ta.last_error()
        assert ta.last_error()


@pytest.mark.parametrize("make,fn,over,code", [
    (_append, "tsfm_kv8_append", dict(flags=0), UNSUPPORTED), (_append, "tsfm_kv8_append", dict(flags=5), INVALID),
    (_append, "tsfm_kv8_append", dict(max_tokens=-1), INVALID), (_append, "tsfm_kv8_append", dict(k=0), INVALID),
    (_append, "tsfm_kv8_append", dict(items=0), INVALID), (_append, "tsfm_kv8_append", dict(k_tok=-8), INVALID),
    (_append, "tsfm_kv8_append", dict(k_tok=132), UNSUPPORTED), (_append, "tsfm_kv8_append", dict(v=P + 8), UNSUPPORTED),
    (_append, "tsfm_kv8_append", dict(k_tok=1 << 45), UNSUPPORTED),
    (_append, "tsfm_kv8_append", dict(max_tokens=(1 << 30) + 1), UNSUPPORTED),
    (_attend, "tsfm_kv8_attend", dict(flags=0), UNSUPPORTED), (_attend, "tsfm_kv8_attend", dict(heads=3), INVALID),
    (_attend, "tsfm_kv8_attend", dict(heads=0), INVALID), (_attend, "tsfm_kv8_attend", dict(max_new=-1), INVALID),
    (_attend, "tsfm_kv8_attend", dict(scale=-0.5), UNSUPPORTED),
    (_attend, "tsfm_kv8_attend", dict(scale=float("nan")), UNSUPPORTED),
    (_attend, "tsfm_kv8_attend", dict(o_tok=128), INVALID), (_attend, "tsfm_kv8_attend", dict(q_tok=250), UNSUPPORTED),
    (_attend, "tsfm_kv8_attend", dict(q=0), INVALID), (_attend, "tsfm_kv8_attend", dict(o=P + 4), UNSUPPORTED),
    (_attend, "tsfm_kv8_attend", dict(cu_tokens=0), INVALID),
    (_attend, "tsfm_kv8_attend", dict(cache=dict(table_width=4096), workspace=0), INVALID),
    (_attend, "tsfm_kv8_attend", dict(cache=dict(table_width=4096), workspace_bytes=64), INVALID),
    (_attend, "tsfm_kv8_attend", dict(cache=dict(table_width=4096), workspace=P + 4), UNSUPPORTED),
    (_attend, "tsfm_kv8_attend", dict(max_tokens=1 << 30, heads=1 << 10, q_tok=1 << 16, o_tok=1 << 16), UNSUPPORTED),
    (_plan, "tsfm_kv8_plan", dict(flags=0), UNSUPPORTED), (_plan, "tsfm_kv8_plan", dict(max_items=4), INVALID),
    (_plan, "tsfm_kv8_plan", dict(max_tokens=0), INVALID), (_plan, "tsfm_kv8_plan", dict(requests=70000), UNSUPPORTED),
    (_plan, "tsfm_kv8_plan", dict(slots=P + 4), UNSUPPORTED), (_plan, "tsfm_kv8_plan", dict(status=0), INVALID),
    (_plan, "tsfm_kv8_plan", dict(n_new=P + 1), UNSUPPORTED), (_plan, "tsfm_kv8_plan", dict(cu_items=0), INVALID),
    (_release, "tsfm_kv8_release", dict(flags=0), UNSUPPORTED), (_release, "tsfm_kv8_release", dict(drop=0), INVALID),
    (_release, "tsfm_kv8_release", dict(blocks=0), INVALID), (_release, "tsfm_kv8_release", dict(len=P + 2), UNSUPPORTED),
    (_quantize, "tsfm_f8_quantize", dict(flags=0), UNSUPPORTED), (_quantize, "tsfm_f8_quantize", dict(dtype=3), INVALID),
    (_quantize, "tsfm_f8_quantize", dict(group_rows=64), UNSUPPORTED), (_quantize, "tsfm_f8_quantize", dict(cols=120), UNSUPPORTED),
    (_quantize, "tsfm_f8_quantize", dict(rows=-1), INVALID), (_quantize, "tsfm_f8_quantize", dict(codes_ld=112), INVALID),
    (_quantize, "tsfm_f8_quantize", dict(codes_ld=130), UNSUPPORTED), (_quantize, "tsfm_f8_quantize", dict(x_ld=132), UNSUPPORTED),
    (_quantize, "tsfm_f8_quantize", dict(x=P + 8), UNSUPPORTED), (_quantize, "tsfm_f8_quantize", dict(scales=0), INVALID),
    (_quantize, "tsfm_f8_quantize", dict(scales_ld=0), INVALID),
    (_gemm, "tsfm_f8_gemm_nt", dict(flags=0), UNSUPPORTED), (_gemm, "tsfm_f8_gemm_nt", dict(out_dtype=3), INVALID),
    (_gemm, "tsfm_f8_gemm_nt", dict(k=0), UNSUPPORTED), (_gemm, "tsfm_f8_gemm_nt", dict(k=250), UNSUPPORTED),
    (_gemm, "tsfm_f8_gemm_nt", dict(m=-1), INVALID), (_gemm, "tsfm_f8_gemm_nt", dict(c_ld=129), INVALID),
    (_gemm, "tsfm_f8_gemm_nt", dict(a_ld=264), UNSUPPORTED), (_gemm, "tsfm_f8_gemm_nt", dict(b=P + 4), UNSUPPORTED),
    (_gemm, "tsfm_f8_gemm_nt", dict(a_ld=1 << 24), UNSUPPORTED), (_gemm, "tsfm_f8_gemm_nt", dict(b_scales=0), INVALID),
    (_gemm, "tsfm_f8_gemm_nt", dict(c=P + 2), UNSUPPORTED), (_gemm, "tsfm_f8_gemm_nt", dict(a_scales_ld=1 << 46), UNSUPPORTED)])
def test_refusals(ta, make, fn, over, code):
    assert getattr(ta.load(), fn)(ctypes.byref(make(ta, **over))) == getattr(ta, code), ta.last_error()
    assert ta.last_error()


def test_null_arguments(ta):
    for fn in ("tsfm_kv8_plan", "tsfm_kv8_release", "tsfm_kv8_append", "tsfm_kv8_attend", "tsfm_f8_quantize", "tsfm_f8_gemm_nt"):
        assert getattr(ta.load(), fn)(None) == ta.E_INVALID
    assert ta.load().tsfm_kv8_attend_workspace(None) == -1


def test_nothing_to_do_needs_no_arrays(ta):
    for a, fn in ((_append(ta, max_tokens=0, k=0, v=0), "tsfm_kv8_append"), (_append(ta, max_items=0), "tsfm_kv8_append"),
                  (_attend(ta, max_tokens=0), "tsfm_kv8_attend"), (_quantize(ta, rows=0, x=0), "tsfm_f8_quantize"),
                  (_gemm(ta, m=0, a=0), "tsfm_f8_gemm_nt"), (_gemm(ta, n=0, b=0), "tsfm_f8_gemm_nt")):
        assert getattr(ta.load(), fn)(ctypes.byref(a)) == ta.OK


def test_workspace_grows_with_the_split(ta):
    """None for contexts of one chunk; the pointers are not read."""
    ws = ta.load().tsfm_kv8_attend_workspace
    none = dict(k=0, v=0, scales=0, k_tail=0, v_tail=0, table=0, len=0)
    assert ws(ctypes.byref(_attend(ta, none, q=0, o=0, cu_tokens=0, workspace=0))) == 0
    long = ws(ctypes.byref(_attend(ta, dict(none, table_width=4096), q=0, o=0, cu_tokens=0, workspace=0, workspace_bytes=0)))
    assert long > 0
    hinted = ws(ctypes.byref(_attend(ta, dict(none, table_width=4096), max_len=100, q=0, o=0, cu_tokens=0)))
    assert hinted == 0
    assert ws(ctypes.byref(_attend(ta, none, heads=3))) == -1 and "heads" in ta.last_error()


_FUZZ = r'''
import ctypes, random, sys
sys.path.insert(0, %r)
sys.path.insert(0, %r)
import os
import tsfm_attn as ta
if os.environ.get("TSFM_FUZZ_LIB"):
    ta._lib = ta.load(os.environ["TSFM_FUZZ_LIB"])
import test_kv8_abi as t
lib = ta.load()
rng = random.Random(5)
ints = [0, 1, 2, 3, 15, 16, 63, 64, 65, 100, 128, 1000, 65536, 65537, 1 << 20, (1 << 25) - 1, 1 << 30, (1 << 31) - 1, -1, -(1 << 31)]
longs = ints + [1 << 40, 1 << 46, (1 << 63) - 1, -(1 << 63)]
ptrs = [0, t.P, t.P, t.P, t.P, t.P + 1, t.P + 4, t.P + 8]
def fill(a, share):
    for f, ty in a._fields_:
        if f == "stream" or rng.random() > share:
            continue
        if issubclass(ty, ctypes.Structure):
            fill(getattr(a, f), share)
        elif ty is ctypes.c_float:
            setattr(a, f, rng.choice([0.0, 1.0, -1.0, float("nan"), float("inf")]))
        elif ty is ctypes.c_void_p:
            setattr(a, f, rng.choice(ptrs))
        elif ty is ctypes.c_int64:
            setattr(a, f, rng.choice(longs))
        elif ty is ctypes.c_uint32:
            setattr(a, f, rng.choice([0, 1, 1, 1, 2, 7]))
        else:
            setattr(a, f, rng.choice(ints))
seen = set()
for it in range(24000):
    make, fn = rng.choice([(t._append, "tsfm_kv8_append"), (t._attend, "tsfm_kv8_attend"), (t._plan, "tsfm_kv8_plan"),
                           (t._release, "tsfm_kv8_release"), (t._quantize, "tsfm_f8_quantize"), (t._gemm, "tsfm_f8_gemm_nt")])
    a = make(ta)
    fill(a, rng.choice([0.0, 0.1, 0.3, 0.9]))
    rc = getattr(lib, fn)(ctypes.byref(a))
    assert rc in (0, 1, 2, 3), (fn, rc)
    seen.add((fn, rc))
    if make is t._attend:
        assert lib.tsfm_kv8_attend_workspace(ctypes.byref(a)) >= -1
print(sorted({r for _, r in seen}), len(seen))
'''


def test_random_arguments_return_codes():
    """Random argument blocks through every entry point in a process whose device is disabled: one of the ABI's codes each
    time, refusals and (where the checks pass) the disabled device among them."""
    env = dict(os.environ, TSFM_HIP_DISABLE="1")
    if os.environ.get("TSFM_TEST_PRODUCT_LIB"):
        env["TSFM_FUZZ_LIB"] = os.environ["TSFM_TEST_PRODUCT_LIB"]
    r = subprocess.run([sys.executable, "-c", _FUZZ % (str(ROOT / "tsfm-zig_amd"), str(ROOT / "tests"))], env=env,
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-3000:]
    assert r.stdout.split("]")[0] == "[0, 1, 2, 3", r.stdout


def test_host_code_under_sanitizers():
    """The same under AddressSanitizer and UndefinedBehaviorSanitizer, with the sanitized build of the library."""
    import glob

    libs = sorted(glob.glob("/opt/rocm/llvm/lib/clang/*/lib/linux/libclang_rt.asan-x86_64.so"))
    if os.environ.get("LD_PRELOAD") or os.environ.get("TSFM_TEST_PRODUCT_LIB") or not libs:
        pytest.skip("the sanitizer runtime has to load first")
    r = subprocess.run(["make", "-C", str(ROOT / "tsfm-zig_amd"), "sanitize"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    lib = ROOT / "tsfm-zig_amd" / "_build" / "san" / "libtsfm_attn_san.so"
    env = dict(os.environ, LD_PRELOAD=libs[-1], ASAN_OPTIONS="detect_leaks=0:halt_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1", TSFM_TEST_PRODUCT_LIB=str(lib))
    r = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-p", "no:cacheprovider", "-m", "not gpu",
                        "tests/test_kv8_abi.py"], cwd=ROOT, env=env, capture_output=True, text=True, timeout=1200)
    out = r.stdout + r.stderr
    assert r.returncode == 0 and "runtime error:" not in out and "AddressSanitizer" not in out, out[-4000:]
