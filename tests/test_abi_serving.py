"""CPU tests of the serving entry points' ABI: no engine, no call; the structs the
binding passes are laid out as the header's."""
import ctypes as C
import os
import subprocess

from conftest import ROOT


def test_null_engine_is_rejected(tla):
    lib = tla.lib()
    cache, rules = tla.PagedCache(), tla.LogitRules()
    one = (C.c_int * 1)(0)
    calls = {
        "tla_paged_cache_alloc": (None, 1, 16, tla.KV_F16, C.byref(cache)),
        "tla_paged_append": (None, C.byref(cache), 1, one, None, 0, 0, None, None),
        "tla_paged_attention": (None, C.byref(cache), 1, one, None, 0, 0, None, None),
        "tla_logits_process": (None, 1, 1, C.byref(rules), None, None, None),
    }
    for name, args in calls.items():
        assert getattr(lib, name)(*args) == tla.TLA_ERR_INVALID_ARGUMENT, name
        assert tla.last_error() == "engine is NULL"


def test_struct_layouts_match_the_header(tla, tmp_path):
    fields = {"tla_paged_cache": (tla.PagedCache, {"table": "table_dev"}),
              "tla_logit_rules": (tla.LogitRules, {f: f + "_dev" for f in ("history", "history_len", "penalties", "bias_token",
                                                                           "bias_value", "bias_len", "mask")})}
    src = "#include <stdio.h>\n#include \"tla_attention.h\"\nint main(void) {\n"
    want = []
    for struct, (cls, names) in fields.items():
        src += f'printf("%zu\\n", sizeof({struct}));\n'
        want.append(C.sizeof(cls))
        for name, _ in cls._fields_:
            src += f'printf("%zu\\n", offsetof({struct}, {names.get(name, name)}));\n'
            want.append(getattr(cls, name).offset)
    (tmp_path / "layout.c").write_text(src + "return 0;\n}\n")
    exe = str(tmp_path / "layout")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want
