"""The key-value cache's entry points without a device: what they refuse before touching it, and the structs that the binding packs."""
import ctypes
import errno
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from bam_amd import _lib
    if not os.path.exists(_lib.lib_path()):
        pytest.skip("libbam_amd.so not built here (needs hipcc): build() compiles it")
    return _lib.load()


def test_null_handles_are_refused(lib):
    from bam_amd import kv
    h, n, info = ctypes.c_void_p(), ctypes.c_uint64(7), (ctypes.c_uint64 * 4)()
    zeros = {s: bytes(s.size) for s in (kv._READ, kv._APPEND, kv._ATTEND)}
    calls = {
        "bam_kv_create": (ctypes.byref(h), None, 0, 1, 1, 64, 0),
        "bam_kv_info": (None, info),
        "bam_kv_append": (None, zeros[kv._APPEND], None),
        "bam_kv_read": (None, zeros[kv._READ], None, None, None),
        "bam_kv_attend_bytes": (None, 1, 1, 1, 1, 0, 0, ctypes.byref(n)),
        "bam_kv_attend": (None, zeros[kv._ATTEND], None),
    }
    for name, args in calls.items():
        assert getattr(lib, name)(*args) == errno.EINVAL, name
        message = lib.bam_last_error()
        assert name.encode() in message and b"null" in message, (name, message)
    assert not h.value and n.value == 7 and not any(info)
    lib.bam_kv_destroy(None)      # like free(NULL)


SEQS = ("seqs.n_rows", "seqs.n_seqs", "seqs.d_starts", "seqs.d_lens", "seqs.d_table", "seqs.table_stride", "seqs.table_width")
MEMBERS = {
    "bam_kv_append_t": SEQS + ("d_k", "k_row", "k_head", "d_v", "v_row", "v_head", "d_q", "q_row", "q_head", "d_q_out", "d_q_norm", "d_k_norm", "d_cos", "d_sin",
                               "n_positions", "q_heads", "rot", "eps", "pairs"),
    "bam_kv_attend_t": SEQS + ("d_q", "q_row", "q_head", "d_out", "d_lse", "d_work", "work_bytes", "max_new", "max_len", "q_heads", "window", "sinks", "scale"),
}


def test_packed_structs_are_the_headers(tmp_path):
    """a C program prints the members of structs that were packed from 1, 2, 3, ..."""
    from bam_amd import kv
    formats = {"bam_kv_append_t": kv._APPEND, "bam_kv_attend_t": kv._ATTEND}
    code = ['#include <stdio.h>', '#include "bam_amd.h"', 'int main(int argc, char** argv) { FILE* f; (void)argc;', 'printf("%zu\\n", sizeof(bam_kv_seqs_t));']
    files = []
    for k, (name, members) in enumerate(MEMBERS.items()):
        path = tmp_path / name
        path.write_bytes(formats[name].pack(*range(1, len(members) + 1)))
        files.append(str(path))
        code.append('{ %s s; f = fopen(argv[%d], "rb"); printf("%%zu %%d", sizeof s, (int)(fread(&s, 1, sizeof s, f) == sizeof s && fgetc(f) == EOF)); fclose(f);' % (name, k + 1))
        code += ['printf(" %%d", (int)%ss.%s);' % ("(size_t)" if m.split(".")[-1].startswith("d_") else "", m) for m in members]
        code.append('printf("\\n"); }')
    code.append("return 0; }")
    src, exe = tmp_path / "members.c", tmp_path / "members"
    src.write_text("\n".join(code))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)] + files, check=True, capture_output=True, text=True).stdout.splitlines()
    assert int(lines[0]) == kv._READ.size
    for line, (name, members) in zip(lines[1:], MEMBERS.items()):
        size, whole, *values = (int(x) for x in line.split())
        assert size == formats[name].size and whole == 1 and values == list(range(1, len(members) + 1)), (name, line)
    assert len(lines) == 1 + len(MEMBERS)
