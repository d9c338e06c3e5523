"""The entry points of the key-value cache in 8 bits, of its reordering and of beam search's selection without a device: what they refuse before touching it, and the structs that the bindings pack."""
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


def _refused(lib, name, *args, about=b""):
    assert getattr(lib, name)(*args) == errno.EINVAL, (name, args)
    message = lib.bam_last_error()
    assert name.encode() in message and about in message, (name, args, message)


def test_null_arguments_are_refused(lib):
    from bam_amd import beam, kv
    h, n = ctypes.c_void_p(), ctypes.c_uint64(7)
    _refused(lib, "bam_kv_create_e4m3", ctypes.byref(h), None, 0, 1, 1, 64, 0, 16, 1 << 20, about=b"null")
    _refused(lib, "bam_kv_create_e4m3", None, None, 0, 1, 1, 64, 0, 16, 1 << 20, about=b"null")
    _refused(lib, "bam_kv_reorder", None, bytes(kv._REORDER.size), None, about=b"null")
    _refused(lib, "bam_beam_select", None, None, about=b"null")
    _refused(lib, "bam_beam_select_bytes", 1, 1, 10, 1, 0, None, about=b"null")
    assert not h.value and n.value == 7
    good = [1, 2, 100, 64, 100, 64, 2, 64, 64, 64, 64, 1 << 30, 4, 0]
    for i in (3, 5, 7, 8, 9, 10):
        _refused(lib, "bam_beam_select", beam._SELECT.pack(*[0 if j == i else x for j, x in enumerate(good)]), None, about=b"null")


def test_sizes_that_do_not_fit_are_refused(lib):
    from bam_amd import beam
    n = ctypes.c_uint64(7)
    # requests, beams, vocab, width, type
    for sizes, about in (((1, 0, 10, 1, 0), b"beams"), ((1, 1025, 10, 1, 0), b"beams"), ((1, 2, 0, 1, 0), b"tokens"), ((1, 2, 10, 0, 0), b"width"), ((1, 2, 10, 21, 0), b"width"), ((1, 2, 1000, 257, 0), b"width"),
                         ((1, 2, 10, 1, 3), b"type"), ((1, 2, 10, 1, -1), b"type"), ((1, 2, 1 << 30, 1, 0), b"31 bits"), ((1 << 31, 1, 10, 1, 0), b"31 bits"), ((1, 1, 1 << 40, 1, 0), b"31 bits")):
        _refused(lib, "bam_beam_select_bytes", *sizes, ctypes.byref(n), about=about)
        requests, beams, vocab, width, kind = sizes
        _refused(lib, "bam_beam_select", beam._SELECT.pack(requests, beams, vocab, 64, vocab, 64, beams, 64, 64, 64, 64, 1 << 40, width, kind), None, about=about)
    assert n.value == 7
    # a workspace for what there is to do: the pieces' keys at least, and nothing where there is nothing
    for sizes in ((1, 4, 32000, 8, 0), (32, 4, 128000, 8, 1), (48, 16, 150001, 32, 2), (1, 1024, 7, 256, 2), (1, 1, 1, 1, 0)):
        assert lib.bam_beam_select_bytes(*sizes, ctypes.byref(n)) == 0 and n.value >= sizes[0] * sizes[1] * sizes[3] * 8, sizes
        requests, beams, vocab, width, kind = sizes
        _refused(lib, "bam_beam_select", beam._SELECT.pack(requests, beams, vocab, 64, vocab, 64, beams, 64, 64, 64, 64, n.value - 1, width, kind), None, about=b"workspace")
        _refused(lib, "bam_beam_select", beam._SELECT.pack(requests, beams, vocab, 64, vocab, 64, beams, 64, 64, 64, 72, n.value, width, kind), None, about=b"aligned")
    assert lib.bam_beam_select_bytes(0, 4, 100, 4, 0, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.bam_beam_select(beam._SELECT.pack(0, 4, 100, 0, 0, 0, 0, 0, 0, 0, 0, 0, 4, 0), None) == 0


MEMBERS = {
    "bam_kv_reorder_t": ("n_old", "n_new", "d_parents", "d_lens", "d_table", "table_stride", "table_width", "d_spare", "d_lens_out", "d_table_out", "d_spare_out", "d_work", "work_bytes"),
    "bam_beam_select_t": ("n_requests", "n_beams", "vocab", "d_logits", "logits_row", "d_scores", "scores_row", "d_sums", "d_beams", "d_tokens", "d_work", "work_bytes", "width", "type"),
}


def test_packed_structs_are_the_headers(tmp_path):
    """a C program prints the members of structs that were packed from 1, 2, 3, ..."""
    from bam_amd import beam, kv
    formats = {"bam_kv_reorder_t": kv._REORDER, "bam_beam_select_t": beam._SELECT}
    code, files = ['#include <stdio.h>', '#include "bam_amd.h"', 'int main(int argc, char** argv) { FILE* f; (void)argc;'], []
    for k, (name, members) in enumerate(MEMBERS.items()):
        path = tmp_path / name
        path.write_bytes(formats[name].pack(*range(1, len(members) + 1)))
        files.append(str(path))
        code.append('{ %s s; f = fopen(argv[%d], "rb"); printf("%%zu %%d", sizeof s, (int)(fread(&s, 1, sizeof s, f) == sizeof s && fgetc(f) == EOF)); fclose(f);' % (name, k + 1))
        code += ['printf(" %%d", (int)%ss.%s);' % ("(size_t)" if m.startswith("d_") else "", m) for m in members]
        code.append('printf("\\n"); }')
    code.append("return 0; }")
    src, exe = tmp_path / "members.c", tmp_path / "members"
    src.write_text("\n".join(code))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    lines = subprocess.run([str(exe)] + files, check=True, capture_output=True, text=True).stdout.splitlines()
    for line, (name, members) in zip(lines, MEMBERS.items()):
        size, whole, *values = (int(x) for x in line.split())
        assert size == formats[name].size and whole == 1 and values == list(range(1, len(members) + 1)), (name, line)
    assert len(lines) == len(MEMBERS)
