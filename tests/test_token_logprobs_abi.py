"""CPU checks of the log probability entry: its struct as the header lays it out, host-side refusals."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_packed_args_match_header(tmp_path):
    from akv import _C
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "akv_b200.h"\nint main(void){\n'
                   'printf("%zu %zu\\n", sizeof(akv_logprobs_args), offsetof(akv_logprobs_args, dtype));return 0;}\n')
    exe = tmp_path / "s"
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    size, off = map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert (_C.LOGPROBS_ARGS.size, _C.LOGPROBS_ARGS.size - 4) == (size, off)


def test_host_refusals():
    """Bad arguments come back as codes before anything is launched."""
    from akv import _C
    lib = _C.load()

    def call(logits=256, tokens=256, out=256, n=1, vocab=10, top=0, dtype=2, ids=256):
        return lib.akv_token_logprobs(_C.LOGPROBS_ARGS.pack(logits, vocab, tokens, out, 256, 256, ids, 256, n, vocab,
                                                            top, dtype), None)

    assert lib.akv_token_logprobs(None, None) == -7
    assert call(logits=0) == -7 and call(tokens=0) == -7 and call(out=0) == -7 and call(top=1, ids=0) == -7
    assert call(n=-1) == -1 and call(vocab=0) == -1 and call(top=33, vocab=99) == -1 and call(top=11) == -1
    assert call(top=-1) == -1 and call(n=(1 << 28) + 1) == -1 and call(vocab=2 ** 31 - 1) == -1
    assert call(dtype=3) == -4 and call(logits=258) == -3 and call(logits=257, dtype=0) == -3 and call(n=0) == 0
