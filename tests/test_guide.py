"""The C examples of the guides compile against the headers as they stand
(what they leave out, their callers' variables, is declared here)."""
import glob
import os
import re
import subprocess

import pytest

import harness

CALLER = """#include <stdint.h>
#include <stdlib.h>
#include "kllm_cuda.h"
void example(kllm_chip *chip, const int *prompt, const int *prompts, int *lens, int n, int max_new, int eos,
             int *out, int n_out, int rank, int world, void *all);
void example(kllm_chip *chip, const int *prompt, const int *prompts, int *lens, int n, int max_new, int eos,
             int *out, int n_out, int rank, int world, void *all)
{
    {   /* an example may declare variables of the same names */
%s
    }
}
"""


def _examples():
    for path in sorted(glob.glob(os.path.join(harness.ROOT, "*.md"))):
        for code in re.findall(r"```c\n(.*?)```", open(path).read(), flags=re.S):
            if "kllm_" in code:
                yield pytest.param(code, id="%s-%s" % (os.path.basename(path), re.findall(r"kllm_\w+\(", code)[0][:-1]))


@pytest.mark.parametrize("code", list(_examples()))
def test_example_compiles(code, tmp_path):
    code = "\n".join(l for l in code.split("\n") if not l.startswith("#include"))
    src = tmp_path / "example.c"
    src.write_text(CALLER % code)
    r = subprocess.run(["gcc", "-std=c11", "-fsyntax-only", "-Wall", "-Werror", "-Wno-unused",
                        "-I" + os.path.join(harness.ROOT, "include"), str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
