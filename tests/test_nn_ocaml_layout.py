"""The argument blocks in ocaml/ccb.ml (not compiled here) against include/ccb.h:
the same fields in the same order and of the same C types."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CTYPES = {"ptr void": "pointer", "llong": "long long", "ullong": "unsigned long long", "double": "double", "int": "int"}


def read(*p):
    with open(os.path.join(ROOT, *p)) as f:
        return f.read()


def header_fields(name):
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", read("include", "ccb.h")).group(1)
    out = []
    for line in filter(None, (v.strip() for v in body.split(";"))):
        kind = "pointer" if "*" in line else re.match(r"(unsigned long long|long long|double|int)\b", line).group(1)
        for field in re.sub(r"\b(const|void|int|unsigned|long|double)\b", " ", line).replace("*", " ").split(","):
            out.append((field.strip(), kind))
    return out


def ocaml_fields(name):
    return [(n, CTYPES[t]) for n, t in re.findall(r"^let \w+ = field " + name + r" \"(\w+)\" \(?([a-z ]+?)\)?$", read("ocaml", "ccb.ml"), re.M)]


BLOCKS = sorted(set(re.findall(r"\} (ccb_nn_\w+_t);", read("include", "ccb.h"))))


def test_every_block_is_there():
    assert len(BLOCKS) == 5
    assert sorted(re.findall(r'structure "(ccb_nn_\w+_t)"', read("ocaml", "ccb.ml"))) == BLOCKS


@pytest.mark.parametrize("block", BLOCKS)
def test_fields(block):
    want = header_fields(block)
    assert len(want) > 10 and ocaml_fields(block[len("ccb_"):]) == want
    src = read("ocaml", "ccb.ml")
    assert src.index(f"let () = seal {block[4:]}") > max(m.start() for m in re.finditer(f"field {block[4:]} ", src))
