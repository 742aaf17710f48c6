"""How kernels that start before the one before them has ended are written, read from their sources on the host.

A kernel that was written the other way round may wait for ever, so what these rules forbid is not run."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fieldrun_b200", "csrc")
LETS_NEXT = re.compile(r"\b(let_next_kernel_start|after_previous_kernel)\(\)")
WAITS = re.compile(r"\b(wait_for_previous_kernel|after_previous_kernel)\(\)")
TAKES_COLUMNS = re.compile(r"\b(tmem_alloc|alloc_columns<\w+>)\(&")


def without_comments(text):
    return re.sub(r"//[^\n]*", "", re.sub(r"/\*.*?\*/", "", text, flags=re.S))


def body_at(text, at):
    """The braces' contents from the first brace at or behind `at`."""
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[start + 1:i]
    raise AssertionError("braces do not match")


def kernels():
    """(file and name, body) of every kernel."""
    found = []
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as handle:
            text = without_comments(handle.read())
        for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", text):
            depth, i = 1, m.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[i], 0)
                i += 1
            if text[i:].lstrip().startswith("{"):
                found.append((f"{os.path.basename(path)}:{m.group(1)}", body_at(text, i)))
    return found


KERNELS = dict(kernels())
WITH_COLUMNS = [name for name, body in KERNELS.items() if TAKES_COLUMNS.search(body)]


def test_the_kernels_are_found():
    assert len(KERNELS) > 100 and {name.split(":")[0] for name in WITH_COLUMNS} == {
        "attention_f32_tc.cu", "attention_pair_tc.cu", "attention_tc.cu", "delta_chunks.cu", "experts_tc.cu", "latent_attention_tc.cu", "products_8bit.cu",
        "products_f32.cu", "state_space_chunks.cu"}


@pytest.mark.parametrize("name", WITH_COLUMNS)
def test_a_kernel_with_tensor_memory_lets_the_next_one_start_only_once_it_has_its_columns(name):
    """Else the next kernel's block could take them first and wait for this kernel, whose block waits for the columns."""
    body = KERNELS[name]
    lets = LETS_NEXT.search(body)
    assert lets is None or lets.start() > TAKES_COLUMNS.search(body).end()


BOUNDED_WAIT = re.compile(r"\b(warp_wait|bar_wait|warp_wait_both)\(")


def roles(body):
    """The contents of a kernel's branches `if (warp == 0) {..} else if (warp == 1) {..} else {..}`."""
    at = re.search(r"\bif \(warp == 0\) \{", body).start()
    found = []
    while True:
        found.append(body_at(body, at))
        end = body.index(found[-1], at) + len(found[-1]) + 1
        follows = re.match(r"\s*else\b", body[end:])
        if not follows:
            return found
        at = end + follows.end()


def test_the_products_roles_wait_for_the_kernel_before_ahead_of_any_wait_with_a_limit():
    """A wait's limit of about a second is for the kernel's own copies and products: what the kernel before still does, beside which this one has
    started, must not be charged to it."""
    body = KERNELS["products_8bit.cu:product_8bit_kernel"]
    assert not BOUNDED_WAIT.search(body[:re.search(r"\bif \(warp == 0\) \{", body).start()])
    branches = roles(body)
    assert len(branches) == 3
    for branch in branches:
        assert WAITS.search(branch).start() < BOUNDED_WAIT.search(branch).start()


def test_every_early_start_asks_the_switch():
    """FIELDRUN_B200_PDL sets the largest grid that starts early, 0 none."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(path) as handle:
            text = without_comments(handle.read())
        assert text.count("cudaLaunchAttributeProgrammaticStreamSerialization") <= len(re.findall(r"<= (?:per_sm \* )?frb_dependent_launch_blocks\(\)", text)), path


@pytest.mark.parametrize("name", [name for name in KERNELS if name.split(":")[0] in ("rows_8bit.cu", "products_8bit.cu")])
def test_kernels_of_products_in_8_bits_let_the_next_one_start_behind_their_own_wait(name):
    """A product asks for weights and reads lists ahead of its wait: what wrote them, two kernels before, has ended by then only if the kernel between
    has waited for it first.  `early` is the callers' word that there is nothing to wait for."""
    body = KERNELS[name]
    waits = WAITS.search(body).start()
    for m in LETS_NEXT.finditer(body):
        assert m.start() > waits or body[:m.start()].rstrip().endswith("if (early)")


def test_rows_as_codes_let_the_product_start_early_only_where_its_weights_are_final():
    with open(os.path.join(CSRC, "linear_8bit.cu")) as handle:
        text = without_comments(handle.read())
    early = [re.sub(r"\s+", " ", call).split(", ")[-2] for call in re.findall(r"rows_codes\(([^;]*)\)\)", text)]
    assert early == ["in_chain || weights_final", "false", "true"]
    # behind the experts' first product, which has waited for the rows before it
    assert re.search(r"FRB_TRY\(product\(p, stream\)\);\s*FRB_TRY\(rows_codes\(hidden,[^;]*, true, stream\)\)", text)
