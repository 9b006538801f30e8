"""Orders in the 4-bit kernels that no run can show to be missing without risking a hang or a read of
bytes that are not there yet: read from the sources."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "neuzip_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def body(text, name):
    start = text.index(name + "(")
    return text[start:text.index("\n}\n", start)]


def test_the_product_reads_inputs_only_behind_the_kernel_that_writes_them():
    text = source("nz_mx4_linear.cu")
    product = body(text, "mx4_product_kernel")
    copies = product[product.index("uint32_t early = 0;"):product.index("} else if (warp == 1)")]
    # W may be asked for before the wait, the inputs' codes only after it
    assert copies.index("load_w(w, k, early)") < copies.index("dependent_wait()") < copies.index("load_x(x, stage)")
    # everyone who uses tables, places or counters waits too
    assert product.count("dependent_wait();") == 3


def test_only_the_product_is_launched_early():
    # it begins to read W as soon as the kernel before it lets it in; that kernel must not itself have
    # been let in before everything older was complete
    text = source("nz_mx4_linear.cu")
    assert "launch_dependent(" not in text
    assert text.count("dependent_trigger();") == 1
    assert "dependent_trigger" not in body(text, "mx4_product_kernel")
    rows = body(text, "mx4_quantize_rows_kernel")
    assert "dependent_trigger();" in rows
    assert re.search(r"rows_kernel<<<", text)


def test_waits_in_the_product_are_bounded():
    text = source("nz_mx4_linear.cu")
    for call in re.finditer(r"mbar_try_wait\(|mbarrier\.try_wait", text):
        before = text[max(0, call.start() - 400):call.start()]
        assert "kMaxWaitIters" in before
