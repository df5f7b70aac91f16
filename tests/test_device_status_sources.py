"""How kernels report and how the host takes it: what no run shows reliably, since a breach is two blocks in one instant or a call
that overtakes a memset."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flat-attention_b200", "csrc")


def text(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_kernels_write_the_status_word_through_one_function_only():
    """Code and place in one atomic maximum: two plain stores of two blocks can pair one's code with the other's place, and the
    last one hides what was there."""
    files = [os.path.basename(f) for f in glob.glob(os.path.join(CSRC, "*.cu*")) + glob.glob(os.path.join(CSRC, "*.h"))]
    assert len(files) > 15
    for name in files:
        src = text(name)
        assert not re.search(r"status\s*(?:->|\.)\s*(?:code|where|word)\s*=[^=]", src), name
        if name != "common.h":
            assert not re.search(r"(?:atomic\w+\(|red\.|\bst\.)[^;]*status", src), name
    body = text("common.h")
    body = body[body.index("void report_status("):]
    body = body[:body.index("}\n")]
    assert body.count(";") == 1 and "atomicMax(&status->word," in body and re.search(r"code << 48 \|[^;]*where\)", body)


def test_a_wait_that_gave_up_has_the_largest_code_that_kernels_report():
    header = open(os.path.join(os.path.dirname(CSRC), "..", "include", "flat_attention_b200.h")).read()
    codes = {name: int(v) for name, v in re.findall(r"(FLAT_ERR_\w+) = (\d+)", header)}
    used = set()
    for f in glob.glob(os.path.join(CSRC, "*.cu*")):
        for call in re.findall(r"report_status\([^;]*;", open(f).read()):
            used |= set(re.findall(r"FLAT_ERR_\w+", call))
    assert "FLAT_ERR_DEVICE_WAIT_TIMEOUT" in used and "FLAT_ERR_PAGE_OUT_OF_RANGE" in used
    assert max(used, key=codes.get) == "FLAT_ERR_DEVICE_WAIT_TIMEOUT"


def test_reading_the_status_clears_in_stream_order_and_waits():
    """A memset of the legacy stream is not ordered before the next launch on a stream that does not synchronise with it."""
    src = text("abi.cu")
    body = src[src.index("int32_t flat_ctx_device_status("):]
    body = body[:body.index("\n}")]
    assert "cudaMemset(" not in body
    clears = [m.start() for m in re.finditer(r"cudaMemsetAsync\([^;]*ctx->stream\)", body)]
    assert len(clears) == 2 and body.rindex("cudaStreamSynchronize(ctx->stream)") > clears[-1]
