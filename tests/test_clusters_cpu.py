"""Shared memory of another CTA is touched only where that CTA is known to run, and none leaves while its own may still be touched: what a
barrier of the cluster says.  Read from the sources, since a kernel without one would nearly always get away with it."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "pratchya_b200" / "csrc"
ENDED = r"cluster\.sync\(\)|cluster_sync_all\(\)|cluster_all_here\(\)|barrier\.cluster\.wait"


def _kernels():
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for m in re.finditer(r"__global__[^;{]*?\b(\w+_kernel)\(((?:[^{};]|\{[^}]*\})*?)\)\s*\{\n", text):
            yield path.name, m.group(1), text[m.end():text.index("\n}\n", m.end())]


def test_remote_shared_memory_lies_between_barriers():
    seen = []
    for name, kernel, body in _kernels():
        first = re.search(r"cluster\.map_shared_rank\(", body)
        if not first:
            continue
        seen.append(kernel)
        before, last = body[:first.start()], body.rindex("cluster.map_shared_rank(")
        assert re.search(ENDED, before), f"{name}: {kernel} touches another CTA's shared memory before it knows that this one runs"
        assert re.search(ENDED, body[last:]), f"{name}: {kernel} may leave while its shared memory is in use"
        assert body.count("cluster_here()") == body.count("cluster_all_here()"), f"{name}: {kernel} begins a barrier that it does not end"
        if "cluster_here()" in body:
            assert body.index("cluster_here()") < body.index("cluster_all_here()")
    assert sorted(seen) == ["int4_product_kernel", "token_logprobs_kernel"]
