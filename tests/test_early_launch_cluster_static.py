"""As tests/test_early_launch_static.py, for kernels launched early in clusters: every kernel passed to
launch_pdl_cluster calls pdl_wait() in its body."""
import re

from test_early_launch_static import CSRC, _kernel_body, _resolve


def test_every_kernel_launched_early_in_clusters_waits():
    found = set()
    for f in sorted(CSRC.glob("*.cu")):
        text = f.read_text()
        for m in re.finditer(r"launch_pdl_cluster\(\s*([A-Za-z_]\w*)", text):
            kernel = _resolve(text, m.group(1))
            body = _kernel_body(text, kernel)
            assert body is not None, f"{f.name}: kernel {kernel} not found"
            assert "pdl_wait()" in body, f"{f.name}: {kernel} is launched early without pdl_wait()"
            found.add(kernel)
    assert found >= {"token_logprobs_kernel", "gated_rows_kernel"}, found
