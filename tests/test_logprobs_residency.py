"""token_logprobs sizes its grid for 1024 threads per SM: its CTAs have to fit there together, with their static shared
memory as ptxas reports it, the ring they are launched with, and the 1 KiB that the system takes for each (of 228 KiB)."""
import re
import subprocess

from bee_b200 import build


def test_forward_ctas_fit_together(tmp_path):
    r = subprocess.run([build.NVCC, *build.ARCH, *build.NVCC_FLAGS, "-Xptxas", "-v", "-c", str(build.CSRC / "logprobs.cu"),
                        "-o", str(tmp_path / "logprobs.o")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, check=True)
    found = 0
    for entry in r.stdout.split("Compiling entry function")[1:]:
        kernel = re.search(r"'\S*token_logprobs_kernelI\S+?Li(\d+)ELb[01]", entry.split("\n")[0])
        if not kernel:
            continue
        threads, used = int(kernel.group(1)), re.search(r"Used (\d+) registers.*?(\d+) bytes smem", entry)
        registers, static = int(used.group(1)), int(used.group(2))
        ring = 16 * 3 * 4 * threads  # three batches of four 16-byte chunks a thread
        ctas = 1024 // threads
        assert (static + ring + 1024) * ctas <= 228 * 1024, entry.split("\n")[0]
        assert registers * 1024 <= 65536, entry.split("\n")[0]
        found += 1
    assert found == 12  # three types, two blocks, with and without alternatives
