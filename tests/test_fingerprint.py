"""CPU: the stamp that ties a traffic measurement of the GEMM kernels to their sources changes with those and with no others."""
import shutil

from fitclip_amd import build


def test_the_fingerprint_is_that_of_the_measured_kernels_sources(tmp_path):
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    for path in [*build.CSRC.glob("*.hip"), *build.CSRC.glob("*.h"), *build.CSRC.glob("*.cpp")]:
        shutil.copy(path, csrc)
    was = build.source_fingerprint(csrc)
    assert was == build.source_fingerprint()
    for name, counts in (("attention_docs.hip", False), ("attention_docs.h", False), ("rotary.hip", False), ("api.hip", False), ("gemm.hip", True),
                         ("gemm_split2.h", True), ("gemm_split3.hip", True), ("gemm_kernel.h", True), ("common.h", True)):
        path = csrc / name
        kept = path.read_text()
        path.write_text(kept + "// one line more\n")
        assert (build.source_fingerprint(csrc) != was) == counts, name
        path.write_text(kept)
    assert build.source_fingerprint(csrc) == was
