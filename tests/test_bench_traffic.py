"""The benchmark's measured traffic: quoted where the kernels are the ones it was measured on, whatever
other operators the library has."""
import bench


def _lines():
    for md in sorted((bench.ROOT / "profiles").glob("*.md")):
        for line in md.read_text().splitlines():
            m = bench._TRAFFIC_LINE.match(line.strip())
            if m:
                yield m.groups()


def test_figures_of_the_summaries_are_quoted():
    lines = list(_lines())
    assert len(lines) >= 10
    for workload, kernel, nbytes, digest in lines:
        assert bench.measured_traffic(workload, kernel)[0] == int(nbytes), (workload, kernel, digest)


def test_only_the_measured_kernels_sources_count(tmp_path, monkeypatch):
    from raf_amd import build

    sources = list(build.OPTIM_SOURCES)
    for f in [build.CSRC / s for s in sources] + list(build.CSRC.glob("*.h")):
        (tmp_path / f.name).write_text(f.read_text())
    here = bench.kernel_sources_digest()
    monkeypatch.setattr(build, "CSRC", tmp_path)
    assert bench.kernel_sources_digest() == here
    for name in sorted(bench._NOT_MEASURED):
        with open(tmp_path / name, "a") as f:
            f.write("\nint another;\n")
        assert bench.kernel_sources_digest() == here, name
    for name in ("lans_kernels.hip", "lans_kernels.h", "sgd.hip", "device_table.h"):
        before, text = bench.kernel_sources_digest(), (tmp_path / name).read_text()
        (tmp_path / name).write_text(text + "\n// a comment\n")
        assert bench.kernel_sources_digest() == before, name
        (tmp_path / name).write_text(text + "\nint another;\n")
        assert bench.kernel_sources_digest() != before, name
    # nothing that counts includes what does not
    for name in sources:
        if name not in bench._NOT_MEASURED:
            assert not any(f'"{x}"' in (tmp_path / name).read_text() for x in bench._NOT_MEASURED), name
