"""CPU check of which sources bench.py ties its traffic records to: those of the linears, which the records are of."""
import importlib.util
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def load():
    spec = importlib.util.spec_from_file_location("bench_sources", ROOT / "bench.py")
    bench = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(bench)
    return bench


def test_the_linears_sources_and_no_others():
    bench = load()
    names = {f.name for f in bench.kernel_sources()}
    csrc = {f.name for f in (ROOT / "vllm-exact_amd" / "csrc").iterdir() if f.is_file()}
    assert names == {n for n in csrc if n.startswith(("exact_", "digitize", "pack")) or n in ("capi.hip", "common.h", "noalloc.hip")}
    for n in names:  # none of them includes a source that is left out
        text = (ROOT / "vllm-exact_amd" / "csrc" / n).read_text()
        assert not any(f'"{other}"' in text for other in bench.OTHER_SOURCES), n


def test_the_hash_follows_the_linears_alone(tmp_path, monkeypatch):
    bench = load()
    csrc = tmp_path / "vllm-exact_amd" / "csrc"
    csrc.mkdir(parents=True)
    monkeypatch.setattr(bench, "ROOT", tmp_path)
    (csrc / "exact_gemm.hip").write_text("a")
    first = bench.kernel_sources_sha16()
    (csrc / "tree_decode.hip").write_text("b")
    assert bench.kernel_sources_sha16() == first
    (csrc / "exact_gemm.hip").write_text("c")
    assert bench.kernel_sources_sha16() != first
