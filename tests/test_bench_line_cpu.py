"""The benchmark's printed line: whole within 3,000 characters, with every
key that says what was measured."""
import json

from conftest import ROOT


def _record():
    """A record with every part, numbers and texts as long as they get."""
    x = 123456789.12345678
    group = {"bound": "tensor", "achieved": x, "peak": x, "unit": "TFLOP/s", "frac": 0.12345678901234567,
             "peak_source": "measured bf16 sustained", "ms_per_step": x, "launches_per_step": x, "flops_per_launch": x,
             "kernels": ["node_gemm", "gemm_small"], "operands": "split bf16 (hi*hi + hi*lo + lo*hi)",
             "flops": "20 H^2 per node and layer (data GEMMs)"}
    names = ["edge_fwd", "edge_bwd", "edge_rows_gemm", "edge_rows_wgrad", "node_gemm", "node_wgrad", "node_pass", "src_pass",
             "edge_rows_u", "edge_rows_agg"]
    line = {"metric": "egnn_train_layer_edges_per_s", "value": x, "unit": "layer-edges/s", "n_gpus": 1, "steps": 1000,
            "warmup": 100, "ms_per_step": x, "higher_is_better": True, "scaling": "strong", "vs_baseline": None,
            "dtype": "bf16", "data": "synthetic (seeded generators, random init)",
            "config": {"workload": "config2", "graphs_per_gpu": 512, "nodes_per_gpu": 1048576, "edges_per_gpu": 33554432,
                       "layers": 7, "hidden": 128, "precision": "bf16", "l2": "flushed between timed steps (252 MB write)",
                       "parallelism": "nodepart8", "optimizer": "Muon on the matrices, SGD on the rest", "node_norm": True,
                       "allreduce": "per-layer buckets, issued as the backward produces them", "cuda_graph": True},
            "molecules_per_s": x, "model_tflops": x,
            "e2e": {"value": x, "unit": "layer-edges/s", "ms_per_step": x, "h2d_bytes_per_step": 10 ** 10,
                    "d2h_bytes_per_step": 4, "molecules_per_s": x, "path": "p" * 250,
                    "eager": {"value": x, "ms_per_step": x, "path": "p" * 200}},
            "gpu_launches": 10 ** 6,
            "roofline": {**group, "kernel": "edge_rows_wgrad", "per_launch_ms": x, "launches": 10 ** 6, "traffic": 10 ** 10,
                         "traffic_unit": "bytes per launch (ncu capture)", "groups": {n: dict(group) for n in names}},
            "kernel_ms_per_step": {f"kernel_{i}": x for i in range(24)},
            "cpu_baseline": {"value": x, "unit": "layer-edges/s", "cores": 128, "kind": "port", "molecules_per_s": x,
                             "step_s": x, "sample": "s" * 200},
            "clocks": {"sm_mhz": 1965.0, "sm_max_mhz": 1965.0, "reasons": ["sw_power_cap"], "samples": 1000,
                       "power_w_max": 999.99},
            "device_status": "error", "peak_vram_gb": x}
    extra = {k: v for k, v in line.items() if k not in ("metric", "unit", "e2e", "data", "n_gpus", "warmup")}
    line["extras"] = {f"config{c}_{p}": json.loads(json.dumps(extra)) for c, p in
                      [(2, "fp32"), (1, "bf16"), (3, "fp32"), (4, "bf16"), (5, "bf16"), (3, "bf16")]}
    return line


def test_printed_line_is_whole_where_the_last_3000_characters_are_kept():
    import sys
    sys.path.insert(0, str(ROOT))
    import bench
    record = _record()
    assert len(json.dumps(record)) > 10000
    text = json.dumps(bench.printed(record))
    assert len(text) < 2900, len(text)
    got = json.loads(text)
    for k in ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling",
              "vs_baseline", "dtype", "data", "gpu_launches", "config", "clocks", "device_status"):
        assert got[k] == record[k], k
    for k in ("unit", "h2d_bytes_per_step", "d2h_bytes_per_step"):
        assert got["e2e"][k] == record["e2e"][k]
    assert abs(got["e2e"]["value"] / record["e2e"]["value"] - 1) < 1e-5
    assert set(got["extras"]) == set(record["extras"]) and set(got["roofline"]["groups"]) == set(record["roofline"]["groups"])
    assert bench.printed({"e2e": None, "value": 1.0}) == {"e2e": None, "value": 1.0}   # runs without those parts
