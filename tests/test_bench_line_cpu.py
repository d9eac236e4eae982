"""The line that bench.py prints: whole, and short enough for the end of a log."""
import json
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

REQUIRED = ("metric", "value", "unit", "n_gpus", "steps", "warmup", "ms_per_step", "higher_is_better", "scaling",
            "vs_baseline", "dtype", "data", "config", "e2e", "gpu_launches", "clocks")


def test_the_line_fits_the_end_of_a_log_and_keeps_what_is_read_from_it():
    import bench
    table = {f"kernel_{i}": {"ms": 0.0123456789012345, "bound": "hbm", "achieved": 1234.56789012345} for i in range(8)}
    config = dict.fromkeys(("workload", "model", "weights", "n_seq", "n_prompt", "parallelism", "l2"), "a text of forty letters and so on, x" * 1)
    roof = {"kernel": "decode_attention", "bound": "hbm", "achieved": 5493.8616040798925, "peak": 6539.9, "unit": "GB/s",
            "frac": 0.8400528454685687, "traffic": 462142208, "peak_source": "measured", "work_per_launch": 454557696}
    line = {k: 918.123456789012 for k in REQUIRED}
    line.update(metric="GPT-2 prefill & decode tokens/s at 1/2/4/8 B200; % of HBM/tensor roofline", unit="tokens/s",
                data="synthetic (seeded random-init weights, seeded uniform token ids)", config=config, e2e=roof, clocks=roof,
                roofline=roof, step_roofline=roof, kernels=table, phases=table, peaks=table,
                workloads={n: {"value": 124838.77214301389, "kernels": table} for n in bench.SUITE},
                cpu_baseline={"value": 48.4, "unit": "tokens/s", "cores": 16, "kind": "port", "sample": "x" * 400,
                              "contexts": [1, 2, 3]}, results_record="bench_results/gpt2_throughput_n1.json",
                details="bench_results/gpt2_throughput_n1_details.json")
    text = json.dumps(bench.short_line(line))
    assert len(text) <= 2900 and "\n" not in text
    out = json.loads(text)
    for k in REQUIRED + ("roofline",):
        assert out[k] == line[k]
    assert set(out["workloads"]) == set(bench.SUITE) and abs(out["workloads"][bench.SUITE[0]] - 124838.77) < 1
    assert out["cpu_baseline"]["value"] == 48.4
