"""Hardware profile and hash-bound run reports for the hip_gemm specialization.

Two pieces, each after a reference format:

* The device profile follows the schema_version 1 target description of the
  reference's Hardware/profile.py:1-25 (same required keys, canonical JSON,
  SHA-256 hash, validation, prompt rendering and the rule that an unknown
  feature never authorises anything, profile.py:410-510) with a "hip"
  backend, which the reference lacks (it probes Metal and CUDA only,
  profile.py:180-265, :350-380). The probe goes through the library's
  vt_device_query (hipGetDeviceProperties, hipRuntimeGetVersion) instead of
  a driver library loaded with ctypes, and it returns None when there is no
  library or no device, as the reference's probe does.

* A run report binds one GEMM result to everything that produced it, like
  the Spike report of specializations/gemmini_gemm/runtime/run_spike.py:77-111
  and the demo report of examples/gemmini_gemm_demo.py:27-113: sha256 of the
  native library, its sources and the Python modules; the device profile and
  its hash; the plan and its digest; sha256 of every operand's raw bytes; the
  verification outcome. Outputs small enough to list are also hashed in the
  reference's own list format (sha256 of json.dumps of the flat int list,
  check_local_execution.py:53), so a report can be compared with the
  reference's recorded output hashes directly.

The verification is the exact projection check of verify.py, on the GPU; a
report never claims more than that check establishes.
"""
from __future__ import annotations

import hashlib
import json
import os
import sys

from ... import _lib
from ..._lib import HipGemmError
from . import backend as _backend
from . import verify as _verify

SCHEMA_VERSION = 1
REPORT_SCHEMA_VERSION = 1
BACKENDS = ("metal", "cuda", "hip")
LIST_DIGEST_MAX_ELEMENTS = 1 << 22

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(os.path.dirname(PKG_DIR)))

# Features a gfx950 code object of this library executes on every GEMM:
# MFMA integer matrix ops (v_mfma_i32_32x32x32_i8 / 16x16x64_i8), direct
# global-to-LDS loads (global_load_lds_dwordx4) and LDS transpose reads
# (ds_read_b64_tr_b8). fp16 / bfloat16 MFMA are in the same ISA.
GFX950_FEATURES = ("matrix_ops", "int8_matrix_ops", "async_copy", "lds_transpose_read",
                   "fp16", "bfloat16")


# ---------------------------------------------------------------------------
# Device profile
# ---------------------------------------------------------------------------

def _hostname():
    try:
        return os.uname().nodename or "unknown"
    except Exception:
        return "unknown"


def hip_version_string(v):
    """HIP_VERSION encoding major*10^7 + minor*10^5 + patch -> "major.minor.patch"."""
    if not isinstance(v, int) or isinstance(v, bool) or v <= 0:
        return "unknown"
    return "%d.%d.%d" % (v // 10_000_000, (v // 100_000) % 100, v % 100_000)


def _target_flag(arch, name):
    """True / False for "name+" / "name-" in a gcnArchName, None if absent."""
    for part in arch.split(":")[1:]:
        if part == name + "+":
            return True
        if part == name + "-":
            return False
    return None


def normalize_hip(raw, host=None):
    """vt_device_query fields -> a schema_version 1 profile with backend "hip".

    A feature is True only when the device's ISA is the library's code-object
    target (raw["supported"]); otherwise it stays None (unknown).
    """
    supported = bool(raw.get("supported"))
    arch = raw.get("arch") or ""
    # The runtime leaves the marketing name empty where the driver does not
    # expose it (containers without the board's product string); the ISA and
    # CU count then name the device, and device_name_source says so.
    name = (raw.get("name") or "").strip()
    name_source = "hip_runtime"
    if not name and arch:
        name = "AMD %s (%s CUs)" % (arch.split(":")[0], raw.get("compute_units"))
        name_source = "gcn_arch_name"
    features = {name: (True if supported else None) for name in GFX950_FEATURES}
    features["xnack"] = _target_flag(arch, "xnack")
    features["sramecc"] = _target_flag(arch, "sramecc")
    return {
        "schema_version": SCHEMA_VERSION,
        "backend": "hip",
        "device_name": name,
        "device_name_source": name_source,
        "max_threads_per_threadgroup": raw.get("max_threads_per_workgroup"),
        "max_threadgroup_memory_bytes": raw.get("lds_per_workgroup_bytes"),
        "simd_width": raw.get("wavefront_size"),
        "gcn_arch_name": arch,
        "compute_units": raw.get("compute_units"),
        "lds_per_cu_bytes": raw.get("lds_per_cu_bytes"),
        "l2_cache_size_bytes": raw.get("l2_cache_bytes"),
        "total_device_memory_bytes": raw.get("total_memory_bytes"),
        "max_clock_khz": raw.get("max_clock_khz"),
        "memory_clock_khz": raw.get("memory_clock_khz"),
        "memory_bus_width_bits": raw.get("memory_bus_width_bits"),
        "pci": {"domain": raw.get("pci_domain"), "bus": raw.get("pci_bus"),
                "device": raw.get("pci_device")},
        "toolchain": {"name": "hip_runtime",
                      "version": hip_version_string(raw.get("hip_runtime_version")),
                      "driver_version": raw.get("hip_driver_version"),
                      "code_target": raw.get("code_object_arch") or None},
        "provenance": {"source": "hip_device_query", "host": host or _hostname()},
        "features": features,
    }


def probe(device=-1):
    """Profile of a HIP device (default: the current one), or None when the
    library cannot be loaded or no device answers (profile.py:350-380)."""
    try:
        raw = _lib.device_query(device)
    except HipGemmError:
        return None
    profile = normalize_hip(raw)
    try:
        validate_schema(profile)
    except ValueError:
        return None
    return profile


def make_hip_profile(device_name="AMD Instinct MI355X", compute_units=256,
                     lds_bytes=160 * 1024, simd_width=64, arch="gfx950:sramecc+:xnack-",
                     supported=True, runtime_version=70051831, host="localhost"):
    """A normalised profile from explicit values (for tests and offline use)."""
    return normalize_hip({
        "name": device_name, "arch": arch, "code_object_arch": "gfx950",
        "total_memory_bytes": 288 * 1024 ** 3, "l2_cache_bytes": 4 * 1024 * 1024,
        "lds_per_workgroup_bytes": lds_bytes, "lds_per_cu_bytes": lds_bytes,
        "compute_units": compute_units, "wavefront_size": simd_width,
        "max_threads_per_workgroup": 1024, "max_clock_khz": 2400000,
        "memory_clock_khz": 2000000, "memory_bus_width_bits": 8192,
        "pci_domain": 0, "pci_bus": 0, "pci_device": 0,
        "hip_runtime_version": runtime_version, "hip_driver_version": runtime_version,
        "supported": int(supported)}, host=host)


# The schema_version 1 shape (profile.py:452-490 lists the same checks):
# these keys must hold positive ints (bools excluded), these sub-objects must
# hold non-empty strings, and every feature is True, False or None.
_POSITIVE_INT_KEYS = ("max_threads_per_threadgroup", "max_threadgroup_memory_bytes",
                      "simd_width")
_STRING_GROUPS = (("toolchain", ("name", "version")), ("provenance", ("source", "host")))


def _schema_violations(profile):
    """Yield, in a fixed order, every way `profile` breaks the schema."""
    if not isinstance(profile, dict):
        yield "profile must be a dict, got %s" % type(profile).__name__
        return
    version = profile.get("schema_version")
    if version != SCHEMA_VERSION:
        yield "unsupported schema_version %r (expected %d)" % (version, SCHEMA_VERSION)
    if profile.get("backend") not in BACKENDS:
        yield "backend must be one of %s, got %r" % (BACKENDS, profile.get("backend"))
    name = profile.get("device_name")
    if not (isinstance(name, str) and name.strip()):
        yield "device_name must be a non-empty string"
    for key in _POSITIVE_INT_KEYS:
        val = profile.get(key)
        if type(val) is not int or val <= 0:
            yield "%s must be a positive int, got %r" % (key, val)
    for group, fields in _STRING_GROUPS:
        sub = profile.get(group)
        if not isinstance(sub, dict):
            yield "%s must be a dict, got %r" % (group, type(sub).__name__)
            continue
        for field in fields:
            val = sub.get(field)
            if not (isinstance(val, str) and val.strip()):
                yield "%s.%s must be a non-empty string, got %r" % (group, field, val)
    features = profile.get("features")
    if not isinstance(features, dict):
        yield "features must be a dict, got %r" % type(features).__name__
        return
    for fname, val in features.items():
        if type(val) not in (type(None), bool):
            yield "feature %r must be bool or None, got %r" % (fname, val)


def validate_schema(profile):
    """Raise ValueError (the first violation) unless `profile` is a valid
    schema_version 1 profile, with "hip" among the backends."""
    for problem in _schema_violations(profile):
        raise ValueError(problem)


def canonical_json(profile, validate=True):
    """Sorted-key, compact JSON of a profile (profile.py:383-392)."""
    if validate:
        validate_schema(profile)
    return json.dumps(profile, sort_keys=True, separators=(",", ":"))


def profile_hash(profile, validate=True):
    """SHA-256 of canonical_json (profile.py:395-398)."""
    return hashlib.sha256(canonical_json(profile, validate).encode("utf-8")).hexdigest()


_FEATURE_STATUS = ((True, "supported"), (False, "unsupported"))


def render_prompt(profile, validate=True):
    """Deterministic text rendering of a profile, in the reference's prompt
    format (profile.py:401-438); unknown values say they cannot authorise."""
    if validate:
        validate_schema(profile)
    get = profile.get

    def shown(value):
        return "unknown" if value is None else str(value)

    toolchain = get("toolchain") or {}
    prov = get("provenance") or {}
    fields = [("schema_version", get("schema_version", "unknown")),
              ("backend", get("backend", "unknown")),
              ("device_name", get("device_name") or "unknown")]
    fields += [(key, shown(get(key))) for key in _POSITIVE_INT_KEYS]
    fields += [("toolchain", ("%s %s" % (toolchain.get("name") or "unknown",
                                         toolchain.get("version") or "")).strip()),
               ("provenance", "%s on %s" % (prov.get("source") or "unknown",
                                            prov.get("host") or "unknown"))]
    text = ["[hardware_profile]"] + ["%s: %s" % kv for kv in fields] + ["features:"]
    for fname, val in sorted((get("features") or {}).items()):
        status = next((word for flag, word in _FEATURE_STATUS if val is flag),
                      "unknown (cannot authorize)")
        text.append("  %s: %s" % (fname, status))
    return "\n".join(text) + "\n"


def feature_authorized(profile, name):
    """Only an explicit True authorises a feature (profile.py:441-448)."""
    validate_schema(profile)
    return (profile.get("features") or {}).get(name) is True


def save(profile, path):
    """Write the canonical profile to `path`; returns its hash."""
    text = canonical_json(profile)
    with open(path, "w") as fh:
        fh.write(text + "\n")
    return profile_hash(profile)


def load(path):
    """Read and validate a saved profile."""
    with open(path) as fh:
        profile = json.load(fh)
    validate_schema(profile)
    return profile


# ---------------------------------------------------------------------------
# Hashes
# ---------------------------------------------------------------------------

def sha256_file(path):
    h = hashlib.sha256()
    with open(path, "rb") as fh:
        for chunk in iter(lambda: fh.read(1 << 20), b""):
            h.update(chunk)
    return h.hexdigest()


def digest(value):
    """sha256 of sorted-key compact JSON (examples/gemmini_gemm_demo.py:18-19)."""
    return hashlib.sha256(json.dumps(value, sort_keys=True,
                                     separators=(",", ":")).encode()).hexdigest()


def list_digest(values):
    """sha256 of json.dumps(values) with the default separators: the output
    hash of check_local_execution.py:53 for a flat int list."""
    return hashlib.sha256(json.dumps(values).encode()).hexdigest()


def _host_array(t):
    import numpy as np
    try:
        import torch
        if isinstance(t, torch.Tensor):
            return t.detach().contiguous().cpu().numpy()
    except ImportError:
        pass
    return np.ascontiguousarray(np.asarray(t))


def array_record(t):
    """{dtype, shape, sha256} of an array's row-major little-endian bytes."""
    a = _host_array(t)
    if a.dtype.byteorder == ">":
        a = a.astype(a.dtype.newbyteorder("<"))
    return {"dtype": str(a.dtype), "shape": list(a.shape),
            "sha256": hashlib.sha256(a.tobytes(order="C")).hexdigest()}


def artifact_paths():
    """name -> absolute path of every file that determines a result."""
    from ... import build
    paths = {"library": _lib.library_path(),
             "header": os.path.join(build.INCLUDE, "vt_hip_gemm.h"),
             "build_recipe": os.path.abspath(build.__file__),
             "binding": os.path.abspath(_lib.__file__)}
    for src in build.SOURCES + build.PARTS:
        paths["hip_source:" + os.path.basename(src)] = src
    for mod in ("backend", "scaled", "verify", "replay", "provenance"):
        paths["module:" + mod] = os.path.join(PKG_DIR, mod + ".py")
    return paths


def artifact_hashes():
    """name -> {path (relative to the repository root), sha256 or None if absent}."""
    out = {}
    for name, path in sorted(artifact_paths().items()):
        rel = os.path.relpath(path, ROOT) if path.startswith(ROOT + os.sep) else path
        out[name] = {"path": rel,
                     "sha256": sha256_file(path) if os.path.isfile(path) else None}
    return out


# ---------------------------------------------------------------------------
# Run reports
# ---------------------------------------------------------------------------

def report_from_result(plan, A, B, D, C, *, profile=None, vectors=16, seed=0,
                       inputs_description=None, timing=None):
    """Hash-bound report of C = D + A.B for tensors already computed.

    Verifies C on the tensors' device with verify.exact_check and records the
    outcome in "success". Every hash is over data read back after the
    computation, so the report describes exactly the bytes that were checked.
    """
    ok, reason = _backend.validate_plan(plan)
    if not ok:
        raise HipGemmError("invalid plan: " + reason)
    check = _verify.exact_check(A, B, C, D, vectors=vectors, seed=seed)
    if profile is None:
        profile = probe()
    operands = {"A": array_record(A), "B": array_record(B)}
    if D is not None:
        operands["D"] = array_record(D)
    report = {
        "schema_version": REPORT_SCHEMA_VERSION,
        "backend": "hip_gemm",
        "performance_claim": ("none" if timing is None else
                              "HIP-event timings of this library's kernels on the profiled "
                              "device, see `timing`"),
        "verification_boundary": ("exact projection check on the device, modulo 2^32: a "
                                  "wrong result passes with probability at most "
                                  "2^-vectors; no formal certificate"),
        "success": bool(check["passed"]),
        "artifacts": artifact_hashes(),
        "device_profile": profile,
        "device_profile_sha256": profile_hash(profile) if profile is not None else None,
        "plan": plan,
        "plan_sha256": digest(plan),
        "inputs": inputs_description or {"kind": "caller-supplied"},
        "operands": operands,
        "input_sha256": digest([operands[k]["sha256"] for k in sorted(operands)]),
        "output": array_record(C),
        "verification": check,
    }
    numel = 1
    for s in C.shape:
        numel *= int(s)
    if plan["batch"] == 1 and numel <= LIST_DIGEST_MAX_ELEMENTS:
        report["output_list_sha256"] = list_digest(_host_array(C).reshape(-1).tolist())
    if timing is not None:
        report["timing"] = timing
    report["report_sha256"] = digest(report)
    return report


def _inputs_for(plan, mode, seed, device):
    import torch
    from . import inputs as _inputs
    from .runner import _device_inputs
    if mode is None:
        A, B, D = _device_inputs(plan, None, device, seed)
        return A, B, D, {"kind": "seeded", "generator": "torch.randint on the device",
                         "seed": seed}
    if plan["batch"] != 1 or plan["has_d"]:
        raise HipGemmError("deterministic input modes cover batch 1 without D")
    a, b = _inputs.deterministic_inputs(plan["m"], plan["n"], plan["k"], seed, mode)
    return (torch.from_numpy(a).to(device), torch.from_numpy(b).to(device), None,
            {"kind": "deterministic_inputs", "mode": mode, "seed": seed})


def run_report(plan, *, mode=None, seed=0, vectors=16, benchmark_runs=0, device=None,
               out_dir=None):
    """Run `plan` once on the GPU and return its hash-bound report.

    mode: None for seeded random operands, else a deterministic_inputs mode
    ("lcg", "max", "minmax", "min", "zero") with `seed`.
    benchmark_runs > 0 adds HIP-event timings from runner.benchmark_gemm on
    the same inputs. With out_dir the report is written to out_dir/report.json.
    """
    import torch
    ok, reason = _backend.validate_plan(plan)
    if not ok:
        raise HipGemmError("invalid plan: " + reason)
    if not torch.cuda.is_available():
        raise HipGemmError("no GPU available: hip_gemm has no CPU path")
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else device
    A, B, D, desc = _inputs_for(plan, mode, seed, device)
    C = _backend.run(plan, A, B, D)
    torch.cuda.synchronize(device)
    timing = None
    if benchmark_runs > 0:
        from .runner import benchmark_gemm
        inputs = {"A": A, "B": B}
        if D is not None:
            inputs["D"] = D
        res = benchmark_gemm(plan, benchmark_runs, inputs=inputs, device=device)
        timing = {k: res[k] for k in ("gpu_time_ms", "gpu_time_ms_min", "gpu_time_ms_p90",
                                      "num_runs", "warmup", "rotated_sets", "tops", "gbps",
                                      "roofline")}
    report = report_from_result(plan, A, B, D, C, vectors=vectors, seed=seed,
                                inputs_description=desc, timing=timing)
    if out_dir is not None:
        os.makedirs(out_dir, exist_ok=True)
        with open(os.path.join(out_dir, "report.json"), "w") as fh:
            json.dump(report, fh, indent=2)
            fh.write("\n")
    return report


def main(argv=None):
    import argparse
    ap = argparse.ArgumentParser(description="hip_gemm hardware profile and run reports")
    sub = ap.add_subparsers(dest="cmd", required=True)
    sub.add_parser("profile", help="probe the current device and print its profile")
    rp = sub.add_parser("report", help="run one GEMM and print its hash-bound report")
    rp.add_argument("--m", type=int, required=True)
    rp.add_argument("--n", type=int, required=True)
    rp.add_argument("--k", type=int, required=True)
    rp.add_argument("--batch", type=int, default=1)
    rp.add_argument("--variant", default="auto")
    rp.add_argument("--mode", default=None,
                    help="deterministic_inputs mode (lcg, max, minmax, min, zero)")
    rp.add_argument("--seed", type=int, default=0)
    rp.add_argument("--vectors", type=int, default=16)
    rp.add_argument("--benchmark-runs", type=int, default=0)
    rp.add_argument("--out", default=None, help="directory for report.json")
    args = ap.parse_args(argv)
    if args.cmd == "profile":
        try:
            p = normalize_hip(_lib.device_query())
            validate_schema(p)
        except (HipGemmError, ValueError) as exc:
            print("no HIP device profile: %s" % exc, file=sys.stderr)
            return 1
        print(canonical_json(p))
        print("hash:", profile_hash(p))
        print(render_prompt(p), end="")
        return 0
    plan = _backend.make_plan(args.m, args.n, args.k, batch=args.batch, variant=args.variant)
    report = run_report(plan, mode=args.mode, seed=args.seed, vectors=args.vectors,
                        benchmark_runs=args.benchmark_runs, out_dir=args.out)
    print(json.dumps(report, indent=2))
    return 0 if report["success"] else 1


if __name__ == "__main__":
    sys.exit(main())
