#!/bin/bash
# Builds libtapir_hip.so for gfx950 (MI355X) in-tree.  hipcc cross-compiles without a GPU.
#   build.sh              the product library (tapnet_amd/csrc/libtapir_hip.so)
#   build.sh --exp        a -DTAPIR_EXPERIMENTS build for tools/kbench.py (phase traces, experiment kernels) into
#                         tools/bin/libtapir_hip_exp.so -- not next to the product library, never loaded by the package
#                         unless TAPIR_HIP_LIB points at it
#   build.sh --slp        engine.hip WITH hipcc's SLP pass into tools/libtapir_hip_slp.so: the build that shows the hazard
#                         below (tools/r06.sh, TAPIR_HIP_LIB=... pytest tests/test_gpu_cotenant.py fails with it); never shipped
#
# -fno-slp-vectorize, and the check behind the build: on MI355X `v_pk_fma_f32 ... op_sel:[0,1,0]` (low result from the HIGH
# half of a source) loses its low result in lanes 48-63 while ANY other wave of the SIMD -- another stream, another process --
# issues MFMAs back to back; a dependent pair of packed FMAs does it every time (stand-alone reproducer without this
# library: tools/micro/run_cotenant_repro.py, log profiles/r06_cotenant_repro.txt).  hipcc's SLP vectoriser writes such forms
# when it packs scalar code (mix_kernel's temporal convolution: the run-to-run differences of the few-row mixer with two
# processes on one GPU, profiles/r06_cotenant_fault.txt); the hand-packed kernels (f32x2 arithmetic) never select a high half
# for a low result.  Without the pass the code object holds no packed-f32 arithmetic with an op_sel modifier at all --
# check_packed_forms.py fails the build if one ever reappears.
set -e
cd "$(dirname "$0")"
BASE="--offload-arch=gfx950 -O3 -std=c++17 -fPIC -Wno-unused-result -fno-slp-vectorize"
LINK="--offload-arch=gfx950 -fPIC -shared"
# attention.hip: no packed-f32 arithmetic at all (its host pass warns that it does not know the feature)
FLAGS_attention="-Xclang -target-feature -Xclang -packed-fp32-ops"
FLAGS_engine=""
if [ "$1" == "--exp" ]; then
  shift
  mkdir -p ../../tools/bin build
  hipcc $BASE $FLAGS_attention -DTAPIR_EXPERIMENTS -c attention.hip -o build/attention_exp.o "$@"
  hipcc $BASE -DTAPIR_EXPERIMENTS -c engine.hip -o build/engine_exp.o "$@"
  hipcc $LINK build/engine_exp.o build/attention_exp.o -o ../../tools/bin/libtapir_hip_exp.so
  exec python3 check_packed_forms.py ../../tools/bin/libtapir_hip_exp.so 2
fi
if [ "$1" == "--slp" ]; then
  shift
  mkdir -p build
  hipcc $BASE $FLAGS_attention -c attention.hip -o build/attention.o
  hipcc ${BASE/ -fno-slp-vectorize/} -c engine.hip -o build/engine_slp.o "$@"
  exec hipcc $LINK build/engine_slp.o build/attention.o -o ../../tools/libtapir_hip_slp.so
fi
# one object per translation unit, compiled side by side (build.sh --unit attention: that one only, then the link)
UNITS="engine attention"
if [ "$1" == "--unit" ]; then UNITS=$2; shift 2; fi
mkdir -p build
PIDS=""
for u in $UNITS; do
  x=FLAGS_$u
  hipcc $BASE ${!x} -c $u.hip -o build/$u.o "$@" &
  PIDS="$PIDS $!"
done
for p in $PIDS; do wait $p; done
hipcc $LINK build/engine.o build/attention.o -o libtapir_hip.so
python3 check_packed_forms.py libtapir_hip.so 2
# the operators on torch tensors (host code: argument checks, autograd nodes)
TORCH=$(python3 -c "import importlib.util, os; print(os.path.dirname(importlib.util.find_spec('torch').origin))")
PYINC=$(python3 -c "import sysconfig; print(sysconfig.get_paths()['include'])")
if [ "$UNITS" == "engine attention" ] || [ torch_ops.cpp -nt ../_torch_ops.so ] || [ ../../include/tapir_hip.h -nt ../_torch_ops.so ]; then
  g++ -O2 -std=c++17 -fPIC -shared -fvisibility=hidden -D__HIP_PLATFORM_AMD__ -DUSE_ROCM -DTORCH_EXTENSION_NAME=_torch_ops \
    -isystem "$TORCH/include" -isystem "$TORCH/include/torch/csrc/api/include" -isystem /opt/rocm/include -isystem "$PYINC" \
    torch_ops.cpp -o ../_torch_ops.so -L. -ltapir_hip -L"$TORCH/lib" -ltorch -ltorch_cpu -ltorch_hip -ltorch_python -lc10 -lc10_hip \
    -Wl,-rpath,'$ORIGIN/csrc'
fi
