#!/bin/bash
# TEST INFRASTRUCTURE ONLY: compiles the unmodified HIP sources for the host
# against tests/hipemu/hip/hip_runtime.h -> tests/hipemu/libtapir_emu.so
#   build_emu.sh [flags]         the emulator the CPU tests load
#   build_emu.sh --asan [flags]  the same with -fsanitize=address,undefined -> libtapir_emu_asan.so: every emulated kernel
#                                test becomes an out-of-bounds test of the global-memory accesses (device buffers are
#                                heap allocations with red zones).  Run through tests/hipemu/run_asan.sh.
set -e
cd "$(dirname "$0")"
OUT=libtapir_emu.so
SAN=""
if [ "$1" == "--asan" ]; then
  shift
  OUT=libtapir_emu_asan.so
  SAN="-fsanitize=address,undefined -fno-sanitize=vptr,function -fno-omit-frame-pointer -shared-libsan -g1"
fi
# one object per translation unit, compiled side by side (build_emu.sh --unit attention: that one only, then the link)
CXX=/opt/rocm/lib/llvm/bin/clang++
OBJ=build/${OUT%.so}
mkdir -p "$OBJ"
UNITS="engine attention"
if [ "$1" == "--unit" ]; then UNITS=$2; shift 2; fi
PIDS=""
for u in $UNITS; do
  $CXX -x c++ -std=c++17 -O2 -fopenmp -fPIC -I. -DTAPIR_EXPERIMENTS $SAN -Wno-unused-value -c ../../tapnet_amd/csrc/$u.hip -o "$OBJ/$u.o" "$@" &
  PIDS="$PIDS $!"
done
for p in $PIDS; do wait $p; done
$CXX -std=c++17 -O2 -fopenmp -fPIC -shared -I. $SAN "$OBJ/engine.o" "$OBJ/attention.o" -x c++ emu_switch.cpp -o $OUT "$@"
