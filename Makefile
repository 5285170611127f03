# Builds libasr_amd.so (gfx950 HIP kernels + C ABI) in-tree.
HIPCC ?= /opt/rocm/bin/hipcc
ARCH ?= gfx950
SRC := $(wildcard asr_amd/csrc/*.hip)
OBJ := $(patsubst asr_amd/csrc/%.hip,build/%.o,$(SRC))
HDR := $(wildcard asr_amd/csrc/*.h) include/asr_amd.h
LIB := asr_amd/lib/libasr_amd.so
# torch bindings of the encoder-layer operators: host code only
NATIVE := asr_amd/lib/_transformer_ops.so
PYTHON ?= python3
CXX := g++
TORCH := $(shell $(PYTHON) -c "import importlib.util as u, os; print(os.path.dirname(u.find_spec('torch').origin))")
PYINC := $(shell $(PYTHON) -c "import sysconfig; print(sysconfig.get_paths()['include'])")
CXXFLAGS := -O3 -std=c++17 -fPIC --offload-arch=$(ARCH) -Wall -Wno-unused-function -Wno-pass-failed -Wno-bitwise-instead-of-logical -Xclang -target-feature -Xclang -packed-fp32-ops

all: $(LIB) $(NATIVE)

build/%.o: asr_amd/csrc/%.hip $(HDR)
	@mkdir -p build
	$(HIPCC) $(CXXFLAGS) -c $< -o $@

$(LIB): $(OBJ)
	@mkdir -p asr_amd/lib
	$(HIPCC) -shared -fPIC --offload-arch=$(ARCH) $(OBJ) -o $@

$(NATIVE): asr_amd/csrc/transformer_ops.cpp include/asr_amd.h | $(LIB)
	$(CXX) -O2 -std=c++17 -fPIC -shared -Wall -D__HIP_PLATFORM_AMD__=1 -DTORCH_EXTENSION_NAME=_transformer_ops -isystem $(TORCH)/include \
	  -isystem $(TORCH)/include/torch/csrc/api/include -isystem /opt/rocm/include -isystem $(PYINC) $< -o $@ \
	  -Lasr_amd/lib -lasr_amd -L$(TORCH)/lib -lc10 -ltorch -ltorch_cpu -ltorch_python -lc10_hip -ltorch_hip '-Wl,-rpath,$$ORIGIN'

clean:
	rm -rf build $(LIB) $(NATIVE)

.PHONY: all clean
