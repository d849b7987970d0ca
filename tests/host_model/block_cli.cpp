// Calls into the CPU build of the operators of sthip_ops.hip, driven by a script (tests/test_block_host.py writes it).  One
// statement per line:
//   buf NAME BYTES [FILE]     a 256-byte aligned buffer of exactly BYTES bytes, filled with 0xA5 or read from FILE
//   save NAME FILE            write a buffer to FILE
//   tile N                    the products' tile (the numbers of sthip_launch7.hpp), -1 = the table's choice
//   dry                       from here on launches are printed (grid x, y, z, block x) instead of run; buffers may be called "@": a place that is never read
//   late 0|1                  direct-to-LDS loads land at once, or not before the lane's wait lets them
//   linear / linear_backward / norm / norm_backward / rotary ARGS...
//                             the entry point of include/strassen_hip.h, arguments in its order without the stream; buffers by
//                             name (NAME+BYTES = a view, "-" = null), strides as three numbers (or "-"), the workspace as one
//                             "ws": the exact size that the query asks for is allocated for the call
#include <stdarg.h>
#include <fstream>
#include <map>
#include <sstream>
#include <string>
#include "host_runtime.h"
#include "strassen_hip.h"

namespace sthip {
int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vfprintf(stderr, fmt, ap);
    va_end(ap);
    fprintf(stderr, "\n");
    return code;
}
void clear_error() {}
static int g_tile = -1;
int debug_tile7() { return g_tile; }
}  // namespace sthip

struct Buf { char* p; size_t n; };
static std::map<std::string, Buf> g_bufs;
static std::vector<HostLaunch> g_launches;
static char* const kNowhere = (char*)((uintptr_t)1 << 40);
static char* alloc(size_t n) { void* p = nullptr; if (posix_memalign(&p, 256, n ? n : 1)) exit(2); memset(p, 0xA5, n); return (char*)p; }

int main(int argc, char** argv) {
    if (argc < 2) return 2;
    std::ifstream script(argv[1]);
    std::string line;
    while (std::getline(script, line)) {
        std::istringstream in(line);
        std::string op;
        if (!(in >> op) || op[0] == '#') continue;
        auto ptr = [&]() -> char* {
            std::string name;
            in >> name;
            if (name == "-") return nullptr;
            if (name == "@" && g_host_dry) return kNowhere;
            const size_t plus = name.find('+');
            const size_t off = plus == std::string::npos ? 0 : std::stoull(name.substr(plus + 1));
            name = name.substr(0, plus);
            if (!g_bufs.count(name)) { fprintf(stderr, "no buffer %s\n", name.c_str()); exit(2); }
            return g_bufs[name].p + off;
        };
        auto num = [&]() { long long v; if (!(in >> v)) { fprintf(stderr, "number expected: %s\n", line.c_str()); exit(2); } return (int64_t)v; };
        auto real = [&]() { double v; if (!(in >> v)) exit(2); return v; };
        Buf ws = {nullptr, 0};
        auto scratch = [&](size_t n) { ws.n = n; if (n) ws.p = g_host_dry ? kNowhere : alloc(n); };
        g_host_global.clear();
        int rc = 0;
        if (op == "buf") {
            std::string name, file;
            in >> name;
            Buf b;
            b.n = num();
            b.p = alloc(b.n);
            if (in >> file) {
                FILE* f = fopen(file.c_str(), "rb");
                if (!f || fread(b.p, 1, b.n, f) != b.n) { fprintf(stderr, "cannot read %s\n", file.c_str()); return 2; }
                fclose(f);
            }
            if (g_bufs.count(name)) free(g_bufs[name].p);
            g_bufs[name] = b;
            continue;
        }
        if (op == "save") {
            std::string name, file;
            in >> name >> file;
            FILE* f = fopen(file.c_str(), "wb");
            if (!f || fwrite(g_bufs[name].p, 1, g_bufs[name].n, f) != g_bufs[name].n) return 2;
            fclose(f);
            continue;
        }
        if (op == "tile") { sthip::g_tile = (int)num(); continue; }
        if (op == "dry") { g_host_dry = &g_launches; continue; }
        if (op == "late") { g_host_late = num() != 0; continue; }
        for (auto& kv : g_bufs) g_host_global.push_back({kv.second.p, kv.second.n});
        if (op == "linear") {
            char *x = ptr(), *W = ptr(), *bias = ptr(), *res = ptr(), *y = ptr(), *pre = ptr();
            int64_t v[7];
            for (auto& e : v) e = num();
            const int dt = num(), act = num();
            scratch(sthip_linear_act_workspace_bytes(v[0], v[1], v[2], dt));
            g_host_global.push_back({ws.p, ws.n});
            rc = sthip_linear_act_forward(x, W, bias, res, y, pre, v[0], v[1], v[2], v[3], v[4], v[5], v[6], dt, act, ws.p, ws.n, nullptr);
        } else if (op == "linear_backward") {
            char *dy = ptr(), *x = ptr(), *W = ptr(), *pre = ptr(), *dx = ptr(), *dW = ptr(), *db = ptr();
            int64_t v[6];
            for (auto& e : v) e = num();
            const int dt = num(), act = num();
            scratch(sthip_linear_act_backward_workspace_bytes(v[0], v[1], v[2], dt, act));
            g_host_global.push_back({ws.p, ws.n});
            rc = sthip_linear_act_backward(dy, x, W, pre, dx, dW, db, v[0], v[1], v[2], v[3], v[4], v[5], dt, act, ws.p, ws.n, nullptr);
        } else if (op == "norm") {
            char *x = ptr(), *w = ptr(), *b = ptr(), *y = ptr(), *mean = ptr(), *rstd = ptr();
            int64_t v[4];
            for (auto& e : v) e = num();
            const int dt = num(), pdt = num();
            rc = sthip_layer_norm_forward(x, w, b, y, (float*)mean, (float*)rstd, v[0], v[1], v[2], v[3], dt, pdt, real(), nullptr);
        } else if (op == "norm_backward") {
            char *dy = ptr(), *x = ptr(), *w = ptr(), *mean = ptr(), *rstd = ptr(), *dx = ptr(), *dw = ptr(), *db = ptr();
            int64_t v[5];
            for (auto& e : v) e = num();
            const int dt = num(), pdt = num();
            scratch(sthip_layer_norm_backward_workspace_bytes(v[0], v[1]));
            rc = sthip_layer_norm_backward(dy, x, w, (float*)mean, (float*)rstd, dx, dw, db, v[0], v[1], v[2], v[3], v[4], dt, pdt, ws.p, ws.n, nullptr);
        } else if (op == "rotary") {
            char *q = ptr(), *k = ptr(), *qo = ptr(), *ko = ptr();
            int64_t v[6], s[4][3];
            for (auto& e : v) e = num();
            for (auto& t : s) for (auto& e : t) e = num();
            char *freq = ptr(), *pos = ptr();
            const int bits = num();
            const int64_t pb = num(), pt = num(), first = num();
            const double gain = real();
            const int inter = num(), inverse = num(), dt = num();
            rc = sthip_rotary(q, k, qo, ko, v[0], v[1], v[2], v[3], v[4], v[5], s[0], s[1], s[2], s[3], (double*)freq, pos, bits, pb, pt, first, gain, inter, inverse, dt, nullptr);
        } else {
            fprintf(stderr, "unknown statement %s\n", op.c_str());
            return 2;
        }
        if (g_host_dry) {
            printf("%d", rc);
            for (const HostLaunch& l : g_launches) printf(" %u,%u,%u,%u", l.grid[0], l.grid[1], l.grid[2], l.block[0]);
            printf("\n");
            g_launches.clear();
            continue;
        }
        free(ws.p);
        if (rc) { fprintf(stderr, "%s returned %d\n", line.c_str(), rc); return 1; }
    }
    for (auto& kv : g_bufs) free(kv.second.p);
    g_bufs.clear();
    return 0;
}
